// Internal interface of the low-rank adapters' and the dropout kernels
// (w4a16_adapters.hip, w4a16_adapters_grad.hip) for the C ABI
// (w4a16_capi_adapters.hip).  Not installed; the public ABI is
// include/drofell_w4a16.h.
#pragma once

#include <algorithm>

#include "w4a16_internal.h"

namespace dw4 {

constexpr int kAdapterMaxRank = 128, kAdapterMaxCount = 1024;
constexpr int kAdapterMaxRows = 1 << 24;

// How the rows of a call are laid out by adapter: rows sorted by adapter (those
// without one last), each adapter's from a tile of its own on.  A tile holds
// `align` positions of one adapter, a chunk up to kChunkTiles(align) tiles of it.
// The counts are bounds that the host knows.
struct AdapterLayout {
  int align, tiles, chunks, chunk_rows;
  int64_t positions;
  // offsets (int32) in the plan
  int64_t tile_adapter, chunk, chunk_start, order, ints;
};
constexpr int kFewRows = 256;  // rows up to which tiles hold 16 positions, above it 64
inline AdapterLayout adapter_layout(int rows, int adapters) {
  AdapterLayout l = {};
  l.align = rows <= kFewRows ? 16 : 64;
  l.chunk_rows = 256;
  const int segs = std::min(adapters + 1, rows);
  l.tiles = rows / l.align + segs;
  l.chunks = rows / l.chunk_rows + segs;
  l.positions = (int64_t)l.tiles * l.align;
  l.tile_adapter = 0;
  l.chunk = (l.tiles + 3) & ~3;
  l.chunk_start = l.chunk + 4 * (int64_t)l.chunks;
  l.order = (l.chunk_start + adapters + 2 + 3) & ~(int64_t)3;
  l.ints = l.order + l.positions;
  return l;
}

struct AdapterArgs {
  AdapterLayout l;
  bool bf16;
  int rows, k, n, r, adapters;
  const int32_t* plan;
  const uint16_t* x;     // [rows][k]
  int64_t ldx;
  const uint16_t* a;     // [adapters][r][k]
  const uint16_t* b;     // [adapters][n][r]
  const float* scaling;  // [adapters]
  int drop;              // of 65536; 0: no dropout
  const int64_t* seed;   // key, offset
  float keep_scale;      // 65536 / (65536 - drop), 0 where that is infinite
  // forward
  const uint16_t* base;  // [rows][n]
  int64_t ldb;
  uint16_t* out;
  int64_t ldo;
  float* h;              // [positions][r], A x of the kept elements, or null
  // backward
  const uint16_t* g;     // [rows][n]
  int64_t ldg;
  uint16_t* dx;          // or null
  int64_t lddx;
  uint16_t* da;          // or null
  uint16_t* db;          // or null
  float* ws;
};

// Forward: the rows' products with A in `splits` parts of k.
int adapter_splits(const AdapterLayout& l, int k, int cus);
inline size_t adapter_ws_floats(const AdapterLayout& l, int splits, int r) { return (size_t)splits * l.positions * r; }
// Backward: dH in a plane per slab of kSlab columns, its sum, and each chunk's share of dA and dB.
constexpr int kSlab = 256;
struct AdapterGradParts {
  size_t dh, da, db, floats;  // offsets (floats) behind the planes, and the whole
};
inline AdapterGradParts adapter_grad_parts(const AdapterLayout& l, int k, int n, int r) {
  AdapterGradParts p;
  const size_t plane = (size_t)l.positions * r;
  p.dh = (size_t)((n + kSlab - 1) / kSlab) * plane;
  p.da = p.dh + plane;
  p.db = p.da + (size_t)l.chunks * r * k;
  p.floats = p.db + (size_t)l.chunks * r * n;
  return p;
}

hipError_t launch_adapter_plan(const AdapterLayout& l, int rows, int adapters, const int32_t* index, int32_t* plan,
                               hipStream_t stream);
hipError_t launch_adapters(const AdapterArgs& a, int splits, hipStream_t stream);
hipError_t launch_adapters_grad(const AdapterArgs& a, hipStream_t stream);
hipError_t launch_dropout(bool bf16, int rows, int cols, const uint16_t* x, int64_t ldx, uint16_t* y, int64_t ldy, int drop,
                          float keep_scale, const int64_t* seed, hipStream_t stream);

}  // namespace dw4
