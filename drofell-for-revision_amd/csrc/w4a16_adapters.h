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
// kTileRows positions of one adapter, a chunk up to kChunkRows rows of it.
// Chunks of an adapter that has several leave a share of its gradients each.
// The counts are bounds that the host knows: an adapter has several chunks from kChunkRows + 1 rows on.
//
// Measured against tiles of 64 positions (both products of a serving call, 4096 x 4096, rank 16): 256 rows of
// 32 adapters 9.9 us against 12.1, 2048 rows of 8 18.4 against 24.5, 8192 of 8 51 against 73.  Rank 64 with
// all rows on one adapter is better off with 64 (4096 rows 58 against 65): one size serves all.
constexpr int kTileRows = 32, kChunkRows = 512;
struct AdapterLayout {
  int tiles, chunks, shares;
  int64_t positions;
  // offsets (int32) in the plan
  int64_t tile_adapter, chunk, chunk_start, order, ints;
};
inline AdapterLayout adapter_layout(int rows, int adapters) {
  AdapterLayout l = {};
  const int segs = std::min(adapters + 1, rows);
  l.tiles = rows / kTileRows + segs;
  l.chunks = rows / kChunkRows + segs;
  l.shares = rows / kChunkRows + std::min(adapters, rows / (kChunkRows + 1));
  if (rows <= kChunkRows) l.shares = 0;
  l.positions = (int64_t)l.tiles * kTileRows;
  l.tile_adapter = 4;  // behind the head: [0] tiles that hold rows
  l.chunk = l.tile_adapter + ((l.tiles + 3) & ~3);
  l.chunk_start = l.chunk + 4 * (int64_t)l.chunks;
  l.order = (l.chunk_start + adapters + 2 + 3) & ~(int64_t)3;
  l.ints = l.order + l.positions;
  return l;
}

// The rank that the matrix instructions see.
inline int padded_rank(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }

// h (or dh) of every position as 16-bit operands in two parts (split16), in two forms:
//   by row     [2][positions][padded rank], with an exponent per position;
//   by column  [2][positions / 8][padded rank][8], the eight positions side by side, with an
//              exponent per 32 positions and column.
// bf16 operands have no exponents.
struct AdapterPacks {
  uint16_t* row;
  int32_t* row_exp;
  uint16_t* col;
  int32_t* col_exp;
};
inline size_t row_pack_bytes(const AdapterLayout& l, int r) { return (size_t)l.positions * (4 * padded_rank(r) + 4); }
inline size_t col_pack_bytes(const AdapterLayout& l, int r) {
  return (size_t)l.positions * 4 * padded_rank(r) + (size_t)l.positions / 32 * padded_rank(r) * 4;
}
inline void place_row(AdapterPacks& p, const AdapterLayout& l, int r, void* at) {
  p.row = static_cast<uint16_t*>(at);
  p.row_exp = reinterpret_cast<int32_t*>(p.row + 2 * (size_t)l.positions * padded_rank(r));
}
inline void place_col(AdapterPacks& p, const AdapterLayout& l, int r, void* at) {
  p.col = static_cast<uint16_t*>(at);
  p.col_exp = reinterpret_cast<int32_t*>(p.col + 2 * (size_t)l.positions * padded_rank(r));
}

struct AdapterArgs {
  AdapterLayout l;
  bool bf16;
  int k, n, r, adapters;
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
  // backward
  const uint16_t* g;     // [rows][n]
  int64_t ldg;
  uint16_t* dx;          // or null
  int64_t lddx;
  uint16_t* da;          // or null
  uint16_t* db;          // or null
  void* h;               // h by column: written by a forward pass that keeps it, read by the backward pass
  unsigned char* ws;
};

// Parts of the reduced axis in which rows are multiplied with A (or their gradients with B).
constexpr int kMaxSplits = 16;
int adapter_splits(const AdapterLayout& l, int width, int cus);

// Workspaces: offsets in bytes.
struct ForwardWs {
  int splits;
  size_t bytes;  // planes [splits][positions][r]
};
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
inline size_t plane_bytes(const AdapterLayout& l, int splits, int r) {
  return up256(sizeof(float) * splits * (size_t)l.positions * r);
}
inline ForwardWs forward_ws(const AdapterLayout& l, int k, int r, int cus) {
  ForwardWs w;
  w.splits = adapter_splits(l, k, cus);
  w.bytes = plane_bytes(l, w.splits, r);
  return w;
}
struct BackwardWs {
  int splits;
  size_t at, bt, row, col, da, db, bytes;
};
inline BackwardWs backward_ws(const AdapterLayout& l, int k, int n, int r, int adapters, int cus) {
  BackwardWs w;
  w.splits = adapter_splits(l, n, cus);
  w.at = plane_bytes(l, w.splits, r);
  w.bt = w.at + up256((size_t)2 * adapters * r * k);
  w.row = w.bt + up256((size_t)2 * adapters * r * n);
  w.col = w.row + up256(row_pack_bytes(l, r));
  w.da = w.col + up256(col_pack_bytes(l, r));
  w.db = w.da + up256(sizeof(float) * l.shares * (size_t)r * k);
  w.bytes = w.db + sizeof(float) * l.shares * (size_t)r * n;
  return w;
}

// What a kernel that multiplies rows with transposed weights reads: in [rows][width],
// weights [adapters][r][width].
struct ShrinkArgs {
  AdapterLayout l;
  const int32_t* plan;
  const uint16_t* in;
  int64_t ld;
  const uint16_t* weights;
  int width, r, adapters, drop;
  const int64_t* seed;
  float* planes;
};
// Workgroups of the gradients' largest launches (w4a16_adapters_grad.hip): the weights turned around with g h^T, and
// dh x^T with dx.
inline int64_t grad_workgroups(const AdapterLayout& l, int k, int n, int r, int adapters) {
  const int64_t kt = (k + 63) / 64, nt = (n + 63) / 64;
  return std::max((r + 63) / 64 * (kt + nt) * adapters + l.chunks * nt, l.chunks * kt);
}
hipError_t launch_shrink(bool bf16, const ShrinkArgs& a, int splits, hipStream_t stream);
hipError_t launch_join(const AdapterArgs& a, const float* planes, int splits, const AdapterPacks& p, hipStream_t stream);
hipError_t launch_adapter_plan(const AdapterLayout& l, int rows, int adapters, const int32_t* index, int32_t* plan,
                               hipStream_t stream);
hipError_t launch_adapters(const AdapterArgs& a, const ForwardWs& w, hipStream_t stream);
hipError_t launch_adapters_grad(const AdapterArgs& a, const BackwardWs& w, hipStream_t stream);
hipError_t launch_dropout(bool bf16, int rows, int cols, const uint16_t* x, int64_t ldx, uint16_t* y, int64_t ldy, int drop,
                          float keep_scale, const int64_t* seed, hipStream_t stream);

}  // namespace dw4
