// Low-rank adapters of many requests beside a shared projection:
//   out_t = base_t + s_a B_a A_a d(x_t),   a = the row's adapter (or none),
// with d dropout whose mask comes from a counter; and that dropout by itself.
//
// Rows are sorted by adapter once per batch (plan_kernel), so that a tile of 32
// positions has one adapter and both its products run on 16 x 16 x 32 matrix
// instructions, rows as their columns.  The rows' products with A are formed in parts of k
// over workgroups and waves (fp32 planes), joined in order into 16-bit operands, and
// multiplied with B on top of the projection's output, which is rounded once.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "w4a16_adapters_device.h"

namespace dw4 {

namespace {

constexpr int kThreads = 256, kJoinThreads = 512;
constexpr int kHalves = kTileRows / 16;
constexpr int kPlanThreads = 512, kPlanWaves = kPlanThreads / 64;

// Exclusive sums of v[0 .. n) in LDS (n at most 1026), in place; v[n] becomes the total.
__device__ void scan_ints(int* v, int n, int* wave_sum) {
  constexpr int kEach = (kAdapterMaxCount + 1 + kPlanThreads - 1) / kPlanThreads;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int own[kEach], sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    own[e] = t * kEach + e < n ? v[t * kEach + e] : 0;
    sum += own[e];
  }
  int x = sum;
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  if (lane == 63) wave_sum[wave] = x;
  __syncthreads();
  int before = x - sum, total = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) before += wave_sum[w];
    total += wave_sum[w];
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (t * kEach + e < n) v[t * kEach + e] = before;
    before += own[e];
  }
  if (t == 0) v[n] = total;
  __syncthreads();
}

// The last segment i with start[i] <= t (start ascending, n segments).
__device__ __forceinline__ int segment_of(const int* start, int n, int t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// One workgroup: rows counted by adapter (each wave a run of them), the adapters'
// first tiles and chunks by a scan, then each row to its place, in order within its adapter.  Bound by
// one CU's passes over the rows' numbers: 1 row 4.6 us, 5325 rows 16, 10175 rows 27, once per batch for
// all projections of all layers.
__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(AdapterLayout l, int rows, int adapters, const int32_t* __restrict__ index, int32_t* __restrict__ plan) {
  extern __shared__ int sm[];
  const int segs = adapters + 1;  // the last: rows without an adapter
  int* const count = sm;                         // [waves][segs], later each wave's next position
  int* const total = count + kPlanWaves * segs;  // [segs]
  int* const tile0 = total + segs;               // [segs + 1]
  int* const chunk0 = tile0 + segs + 1;          // [segs + 1]
  int* const share0 = chunk0 + segs + 1;         // [segs + 1]
  int* const wave_sum = share0 + segs + 1;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int i = t; i < kPlanWaves * segs; i += kPlanThreads) count[i] = 0;
  __syncthreads();
  const int run = ((rows + kPlanWaves - 1) / kPlanWaves + 63) & ~63;
  const int from = min(wave * run, rows), to = min(from + run, rows);
  auto segment = [&](int row) {
    const int a = index[row];
    return a >= 0 && a < adapters ? a : adapters;
  };
  for (int row = from + lane; row < to; row += 64) atomicAdd(&count[wave * segs + segment(row)], 1);
  __syncthreads();
  for (int s = t; s < segs; s += kPlanThreads) {
    int n = 0;
    for (int w = 0; w < kPlanWaves; ++w) n += count[w * segs + s];
    total[s] = n;
    tile0[s] = (n + kTileRows - 1) / kTileRows;
    chunk0[s] = (n + kChunkRows - 1) / kChunkRows;
    share0[s] = s < adapters && n > kChunkRows ? chunk0[s] : 0;
  }
  __syncthreads();
  scan_ints(tile0, segs, wave_sum);
  scan_ints(chunk0, segs, wave_sum);
  const bool several = l.shares > 0;  // adapters of several chunks there may be
  if (several) scan_ints(share0, segs, wave_sum);
  for (int s = t; s < segs; s += kPlanThreads) {
    int at = tile0[s] * kTileRows;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int n = count[w * segs + s];
      count[w * segs + s] = at;
      at += n;
    }
  }
  if (t == 0) plan[0] = tile0[segs];
  for (int s = t; s <= segs; s += kPlanThreads) plan[l.chunk_start + s] = chunk0[s];
  for (int i = t; i < l.tiles; i += kPlanThreads)
    plan[l.tile_adapter + i] = i < tile0[segs] ? segment_of(tile0, segs, i) : -1;
  for (int i = t; i < l.chunks; i += kPlanThreads) {
    int4 c = make_int4(-1, 0, 0, -1);  // adapter, first position, rows, share or -1
    if (i < chunk0[segs]) {
      const int s = segment_of(chunk0, segs, i), j = i - chunk0[s], at = j * kChunkRows;
      c = make_int4(s, tile0[s] * kTileRows + at, min(kChunkRows, total[s] - at), several && share0[s] < share0[s + 1] ? share0[s] + j : -1);
    }
    *(int4*)(plan + l.chunk + 4 * i) = c;
  }
  for (int i = t; i < l.positions; i += kPlanThreads) {  // positions without a row
    const int tile = i / kTileRows;
    const int s = tile < tile0[segs] ? segment_of(tile0, segs, tile) : -1;
    if (s < 0 || i - tile0[s] * kTileRows >= total[s]) plan[l.order + i] = -1;
  }
  __syncthreads();
  for (int first = from; first < to; first += 64) {
    const int row = first + lane;
    const int s = row < to ? segment(row) : -1;
    uint64_t left = __ballot(s >= 0);
    while (left) {
      const int lead = __builtin_ctzll(left);
      const int key = __shfl(s, lead);
      const uint64_t same = __ballot(s == key);
      const int at = count[wave * segs + key];
      if (s == key) plan[l.order + at + __popcll(same & ((1ull << lane) - 1))] = row;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the other lanes have read it
      if (lane == lead) count[wave * segs + key] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      left &= ~same;
    }
  }
}

// Rows' products with A (or gradients' with B): a tile's positions and a part of the reduced axis, of which
// each wave takes a part of its own, 64 columns a step.  What bounds it is the rows, read once (nontemporal,
// whole lines); A stays in the XCD's L2, and neighbouring items share it.  Two steps' loads are in flight
// where the registers allow it.  10175 rows of 11008 against rank 16: 42 us for 222 MB, 5.3 TB/s; 1 row of
// 4096 3.8 us, a launch and two trips to memory.
template <bool BF, int NT, bool DROP>
__global__ void __launch_bounds__(kThreads) shrink_kernel(ShrinkArgs p, int splits) {
  constexpr int kAhead = NT <= 2 ? 2 : 1;  // steps whose loads are in flight together
  __shared__ __attribute__((aligned(16))) float red[4][kTileRows][20];
  __shared__ u4 lines[4][128];
  const int item = item_of_xcd(blockIdx.x, p.plan[0] * splits);
  if (item < 0) return;
  const int tile = item / splits, split = item - tile * splits;
  const int ad = p.plan[p.l.tile_adapter + tile];
  if (ad >= p.adapters) return;
  const int lane = threadIdx.x & 63, wave = wave_index(), g = lane >> 4, c = lane & 15, unit = lane & 7, line = lane >> 3;
  const int32_t* order = p.plan + p.l.order + (int64_t)tile * kTileRows;
  const uint16_t* xr[kHalves][2];
  int row[kHalves][2];
#pragma unroll
  for (int t = 0; t < kHalves; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      row[t][i] = max(order[t * 16 + 8 * i + line], 0);
      xr[t][i] = p.in + row[t][i] * p.ld;
    }
  const uint16_t* ar[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) ar[t][i] = p.weights + ((int64_t)ad * p.r + min(t * 16 + 8 * i + line, p.r - 1)) * p.width;
  // a tile of few rows: its second half may hold none
  const bool two = __builtin_amdgcn_readfirstlane(order[16]) >= 0;
  f4 acc[kHalves][NT] = {};
  const Philox philox(DROP ? p.seed : reinterpret_cast<const int64_t*>(p.plan));
  const int steps = (p.width + 63) / 64, parts = splits * 4, part = split * 4 + wave;
  const int s0 = (int)((int64_t)steps * part / parts), s1 = (int)((int64_t)steps * (part + 1) / parts);
  struct Step {
    u4 x[kHalves][2], a[NT][2];
  };
  auto load = [&](int at, Step& v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int t = 0; t < kHalves; ++t)
        if (t == 0 || two) v.x[t][i] = stream_load(xr[t][i] + at);
#pragma unroll
      for (int t = 0; t < NT; ++t) v.a[t][i] = *(const u4*)(ar[t][i] + at);
    }
  };
  auto multiply = [&](int s, Step& v) {
#pragma unroll
    for (int t = 0; t < NT; ++t) to_operands(v.a[t][0], v.a[t][1], lines[wave]);
#pragma unroll
    for (int t = 0; t < kHalves; ++t) {
      if (t > 0 && !two) break;
      if constexpr (DROP) {
#pragma unroll
        for (int i = 0; i < 2; ++i) v.x[t][i] &= philox.mask(s * 8 + unit, row[t][i], p.drop);
      }
      to_operands(v.x[t][0], v.x[t][1], lines[wave]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = mfma16_of<BF>(v.a[u][i], v.x[t][i], acc[t][u]);
    }
  };
  const int whole = min(s1, p.width / 64);
  int s = s0;
  for (; s + kAhead <= whole; s += kAhead) {
    Step v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load((s + i) * 64 + unit * 8, v[i]);
    __builtin_amdgcn_sched_barrier(0);  // (else the loads sink to where they are used)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) multiply(s + i, v[i]);
  }
  for (; s < s1; ++s) {  // (the last may be a part of a step)
    const bool in = s * 64 + unit * 8 < p.width;
    Step v;
    load(in ? s * 64 + unit * 8 : 0, v);
    if (!in) v = Step{};
    multiply(s, v);
  }
  float* plane = p.planes + ((int64_t)split * p.l.positions + (int64_t)tile * kTileRows) * p.r;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    if (u) __syncthreads();
#pragma unroll
    for (int t = 0; t < kHalves; ++t) *(f4*)&red[wave][t * 16 + c][4 * g] = acc[t][u];
    __syncthreads();
    const int i = threadIdx.x >> 2, q = (threadIdx.x & 3) * 4;
    if (i < kTileRows && u * 16 + q < p.r) {
      f4 v = *(const f4*)&red[0][i][q];
#pragma unroll
      for (int w = 1; w < 4; ++w) v += *(const f4*)&red[w][i][q];
      if (order[i] < 0) v = f4{};
      *(f4*)(plane + (int64_t)i * p.r + u * 16 + q) = v;
    }
  }
}

// The sum of a value's planes, in order, all their loads in flight.
__device__ __forceinline__ f4 sum_planes(const float* at, int64_t plane, int splits) {
  f4 x[kMaxSplits], v = {};
#pragma unroll
  for (int e = 0; e < kMaxSplits; ++e) x[e] = *(const f4*)(at + min(e, splits - 1) * plane);
#pragma unroll
  for (int e = 0; e < kMaxSplits; ++e)
    if (e < splits) v += x[e];
  return v;
}

// 32 positions' h (or dh) v [32][kR + 1], from position `first` on, by column (AdapterPacks).
template <bool BF, int kR>
__device__ __forceinline__ void pack_columns(const float* v, const AdapterPacks& packs, int64_t first, int64_t positions,
                                             int threads) {
  for (int i = threadIdx.x; i < 4 * kR; i += threads) {  // column i % kR, eight rows
    const int col = i % kR, r0 = i / kR * 8;
    int ex = 0;
    if constexpr (!BF) {
      float m = 0.f;
      for (int e = 0; e < 32; ++e) m = fmaxf(m, finite_magnitude(v[e * (kR + 1) + col]));
      ex = range_exponent<BF>(m);
      if (r0 == 0) packs.col_exp[first / 32 * kR + col] = -ex;
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = BF ? v[(r0 + e) * (kR + 1) + col] : times_pow2(v[(r0 + e) * (kR + 1) + col], ex);
    u4 hi, lo;
    split16<BF>(x, hi, lo);
    uint16_t* to = packs.col + ((first + r0) * kR + col * 8);
    *(u4*)to = hi;
    *(u4*)(to + positions * kR) = lo;
  }
}

// 32 positions' dh: planes summed in order, times s_a / kept share, packed by row and by column.  Bound
// by its launch and the trip to the planes: 5325 rows of rank 16 3.6 us, 1763 of rank 64 5.2.
template <bool BF, int NT>
__global__ void __launch_bounds__(kJoinThreads)
join_kernel(AdapterArgs p, const float* planes, int splits, AdapterPacks packs) {
  constexpr int kR = NT * 16;
  __shared__ float v[32][kR + 1];
  __shared__ int exps[32];
  const int64_t first = (int64_t)blockIdx.x * 32;
  const int ad = p.plan[p.l.tile_adapter + first / kTileRows];
  if (ad < 0 || ad >= p.adapters) return;
  const float scale = p.scaling[ad] * p.keep_scale;
  for (int i = threadIdx.x; i < 32 * (kR / 4); i += kJoinThreads) {
    const int at = i / (kR / 4), q = i % (kR / 4) * 4;
    f4 s = {};
    if (q < p.r) s = sum_planes(planes + (first + at) * p.r + q, p.l.positions * p.r, splits) * scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[at][q + e] = s[e];
  }
  __syncthreads();
  if (packs.row != nullptr) {
    if constexpr (!BF) {  // sixteen threads a row
      const int at = threadIdx.x >> 4;
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < kR / 16; ++e) m = fmaxf(m, finite_magnitude(v[at][(threadIdx.x & 15) + 16 * e]));
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
      if ((threadIdx.x & 15) == 0) {
        exps[at] = range_exponent<BF>(m);
        packs.row_exp[first + at] = -exps[at];
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 32 * (kR / 8); i += kJoinThreads) {
      const int at = i / (kR / 8), q = i % (kR / 8) * 8;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = BF ? v[at][q + e] : times_pow2(v[at][q + e], exps[at]);
      u4 hi, lo;
      split16<BF>(x, hi, lo);
      uint16_t* to = packs.row + (first + at) * kR + q;
      *(u4*)to = hi;
      *(u4*)(to + p.l.positions * kR) = lo;
    }
  }
  if (packs.col != nullptr) pack_columns<BF, kR>(&v[0][0], packs, first, p.l.positions, kJoinThreads);
}

// The products with B, added in 32 bits to the projection's output: a tile's rows, a part of the columns, of
// which each wave takes every fourth group of 64.  A workgroup sums the tile's planes itself; h goes into the
// product as two 16-bit parts, so that nothing but the result is rounded to 16 bits.  Where h is kept, the tile's
// first workgroup packs it by column: 5325 rows of rank 16 20.2 us that way, 18.7 by rows that a launch of
// 4.1 had packed before; 1763 of rank 64 35.1, and 28.5 behind 5.1.
// Bound by the output, read and written once as whole lines: 10175 rows of 4096 by rank 16 40 us for 169 MB,
// 4.2 TB/s; rank 64 by 11008 by its reads of the L2, 241 MB for 91 (1763 rows 35 us): about 124 of planes, which
// each of a tile's 17 workgroups sums anew, and 80 of B, which goes to every tile.
// The first group's loads before the planes' sums take the registers of a wave (10175 rows 50.5 us for 40.2).
template <bool BF, int NT>
__global__ void __launch_bounds__(kThreads) expand_kernel(AdapterArgs p, int splits, AdapterPacks packs, int wide) {
  constexpr int kR = NT * 16, kPitch = kR + 8, kJ = NT == 1 ? 1 : NT / 2;
  const int item = item_of_xcd(blockIdx.x, p.plan[0] * wide);
  if (item < 0) return;
  const int tile = item / wide, column_part = item - tile * wide;
  const int ad = p.plan[p.l.tile_adapter + tile];
  const int lane = threadIdx.x & 63, wave = wave_index(), g = lane >> 4, c = lane & 15;
  const int32_t* order = p.plan + p.l.order + (int64_t)tile * kTileRows;
  const int groups = (p.n + 63) / 64;
  const int g0 = (int)((int64_t)groups * column_part / wide), g1 = (int)((int64_t)groups * (column_part + 1) / wide);
  if (ad >= p.adapters) {  // rows without an adapter keep the projection's output
    if (p.out == p.base) return;
    const int units = min(g1 * 8, p.n / 8) - g0 * 8;
    for (int i = threadIdx.x; i < kTileRows * units; i += kThreads) {
      const int row = order[i / units], at = (g0 * 8 + i % units) * 8;
      if (row >= 0) *(u4*)(p.out + row * p.ldo + at) = stream_load(p.base + row * p.ldb + at);
    }
    return;
  }
  // rows as loads and stores take them (to_operands())
  int row[kHalves][2];
  const uint16_t* from[kHalves][2];
#pragma unroll
  for (int t = 0; t < kHalves; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      row[t][i] = order[t * 16 + 8 * i + (lane >> 3)];
      from[t][i] = p.base + max(row[t][i], 0) * p.ldb;
    }
  // a tile of few rows: its second half may hold none
  const bool two = __builtin_amdgcn_readfirstlane(order[16]) >= 0;
  const int unit = lane & 7;
  const uint16_t* const bw = p.b + (int64_t)ad * p.n * p.r;
  struct Group {
    u4 y[kHalves][2], b[4][kJ];
  };
  // the lane's eight columns of unit g (operands 0 and 1) and of unit 4 + g (2 and 3)
  auto load = [&](int grp, Group& v) {
    const int n = grp * 64 + unit * 8;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int col = min(grp * 64 + (u >> 1) * 32 + (c >> 2) * 8 + (u & 1) * 4 + (c & 3), p.n - 1);
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int r = NT == 1 ? (g & 1) * 8 : 32 * j + 8 * g;
        v.b[u][j] = *(const u4*)(bw + (int64_t)col * p.r + (r < p.r ? r : 0));
      }
    }
#pragma unroll
    for (int t = 0; t < kHalves; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (t == 0 || two) v.y[t][i] = stream_load(from[t][i] + (n < p.n ? n : 0));
  };
  // the waves' own parts of the sums below; before them, where h is kept, its 32-bit values
  __shared__ __attribute__((aligned(16))) float sums[4][16 * 68];
  static_assert(kTileRows * (kR + 1) <= 4 * 16 * 68, "h takes the sums' place");
  const bool keep = packs.col != nullptr && column_part == 0;
  // rank 16: both parts in one instruction, the second in the reduction's upper half
  u4 hv[kHalves][kJ], lv[kHalves][kJ];
  float back[kHalves];
  __shared__ __attribute__((aligned(16))) uint16_t part[2][kTileRows][kPitch];
  __shared__ int back_s[kTileRows];
  const float scale = p.scaling[ad] * p.keep_scale;
  const float* planes = reinterpret_cast<const float*>(p.ws);
  for (int i = threadIdx.x; i < kTileRows * NT * 4; i += kThreads) {
    const int at = i / (NT * 4), q = i % (NT * 4) * 4;
    f4 v = {};
    if (q < p.r && order[at] >= 0)
      v = sum_planes(planes + ((int64_t)tile * kTileRows + at) * p.r + q, p.l.positions * p.r, splits) * scale;
    if (keep) {
#pragma unroll
      for (int e = 0; e < 4; ++e) (&sums[0][0])[at * (kR + 1) + q + e] = v[e];
    }
    if constexpr (!BF) {
      float m = fmaxf(fmaxf(finite_magnitude(v[0]), finite_magnitude(v[1])), fmaxf(finite_magnitude(v[2]), finite_magnitude(v[3])));
#pragma unroll
      for (int o = 1; o < NT * 4; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
      const int e = range_exponent<BF>(m);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = times_pow2(v[j], e);
      if (q == 0) back_s[at] = -e;
    }
    uint2 hi, lo;
    split16<BF>(v[0], v[1], hi.x, lo.x);
    split16<BF>(v[2], v[3], hi.y, lo.y);
    *(uint2*)&part[0][at][q] = hi;
    *(uint2*)&part[1][at][q] = lo;
  }
  __syncthreads();
  if (keep) {
    pack_columns<BF, kR>(&sums[0][0], packs, (int64_t)tile * kTileRows, p.l.positions, kThreads);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < kHalves; ++t) {
    if constexpr (!BF) back[t] = pow2(back_s[t * 16 + c]);
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int r = NT == 1 ? (g & 1) * 8 : 32 * j + 8 * g;
      hv[t][j] = *(const u4*)&part[NT == 1 ? g >> 1 : 0][t * 16 + c][r];
      if constexpr (NT > 1) lv[t][j] = *(const u4*)&part[1][t * 16 + c][r];
    }
  }
  float* const own = sums[wave];
  for (int grp = g0 + wave; grp < g1; grp += 4) {
    Group v;
    load(grp, v);
    __builtin_amdgcn_sched_barrier(0);
    const bool in = grp * 64 + unit * 8 < p.n;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        if ((NT == 1 ? (g & 1) * 8 : 32 * j + 8 * g) >= p.r) v.b[u][j] = u4{};
#pragma unroll
    for (int t = 0; t < kHalves; ++t) {
      if (t > 0 && !two) break;
      f4 acc[4] = {};
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          acc[u] = mfma16_of<BF>(v.b[u][j], hv[t][j], acc[u]);
          if constexpr (NT > 1) acc[u] = mfma16_of<BF>(v.b[u][j], lv[t][j], acc[u]);
        }
      if (nan_among(acc)) {  // an infinite B, or h
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          acc[u] = f4{};
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            const u4 b = finite_only<BF>(v.b[u][j]);
            acc[u] = mfma16_of<BF>(NT == 1 && g >= 2 ? b : v.b[u][j], hv[t][j], acc[u]);
            if constexpr (NT > 1) acc[u] = mfma16_of<BF>(b, lv[t][j], acc[u]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if constexpr (!BF) acc[u] *= back[t];
        *(f4*)(own + c * 68 + (4 * (u >> 1) + g) * 8 + (u & 1) * 4) = acc[u];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* at = own + (8 * i + (lane >> 3)) * 68 + unit * 8;
        const f4 lo = *(const f4*)at, hi = *(const f4*)(at + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f4& d = e < 2 ? lo : hi;
          const uint32_t y = v.y[t][i][e];
          v.y[t][i][e] = pack16<BF>(unpack16<BF>(y, 0) + d[(e & 1) * 2], unpack16<BF>(y, 1) + d[(e & 1) * 2 + 1]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int to = row[t][i];
        asm volatile("" : "+v"(to));  // (addresses kept over the groups took 8 registers)
        if (in && to >= 0) *(u4*)(p.out + to * p.ldo + grp * 64 + unit * 8) = v.y[t][i];
      }
    }
  }
}

// y = x of the kept elements times keep_scale: eight elements a thread, one counter.  9001 rows of 4096 (bf16)
// 27.2 us for 147 MB, 5.4 TB/s; the counter's ten rounds take 54 % of the vector units' time and hide
// behind the loads.
template <bool BF, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(int rows, int cols, const uint16_t* __restrict__ x, int64_t ldx, uint16_t* __restrict__ y, int64_t ldy, int drop,
               float keep_scale, const int64_t* __restrict__ seed) {
  const int units = (cols + 7) / 8;
  const Philox philox(seed);
  const int64_t items = (int64_t)rows * units;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < items; i += (int64_t)gridDim.x * kThreads) {
    const int row = (int)(i / units), unit = (int)(i - (int64_t)row * units);
    const uint16_t* xr = x + row * ldx + unit * 8;
    uint16_t* yr = y + row * ldy + unit * 8;
    const u4 m = philox.mask(unit, row, drop);
    const int n = min(8, cols - unit * 8);
    u4 v = {};
    if constexpr (VEC) {
      v = stream_load(xr);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) v[e >> 1] |= (uint32_t)xr[e] << (16 * (e & 1));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = pack16<BF>(unpack16<BF>(v[e], 0) * keep_scale, unpack16<BF>(v[e], 1) * keep_scale) & m[e];
    if constexpr (VEC) {
      *(u4*)yr = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) yr[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <bool BF, int NT>
void shrink_of(const ShrinkArgs& a, int splits, hipStream_t stream) {
  const unsigned grid = (unsigned)a.l.tiles * splits;
  if (a.drop) shrink_kernel<BF, NT, true><<<grid, kThreads, 0, stream>>>(a, splits);
  else shrink_kernel<BF, NT, false><<<grid, kThreads, 0, stream>>>(a, splits);
}
template <bool BF>
void shrink_rank(const ShrinkArgs& a, int splits, hipStream_t stream) {
  if (a.r <= 16) shrink_of<BF, 1>(a, splits, stream);
  else if (a.r <= 32) shrink_of<BF, 2>(a, splits, stream);
  else if (a.r <= 64) shrink_of<BF, 4>(a, splits, stream);
  else shrink_of<BF, 8>(a, splits, stream);
}

template <bool BF, int NT>
void expand_of(const AdapterArgs& a, int splits, const AdapterPacks& packs, hipStream_t stream) {
  const int groups = (a.n + 63) / 64;
  // About four workgroups per CU (of 256) of four waves each, by the bound of tiles (adapter_splits()).  Half as
  // many: 10175 rows against rank 16 76 us for 40; twice as many 39.6, but each sums the planes anew.
  const int wide = std::max(1, std::min((groups + 3) / 4, 1024 / a.l.tiles));
  expand_kernel<BF, NT><<<(unsigned)a.l.tiles * wide, kThreads, 0, stream>>>(a, splits, packs, wide);
}
template <bool BF>
void expand_rank(const AdapterArgs& a, int splits, const AdapterPacks& packs, hipStream_t stream) {
  if (a.r <= 16) expand_of<BF, 1>(a, splits, packs, stream);
  else if (a.r <= 32) expand_of<BF, 2>(a, splits, packs, stream);
  else if (a.r <= 64) expand_of<BF, 4>(a, splits, packs, stream);
  else expand_of<BF, 8>(a, splits, packs, stream);
}

}  // namespace

int adapter_splits(const AdapterLayout& l, int width, int cus) {
  // About four workgroups per CU, parts of at least 64 values per wave, up to 16 planes.  Up to 8: 1 row of
  // 11008 by rank 16 7.1 us for 6.75 (both products), 2048 rows by rank 64 40.0 for 41.9; up to 4: 8.1 and 40.4.
  // The bound of tiles counts one more for each adapter of the bank: in a bank of many hundred, of which few are
  // used, there are fewer workgroups (1024 rows of 3 adapters 11.7 us in a bank of 8, 18 in one of 256, 40 in 1024).
  const int want = (4 * cus + l.tiles - 1) / l.tiles;
  return std::max(1, std::min({want, width / 256, kMaxSplits}));
}

hipError_t launch_adapter_plan(const AdapterLayout& l, int rows, int adapters, const int32_t* index, int32_t* plan,
                               hipStream_t stream) {
  const size_t smem = sizeof(int) * ((kPlanWaves + 4) * (size_t)(adapters + 1) + 3 + kPlanWaves);
  plan_kernel<<<1, kPlanThreads, smem, stream>>>(l, rows, adapters, index, plan);
  return hipGetLastError();
}

hipError_t launch_shrink(bool bf16, const ShrinkArgs& a, int splits, hipStream_t stream) {
  bf16 ? shrink_rank<true>(a, splits, stream) : shrink_rank<false>(a, splits, stream);
  return hipGetLastError();
}

hipError_t launch_join(const AdapterArgs& a, const float* planes, int splits, const AdapterPacks& p, hipStream_t stream) {
  const unsigned grid = (unsigned)(a.l.positions / 32);
  auto go = [&](auto kernel) { kernel<<<grid, kJoinThreads, 0, stream>>>(a, planes, splits, p); };
  switch (padded_rank(a.r)) {
    case 16: a.bf16 ? go(&join_kernel<true, 1>) : go(&join_kernel<false, 1>); break;
    case 32: a.bf16 ? go(&join_kernel<true, 2>) : go(&join_kernel<false, 2>); break;
    case 64: a.bf16 ? go(&join_kernel<true, 4>) : go(&join_kernel<false, 4>); break;
    default: a.bf16 ? go(&join_kernel<true, 8>) : go(&join_kernel<false, 8>);
  }
  return hipGetLastError();
}

hipError_t launch_adapters(const AdapterArgs& a, const ForwardWs& w, hipStream_t stream) {
  float* const planes = reinterpret_cast<float*>(a.ws);
  const ShrinkArgs s = {a.l, a.plan, a.x, a.ldx, a.a, a.k, a.r, a.adapters, a.drop, a.seed, planes};
  hipError_t e = launch_shrink(a.bf16, s, w.splits, stream);
  if (e != hipSuccess) return e;
  AdapterPacks packs = {};
  if (a.h != nullptr) place_col(packs, a.l, a.r, a.h);
  a.bf16 ? expand_rank<true>(a, w.splits, packs, stream) : expand_rank<false>(a, w.splits, packs, stream);
  return hipGetLastError();
}

hipError_t launch_dropout(bool bf16, int rows, int cols, const uint16_t* x, int64_t ldx, uint16_t* y, int64_t ldy, int drop,
                          float keep_scale, const int64_t* seed, hipStream_t stream) {
  const int64_t items = (int64_t)rows * ((cols + 7) / 8);
  const unsigned grid = (unsigned)std::min<int64_t>((items + kThreads - 1) / kThreads, 8192);
  const bool vec = cols % 8 == 0 && ldx % 8 == 0 && ldy % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(y) % 16 == 0;
  auto kernel = bf16 ? (vec ? &dropout_kernel<true, true> : &dropout_kernel<true, false>)
                     : (vec ? &dropout_kernel<false, true> : &dropout_kernel<false, false>);
  kernel<<<grid, kThreads, 0, stream>>>(rows, cols, x, ldx, y, ldy, drop, keep_scale, seed);
  return hipGetLastError();
}

}  // namespace dw4
