// Low-rank adapters of many requests beside a shared projection:
//   out_t = base_t + s_a B_a A_a d(x_t),   a = the row's adapter (or none),
// with d dropout whose mask comes from a counter; and that dropout by itself.
//
// Rows are sorted by adapter once per batch (plan_kernel), so that a tile of 16 or 64
// positions has one adapter and both its products run on 16 x 16 x 32 matrix
// instructions, rows as their columns.  Two launches: the rows' products with A, in
// parts of k over workgroups and waves (fp32 planes, joined in order), then the
// products with B added to the projection's output, rounded once.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "w4a16_adapters_device.h"

namespace dw4 {

namespace {

constexpr int kThreads = 256;
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
// first tiles and chunks by a scan, then each row to its place, in order within its adapter.
__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(AdapterLayout l, int rows, int adapters, const int32_t* __restrict__ index, int32_t* __restrict__ plan) {
  extern __shared__ int sm[];
  const int segs = adapters + 1;  // the last: rows without an adapter
  int* const count = sm;                         // [waves][segs], later each wave's next position
  int* const total = count + kPlanWaves * segs;  // [segs]
  int* const tile0 = total + segs;               // [segs + 1]
  int* const chunk0 = tile0 + segs + 1;          // [segs + 1]
  int* const wave_sum = chunk0 + segs + 1;
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
    tile0[s] = (n + l.align - 1) / l.align;
    chunk0[s] = (n + l.chunk_rows - 1) / l.chunk_rows;
  }
  __syncthreads();
  scan_ints(tile0, segs, wave_sum);
  scan_ints(chunk0, segs, wave_sum);
  for (int s = t; s < segs; s += kPlanThreads) {
    int at = tile0[s] * l.align;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int n = count[w * segs + s];
      count[w * segs + s] = at;
      at += n;
    }
  }
  for (int s = t; s <= segs; s += kPlanThreads) plan[l.chunk_start + s] = chunk0[s];
  for (int i = t; i < l.tiles; i += kPlanThreads)
    plan[l.tile_adapter + i] = i < tile0[segs] ? segment_of(tile0, segs, i) : -1;
  for (int i = t; i < l.chunks; i += kPlanThreads) {
    int4 c = make_int4(-1, 0, 0, 0);  // adapter, first position, rows, none
    if (i < chunk0[segs]) {
      const int s = segment_of(chunk0, segs, i), at = (i - chunk0[s]) * l.chunk_rows;
      c = make_int4(s, tile0[s] * l.align + at, min(l.chunk_rows, total[s] - at), 0);
    }
    *(int4*)(plan + l.chunk + 4 * i) = c;
  }
  for (int i = t; i < l.positions; i += kPlanThreads) {  // positions without a row
    const int tile = i / l.align;
    const int s = tile < tile0[segs] ? segment_of(tile0, segs, tile) : -1;
    if (s < 0 || i - tile0[s] * l.align >= total[s]) plan[l.order + i] = -1;
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

// Rows' products with A: tile blockIdx.x's RT * 16 positions, part blockIdx.y of k, of
// which each wave takes a part of its own.
template <bool BF, int RT, int NT, bool DROP>
__global__ void __launch_bounds__(kThreads) shrink_kernel(AdapterArgs p, int splits) {
  __shared__ __attribute__((aligned(16))) float red[4][RT * 16][20];
  const int tile = blockIdx.x;
  const int ad = p.plan[p.l.tile_adapter + tile];
  if (ad < 0 || ad >= p.adapters) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int32_t* order = p.plan + p.l.order + (int64_t)tile * (RT * 16);
  const uint16_t* xr[RT];
  int row[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    row[t] = max(order[t * 16 + c], 0);
    xr[t] = p.x + row[t] * p.ldx;
  }
  const uint16_t* ar[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) ar[t] = p.a + ((int64_t)ad * p.r + min(t * 16 + c, p.r - 1)) * p.k;
  f4 acc[RT][NT] = {};
  const Philox philox(DROP ? p.seed : reinterpret_cast<const int64_t*>(p.plan));
  const int steps = (p.k + 31) / 32, parts = splits * 4, part = blockIdx.y * 4 + wave;
  const int s0 = (int)((int64_t)steps * part / parts), s1 = (int)((int64_t)steps * (part + 1) / parts);
  for (int s = s0; s < s1; ++s) {
    const int k = s * 32 + 8 * g, kc = k < p.k ? k : 0;
    u4 xv[RT], av[NT];
#pragma unroll
    for (int t = 0; t < RT; ++t) xv[t] = *(const u4*)(xr[t] + kc);
#pragma unroll
    for (int t = 0; t < NT; ++t) av[t] = *(const u4*)(ar[t] + kc);
    if (s * 32 + 32 > p.k) {
#pragma unroll
      for (int t = 0; t < RT; ++t) xv[t] = k < p.k ? xv[t] : u4{};
#pragma unroll
      for (int t = 0; t < NT; ++t) av[t] = k < p.k ? av[t] : u4{};
    }
    if constexpr (DROP) {
#pragma unroll
      for (int t = 0; t < RT; ++t) xv[t] &= philox.mask(k >> 3, row[t], p.drop);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) acc[t][u] = mfma16_of<BF>(av[u], xv[t], acc[t][u]);
  }
  float* plane = p.ws + ((int64_t)blockIdx.y * p.l.positions + (int64_t)tile * (RT * 16)) * p.r;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    if (u) __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t) *(f4*)&red[wave][t * 16 + c][4 * g] = acc[t][u];
    __syncthreads();
    const int i = threadIdx.x >> 2, q = (threadIdx.x & 3) * 4;
    if (i < RT * 16 && u * 16 + q < p.r) {
      f4 v = *(const f4*)&red[0][i][q];
#pragma unroll
      for (int w = 1; w < 4; ++w) v += *(const f4*)&red[w][i][q];
      if (order[i] < 0) v = f4{};
      *(f4*)(plane + (int64_t)i * p.r + u * 16 + q) = v;
    }
  }
}

// The products with B, added to the projection's output: tile blockIdx.x, part
// blockIdx.y of the columns.
template <bool BF, int RT, int NT>
__global__ void __launch_bounds__(kThreads) expand_kernel(AdapterArgs p, int splits) {
  constexpr int kRows = RT * 16, kPitch = NT * 16 + 8, kJ = NT == 1 ? 1 : NT / 2;
  __shared__ __attribute__((aligned(16))) uint16_t part[2][kRows][kPitch];
  __shared__ int back[kRows];
  const int tile = blockIdx.x;
  const int ad = p.plan[p.l.tile_adapter + tile];
  if (ad < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int32_t* order = p.plan + p.l.order + (int64_t)tile * kRows;
  const int groups = (p.n + 31) / 32;
  const int g0 = (int)((int64_t)groups * blockIdx.y / gridDim.y), g1 = (int)((int64_t)groups * (blockIdx.y + 1) / gridDim.y);
  if (ad >= p.adapters) {  // rows without an adapter keep the projection's output
    if (p.out == p.base) return;
    const int units = min(g1 * 4, p.n / 8) - g0 * 4;
    for (int i = 0; i < kRows; ++i) {
      const int row = order[i];
      if (row < 0) break;
      for (int u = threadIdx.x; u < units; u += kThreads)
        *(u4*)(p.out + row * p.ldo + (g0 * 4 + u) * 8) = *(const u4*)(p.base + row * p.ldb + (g0 * 4 + u) * 8);
    }
    return;
  }
  const float scale = p.scaling[ad] * p.keep_scale;
  for (int i = threadIdx.x; i < kRows * NT * 4; i += kThreads) {
    const int at = i / (NT * 4), q = i % (NT * 4) * 4;
    f4 v = {};
    if (q < p.r) {
      const int64_t pos = ((int64_t)tile * kRows + at) * p.r + q;
      for (int s = 0; s < splits; ++s) v += *(const f4*)(p.ws + (int64_t)s * p.l.positions * p.r + pos);
      if (p.h != nullptr && blockIdx.y == 0) *(f4*)(p.h + pos) = v;
      v *= scale;
    }
    int e = 0;
    if constexpr (!BF) {
      float m = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
      for (int o = 1; o < NT * 4; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
      e = range_exponent<BF>(m);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = times_pow2(v[j], e);
    }
    if (q == 0) back[at] = -e;
    uint2 hi, lo;
    split16<BF>(v[0], v[1], hi.x, lo.x);
    split16<BF>(v[2], v[3], hi.y, lo.y);
    *(uint2*)&part[0][at][q] = hi;
    *(uint2*)&part[1][at][q] = lo;
  }
  __syncthreads();
  // rank 16: both parts in one instruction, the second in the reduction's upper half
  u4 hv[RT][kJ], lv[RT][kJ];
  int row[RT], scale_back[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    row[t] = order[t * 16 + c];
    scale_back[t] = back[t * 16 + c];
    if constexpr (NT == 1) {
      hv[t][0] = *(const u4*)&part[g >> 1][t * 16 + c][(g & 1) * 8];
    } else {
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        hv[t][j] = *(const u4*)&part[0][t * 16 + c][32 * j + 8 * g];
        lv[t][j] = *(const u4*)&part[1][t * 16 + c][32 * j + 8 * g];
      }
    }
  }
  for (int grp = g0 + wave; grp < g1; grp += 4) {
    const int n = grp * 32 + 8 * g;  // the lane's eight output columns
    const bool in = n < p.n;
    u4 y[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) y[t] = *(const u4*)(p.base + max(row[t], 0) * p.ldb + (in ? n : 0));
    f4 acc[RT][2] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int col = min(grp * 32 + (c >> 2) * 8 + u * 4 + (c & 3), p.n - 1);
      const uint16_t* br = p.b + ((int64_t)ad * p.n + col) * p.r;
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int r = NT == 1 ? (g & 1) * 8 : 32 * j + 8 * g;
        u4 bv = *(const u4*)(br + (r < p.r ? r : 0));
        if (r >= p.r) bv = u4{};
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          acc[t][u] = mfma16_of<BF>(bv, hv[t][j], acc[t][u]);
          if constexpr (NT > 1) acc[t][u] = mfma16_of<BF>(bv, lv[t][j], acc[t][u]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      u4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float d = acc[t][e >> 1][(e & 1) * 2 + j];
          v[j] = unpack16<BF>(y[t][e], j) + (BF ? d : times_pow2(d, scale_back[t]));
        }
        o[e] = pack16<BF>(v[0], v[1]);
      }
      if (in && row[t] >= 0) *(u4*)(p.out + row[t] * p.ldo + n) = o;
    }
  }
}

// y = x of the kept elements times keep_scale: eight elements a thread.
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
      v = *(const u4*)xr;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) v[e >> 1] |= (uint32_t)xr[e] << (16 * (e & 1));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = pack16<BF>(unpack16<BF>(v[e], 0) * keep_scale, unpack16<BF>(v[e], 1) * keep_scale) & m[e];
    if constexpr (VEC) {
      *(u4*)yr = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) yr[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <bool BF, int RT, int NT>
void launch_forward(const AdapterArgs& a, int splits, hipStream_t stream) {
  const dim3 grid(a.l.tiles, splits);
  if (a.drop) shrink_kernel<BF, RT, NT, true><<<grid, kThreads, 0, stream>>>(a, splits);
  else shrink_kernel<BF, RT, NT, false><<<grid, kThreads, 0, stream>>>(a, splits);
  const int groups = (a.n + 31) / 32;
  const int wide = std::max(1, std::min((groups + 3) / 4, 1024 / a.l.tiles));
  expand_kernel<BF, RT, NT><<<dim3(a.l.tiles, wide), kThreads, 0, stream>>>(a, splits);
}
template <bool BF, int RT>
void launch_rank(const AdapterArgs& a, int splits, hipStream_t stream) {
  if (a.r <= 16) launch_forward<BF, RT, 1>(a, splits, stream);
  else if (a.r <= 32) launch_forward<BF, RT, 2>(a, splits, stream);
  else if (a.r <= 64) launch_forward<BF, RT, 4>(a, splits, stream);
  else launch_forward<BF, RT, 8>(a, splits, stream);
}

}  // namespace

int adapter_splits(const AdapterLayout& l, int k, int cus) {
  // about three workgroups per CU, parts of at least 64 values of k per wave
  const int want = (3 * cus + l.tiles - 1) / l.tiles;
  return std::max(1, std::min({want, k / 256, 32}));
}

hipError_t launch_adapter_plan(const AdapterLayout& l, int rows, int adapters, const int32_t* index, int32_t* plan,
                               hipStream_t stream) {
  const size_t smem = sizeof(int) * ((kPlanWaves + 3) * (size_t)(adapters + 1) + 2 + kPlanWaves);
  plan_kernel<<<1, kPlanThreads, smem, stream>>>(l, rows, adapters, index, plan);
  return hipGetLastError();
}

hipError_t launch_adapters(const AdapterArgs& a, int splits, hipStream_t stream) {
  if (a.l.align == 16) a.bf16 ? launch_rank<true, 1>(a, splits, stream) : launch_rank<false, 1>(a, splits, stream);
  else a.bf16 ? launch_rank<true, 4>(a, splits, stream) : launch_rank<false, 4>(a, splits, stream);
  return hipGetLastError();
}

hipError_t launch_dropout(bool bf16, int rows, int cols, const uint16_t* x, int64_t ldx, uint16_t* y, int64_t ldy, int drop,
                          float keep_scale, const int64_t* seed, hipStream_t stream) {
  const int64_t items = (int64_t)rows * ((cols + 7) / 8);
  const unsigned grid = (unsigned)std::min<int64_t>((items + kThreads - 1) / kThreads, 1 << 16);
  const bool vec = cols % 8 == 0 && ldx % 8 == 0 && ldy % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(y) % 16 == 0;
  auto kernel = bf16 ? (vec ? &dropout_kernel<true, true> : &dropout_kernel<true, false>)
                     : (vec ? &dropout_kernel<false, true> : &dropout_kernel<false, false>);
  kernel<<<grid, kThreads, 0, stream>>>(rows, cols, x, ldx, y, ldy, drop, keep_scale, seed);
  return hipGetLastError();
}

}  // namespace dw4
