// Gradients of the low-rank adapters (w4a16_adapters.hip): with g_t the output's gradient,
// h_t = s_a A_a d(x_t) and dh_t = s_a B_a^T g_t,
//   dx_t = d'(A_a^T dh_t),  dA_a = sum of dh_t d(x_t)^T,  dB_a = sum of g_t h_t^T.
//
// Five launches.  The weights are turned around, so that dh is the forward's first product
// over g and B; beside that, in the same launch, g h^T, which needs neither.  Then dh, and dh x^T
// with dx.  The sums over rows (outer()) come from tiles of 32 rows by 64 columns turned around by
// way of LDS (rows as the matrix instruction's reduction), a chunk of 512 rows of one adapter per
// workgroup; dx comes from the same tile of x and its dropout mask.  The chunks' shares of
// dA and dB are added up in order: no float atomics.
//
// Bound by memory: x, g and dx pass once, g a second time on its way to dh, with two to four waves a SIMD at ranks up
// to 32 and two at 64; rank 64 with dropout, and 128 with dx, hold operands and sums of the whole rank in one
// wave's registers.  Chunks of 256 rows took longer
// for their shares, chunks of 1024 left CUs idle; workgroups of eight waves were slower than of four.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "w4a16_adapters_device.h"

namespace dw4 {

namespace {

constexpr int kThreads = 256, kOuterThreads = 256, kOuterWaves = kOuterThreads / 64;
constexpr int kStep = 32;    // rows a step
constexpr int kTurn = 72;    // halfs per row of a wave's tile of 64 columns in LDS

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4 lds_s4;

// The A operand of a tile [32 rows][64 columns] in LDS turned around: column
// 16 ct + lane % 16, rows 8 (lane / 16) .. + 7, by two transposing reads.  Lane l of 16
// gives the address of four columns of row l / 4 and receives column l of the four rows.
__device__ __forceinline__ u4 turned(const uint16_t* tile, int ct) {
  const int lane = threadIdx.x & 63;
  const uint16_t* at = tile + (8 * (lane >> 4) + ((lane >> 2) & 3)) * kTurn + ct * 16 + 4 * (lane & 3);
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 4 * kTurn));
  return __builtin_bit_cast(u4, (s8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// out[c][r] = in[r][c], 16-bit: 64 x 64 at a time.
__device__ __forceinline__ void turn_tile(const uint16_t* in, uint16_t* out, int rows, int cols, int r0, int c0,
                                          uint16_t* tile) {
  constexpr int kPitch = 66, kRows = kOuterThreads / 32;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 64 / kRows; ++i) {
    const int r = r0 + y + kRows * i, c = c0 + 2 * x;
    if (r < rows && c < cols)
      *(uint32_t*)(tile + (y + kRows * i) * kPitch + 2 * x) = *(const uint32_t*)(in + (int64_t)r * cols + c);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 64 / kRows; ++i) {
    const int c = c0 + y + kRows * i, r = r0 + 2 * x;
    if (c < cols && r < rows)
      *(uint32_t*)(out + (int64_t)c * rows + r) = (uint32_t)tile[2 * x * kPitch + y + kRows * i] |
                                                  (uint32_t)tile[(2 * x + 1) * kPitch + y + kRows * i] << 16;
  }
}

struct OuterArgs {
  const uint16_t* in;    // [rows][width]
  int64_t ld;
  int width;
  AdapterPacks packs;
  float* share;          // [shares][r * width], or null: no such gradient
  uint16_t* grad;        // [adapters][r * width], with share
  const uint16_t* at;    // DX: [adapters][width][r]
};
constexpr int kOuterLds = sizeof(uint16_t) * kOuterWaves * kStep * kTurn;
constexpr int kSumPitch = 68;
static_assert(sizeof(float) * kOuterWaves * 16 * kSumPitch <= kOuterLds, "the waves' sums take the tiles' place");

// A chunk's rows of in, columns k0 .. k0 + 63, of which each wave takes every fourth step of 32 rows: the
// chunk's share of sum of in_t h_t^T (COLS: stored [width][r], else [r][width]), which is the gradient
// itself where the adapter has no other chunk, and with DX dx of the same places.
template <bool BF, int NT, bool DX, bool DROP, bool COLS>
__device__ __forceinline__ void outer(const AdapterArgs& p, const OuterArgs& o, int chunk_index, int k0, unsigned char* lds) {
  constexpr int kR = NT * 16, kJ = NT == 1 ? 1 : NT / 2;
  const int4 chunk = *(const int4*)(p.plan + p.l.chunk + 4 * chunk_index);
  const int ad = chunk.x;
  if (ad < 0) return;
  const int lane = threadIdx.x & 63, wave = wave_index(), g = lane >> 4, c = lane & 15;
  const int32_t* order = p.plan + p.l.order + chunk.y;
  if (ad >= p.adapters) {  // rows without an adapter
    if (!DX) return;
    const int units = min(64, o.width - k0) / 8;
    for (int i = threadIdx.x; i < chunk.z * units; i += kOuterThreads)
      *(u4*)(p.dx + order[i / units] * p.lddx + k0 + i % units * 8) = u4{};
    return;
  }
  uint16_t* const tile = reinterpret_cast<uint16_t*>(lds) + wave * (kStep * kTurn);
  // rows as loads and stores take them (to_operands()), -1 behind the chunk and the width
  const int unit = lane & 7, line = lane >> 3, k = k0 + unit * 8;
  __shared__ u4 lines[4][128];
  int row[2][2], row2[2][2], row3[2][2];  // this step's, the next two's
  auto rows_of = [&](int first, int (&r)[2][2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = first + t * 16 + 8 * i + line;
        r[t][i] = order[at < chunk.z ? at : 0];
        if (at >= chunk.z || k >= o.width) r[t][i] = -1;
      }
  };
  // A turned around: the operand's row is a column of x, eight values of r
  u4 at[2][2][DX ? kJ : 1];
  if constexpr (DX) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int col = k0 + 32 * q + (c >> 2) * 8 + u * 4 + (c & 3);
          const int r = NT == 1 ? (g & 1) * 8 : 32 * j + 8 * g;
          const bool in = col < o.width && r < p.r;
          at[q][u][j] = *(const u4*)(o.at + (in ? ((int64_t)ad * o.width + col) * p.r + r : 0));
          if (!in) at[q][u][j] = u4{};
        }
  }
  bool odd_a = false;  // whether A has values that are not finite
  if constexpr (DX) {
    uint32_t bits = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < kJ; ++j) add_nonfinite<BF>(at[q][u][j], bits);
    odd_a = __ballot((bits & 0x80008000u) != 0) != 0;
  }
  const Philox philox(DROP ? p.seed : reinterpret_cast<const int64_t*>(p.plan));
  const int64_t half = p.l.positions * kR;
  f4 acc[4][NT] = {};
  auto load = [&](const int (&r)[2][2], u4 (&x)[2][2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) x[t][i] = stream_load(o.in + (r[t][i] >= 0 ? r[t][i] * o.ld + k : 0));
  };
  constexpr int kStride = kOuterWaves * kStep;
  u4 x[2][2], x2[2][2];
  rows_of(wave * kStep, row);
  rows_of(wave * kStep + kStride, row2);
  load(row, x);
  for (int first = wave * kStep; first < chunk.z; first += kStride) {
    // h (or dh) first, the next step's rows last: loads return in order, and a wait for the former
    // then leaves the latter in flight
    const int64_t pos = chunk.y + first;
    u4 hi[NT], lo[NT], rhi[2][DX ? kJ : 1], rlo[2][DX ? kJ : 1];
    int col_exp[NT], row_exp[2];
    if (o.share != nullptr) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const uint16_t* from = o.packs.col + (pos + 8 * g) * kR + (u * 16 + c) * 8;
        hi[u] = *(const u4*)from;
        lo[u] = *(const u4*)(from + half);
        if constexpr (!BF) col_exp[u] = o.packs.col_exp[pos / 32 * kR + u * 16 + c];
      }
    }
    if constexpr (DX) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint16_t* from = o.packs.row + (pos + t * 16 + c) * kR;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          rhi[t][j] = *(const u4*)(from + (NT == 1 ? (g >> 1) * half + (g & 1) * 8 : 32 * j + 8 * g));
          if constexpr (NT > 1) rlo[t][j] = *(const u4*)(from + 32 * j + 8 * g + half);
        }
        if constexpr (!BF) row_exp[t] = o.packs.row_exp[pos + t * 16 + c];
      }
    }
    rows_of(first + 2 * kStride, row3);
    load(row2, x2);
    if constexpr (NT < 8) __builtin_amdgcn_sched_barrier(0);  // (else the loads sink to where they are used)
    u4 keep[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (DROP) {
          keep[t][i] = philox.mask(k >> 3, row[t][i], p.drop);
          x[t][i] &= keep[t][i];
        }
        if (row[t][i] < 0) x[t][i] = u4{};
        *(u4*)(tile + (t * 16 + 8 * i + line) * kTurn + unit * 8) = x[t][i];
      }
    if constexpr (DX) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f4 d[2][2] = {};
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int u = 0; u < 2; ++u) d[q][u] = mfma16_of<BF>(at[q][u][j], rhi[t][j], d[q][u]);
          if constexpr (NT > 1) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int u = 0; u < 2; ++u) d[q][u] = mfma16_of<BF>(at[q][u][j], rlo[t][j], d[q][u]);
          }
        }
        const float back = BF ? 1.f : pow2(row_exp[t]);
        u4 w[2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a = d[q][i >> 1][(i & 1) * 2], b = d[q][i >> 1][(i & 1) * 2 + 1];
            if constexpr (!BF) {
              a *= back;
              b *= back;
            }
            w[q][i] = pack16<BF>(a, b);
          }
        from_operands(w[0], w[1], lines[wave]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (DROP) w[i] &= keep[t][i];
          if (row[t][i] >= 0) *(u4*)(p.dx + row[t][i] * p.lddx + k) = w[i];
        }
      }
    }
    if (o.share != nullptr) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      u4 xt[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) xt[t] = turned(tile, t);
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        if constexpr (BF) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            acc[t][u] = mfma16_of<BF>(xt[t], hi[u], acc[t][u]);
            acc[t][u] = mfma16_of<BF>(xt[t], lo[u], acc[t][u]);
          }
        } else {
          const float back = pow2(col_exp[u]);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            f4 d = mfma16_of<BF>(xt[t], hi[u], f4{});
            d = mfma16_of<BF>(xt[t], lo[u], d);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][u][i] = fmaf(d[i], back, acc[t][u][i]);
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row[t][i] = row2[t][i];
        row2[t][i] = row3[t][i];
        x[t][i] = x2[t][i];
      }
  }
  // Infinities (finite_only()): a sum that is NaN may be so by its second parts alone.  It is formed once more, by
  // itself, from the first parts, beside which nothing finite counts.  dx: where A holds some, by the lanes that
  // stored it.
  if constexpr (DX) {
    if (odd_a) {
      asm volatile("" ::: "memory");  // what the lane has stored is written over as another type
#pragma unroll 1
      for (int i = 0; wave * kStep + i / 4 * kStride < chunk.z; ++i) {
        const int from = wave * kStep + i / 4 * kStride + i % 4 * 8 + line;
        if (from >= chunk.z) continue;
        const int to = order[from];
        const uint16_t* dh = o.packs.row + (int64_t)(chunk.y + from) * kR;
        const u4 kept = DROP ? philox.mask(k >> 3, to, p.drop) : ~u4{};
#pragma unroll 1
        for (int e = 0; e < 8 && k + e < o.width; ++e) {
          const uint16_t* a = o.at + ((int64_t)ad * o.width + k + e) * p.r;
          float s = 0.f;
          for (int r = 0; r < p.r; ++r) s += unpack16<BF>(a[r], 0) * unpack16<BF>(dh[r], 0);
          if (!isfinite(s) && (kept[e >> 1] >> (16 * (e & 1)) & 1)) p.dx[to * p.lddx + k + e] = (uint16_t)pack16<BF>(s, 0.f);
        }
      }
    }
  }
  if (o.share == nullptr) return;
  // the waves' sums, 16 columns of h at a time
  float* const sums = reinterpret_cast<float*>(lds);  // [waves][16][kSumPitch]
  const bool alone = chunk.w < 0;
  float* share = o.share + (int64_t)max(chunk.w, 0) * o.width * p.r;
  uint16_t* grad = o.grad + (int64_t)ad * o.width * p.r;
  auto store = [&](int64_t at, f4 v) {
    if (alone) *(uint2*)(grad + at) = make_uint2(pack16<BF>(v[0], v[1]), pack16<BF>(v[2], v[3]));
    else *(f4*)(share + at) = v;
  };
  bool odd = false;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 4; ++t) *(f4*)(sums + (wave * 16 + c) * kSumPitch + t * 16 + 4 * g) = acc[t][u];
    __syncthreads();
    f4 v = {};
    if constexpr (COLS) {
      const int col = threadIdx.x >> 2, r = (threadIdx.x & 3) * 4;
#pragma unroll
      for (int w = 0; w < kOuterWaves; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += sums[(w * 16 + r + e) * kSumPitch + col];
      if (k0 + col < o.width && u * 16 + r < p.r) {
        odd = odd || isnan(v[0] + v[1] + v[2] + v[3]);
        store((int64_t)(k0 + col) * p.r + u * 16 + r, v);
      }
    } else {
      const int r = threadIdx.x >> 4, col = (threadIdx.x & 15) * 4;
#pragma unroll
      for (int w = 0; w < kOuterWaves; ++w) v += *(const f4*)(sums + (w * 16 + r) * kSumPitch + col);
      if (k0 + col < o.width && u * 16 + r < p.r) {
        odd = odd || isnan(v[0] + v[1] + v[2] + v[3]);
        store((int64_t)(u * 16 + r) * o.width + k0 + col, v);
      }
    }
  }
  if (!odd) return;
  asm volatile("" ::: "memory");  // what the thread has stored is read as another type
#pragma unroll 1
  for (int i = 0; i < 4 * NT; ++i) {  // (the thread's places: once more behind the sums, whose registers are free now)
    const int r = i / 4 * 16 + (COLS ? (threadIdx.x & 3) * 4 + i % 4 : threadIdx.x >> 4);
    const int col = COLS ? threadIdx.x >> 2 : (threadIdx.x & 15) * 4 + i % 4;
    if (k0 + col >= o.width || r >= p.r) continue;
    const int64_t to = COLS ? (int64_t)(k0 + col) * p.r + r : (int64_t)r * o.width + k0 + col;
    if (!isnan(alone ? unpack16<BF>(grad[to], 0) : share[to])) continue;
    float s = 0.f;
#pragma unroll 1
    for (int t = 0; t < chunk.z && !isnan(s); t += 8) {  // eight positions' h side by side
      u4 h = *(const u4*)(o.packs.col + (int64_t)(chunk.y + t) * kR + r * 8);
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = t + e < chunk.z ? o.in[order[t + e] * o.ld + k0 + col] : 0;
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        if (DROP && t + e < chunk.z)
          v[0] &= philox.mask((k0 + col) >> 3, order[t + e], p.drop)[(col & 7) >> 1] >> (16 * (col & 1));
        s += unpack16<BF>(v[0], 0) * unpack16<BF>(h[0], 0);
#pragma unroll
        for (int j = 0; j < 7; ++j) v[j] = v[j + 1];
        h = u4{h[0] >> 16 | h[1] << 16, h[1] >> 16 | h[2] << 16, h[2] >> 16 | h[3] << 16, h[3] >> 16};
      }
    }
    if (isfinite(s)) continue;
    if (alone) grad[to] = (uint16_t)pack16<BF>(s, 0.f);
    else share[to] = s;
  }
}

// The first launch of a backward pass: A [r][k] turned to [k][r] and B [n][r] to [r][n], and g h^T.  5325 rows
// of 4096 by rank 16 14.3 us for 51 MB (3.5 TB/s), 1763 of 11008 by rank 64 22.0 us for 63 MB (2.9 TB/s).
template <bool BF, int NT>
__global__ void __launch_bounds__(kOuterThreads)
first_kernel(AdapterArgs p, OuterArgs o, uint16_t* at, uint16_t* bt, int a_tiles, int b_tiles) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kOuterLds];
  int i = blockIdx.x;
  const int rt = (p.r + 63) / 64, turns = (a_tiles + b_tiles) * p.adapters;
  if (i < turns) {
    const int ad = i / (a_tiles + b_tiles);
    i -= ad * (a_tiles + b_tiles);
    uint16_t* tile = reinterpret_cast<uint16_t*>(lds);
    if (i < a_tiles) {
      const int64_t m = (int64_t)ad * p.r * p.k;
      turn_tile(p.a + m, at + m, p.r, p.k, i % rt * 64, i / rt * 64, tile);
    } else {
      i -= a_tiles;
      const int64_t m = (int64_t)ad * p.r * p.n;
      turn_tile(p.b + m, bt + m, p.n, p.r, i / rt * 64, i % rt * 64, tile);
    }
    return;
  }
  i -= turns;
  const int cols = (o.width + 63) / 64;
  outer<BF, NT, false, false, true>(p, o, i / cols, i % cols * 64, lds);
}
// dh x^T and dx, of the same tiles of x.  5325 rows of 4096 by rank 16 with dropout 26.5 us for 96 MB
// (3.6 TB/s), 1763 by rank 64 16.2 us for 41 MB (2.5 TB/s).
template <bool BF, int NT, bool DX, bool DROP>
__global__ void __launch_bounds__(kOuterThreads) outer_kernel(AdapterArgs p, OuterArgs o) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kOuterLds];
  const int i = blockIdx.x, cols = (o.width + 63) / 64;
  outer<BF, NT, DX, DROP, false>(p, o, i / cols, i % cols * 64, lds);
}

// dA and dB of the adapters of several chunks, whose shares are summed in order, and of none; four
// elements a thread.  4.0 us, a launch and two trips to memory.
template <bool BF>
__global__ void __launch_bounds__(kThreads) reduce_kernel(AdapterArgs p, const float* share_a, const float* share_b) {
  const int64_t each_a = p.da ? (int64_t)p.r * p.k / 4 : 0, each_b = p.db ? (int64_t)p.r * p.n / 4 : 0;
  const int64_t items = (each_a + each_b) * p.adapters;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < items; i += (int64_t)gridDim.x * kThreads) {
    const int ad = (int)(i / (each_a + each_b));
    const int64_t at = i - ad * (each_a + each_b);
    const bool is_a = at < each_a;
    const int64_t q = is_a ? at : at - each_a, each = is_a ? each_a : each_b;
    const float* share = (is_a ? share_a : share_b) + q * 4;
    const int c0 = p.plan[p.l.chunk_start + ad], c1 = p.plan[p.l.chunk_start + ad + 1];
    if (c1 - c0 == 1) continue;  // stored already
    f4 v = {};
    if (c0 < c1) share += p.plan[p.l.chunk + 4 * c0 + 3] * each * 4;
    for (int c = 0; c < c1 - c0; c += 4) {  // four loads in flight
      f4 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = *(const f4*)(share + min(c + e, c1 - c0 - 1) * each * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < c1 - c0) v += x[e];
    }
    *(uint2*)((is_a ? p.da : p.db) + (ad * each + q) * 4) = make_uint2(pack16<BF>(v[0], v[1]), pack16<BF>(v[2], v[3]));
  }
}

template <bool BF, int NT>
hipError_t launch_grad(const AdapterArgs& a, const BackwardWs& w, hipStream_t stream) {
  uint16_t* const at = reinterpret_cast<uint16_t*>(a.ws + w.at);
  uint16_t* const bt = reinterpret_cast<uint16_t*>(a.ws + w.bt);
  float* const share_a = reinterpret_cast<float*>(a.ws + w.da);
  float* const share_b = reinterpret_cast<float*>(a.ws + w.db);
  const bool inner = a.dx != nullptr || a.da != nullptr;
  const int rt = (a.r + 63) / 64;
  const int a_tiles = a.dx ? rt * ((a.k + 63) / 64) : 0, b_tiles = inner ? rt * ((a.n + 63) / 64) : 0;
  const int outer_items = a.db ? a.l.chunks * ((a.n + 63) / 64) : 0;
  OuterArgs g = {a.g, a.ldg, a.n, {}, share_b, a.db, nullptr};
  place_col(g.packs, a.l, a.r, a.h);
  const unsigned first = (unsigned)((a_tiles + b_tiles) * a.adapters + outer_items);
  if (first) first_kernel<BF, NT><<<first, kOuterThreads, 0, stream>>>(a, g, at, bt, a_tiles, b_tiles);
  if (inner) {
    AdapterPacks packs = {};
    hipError_t e;
    if (a.adapters > 0) {
      float* const planes = reinterpret_cast<float*>(a.ws);
      const ShrinkArgs s = {a.l, a.plan, a.g, a.ldg, bt, a.n, a.r, a.adapters, 0, nullptr, planes};
      if ((e = launch_shrink(a.bf16, s, w.splits, stream)) != hipSuccess) return e;
      if (a.dx != nullptr) place_row(packs, a.l, a.r, a.ws + w.row);
      if (a.da != nullptr) place_col(packs, a.l, a.r, a.ws + w.col);
      if ((e = launch_join(a, planes, w.splits, packs, stream)) != hipSuccess) return e;
    }
    const OuterArgs x = {a.x, a.ldx, a.k, packs, a.da ? share_a : nullptr, a.da, at};
    const unsigned grid = (unsigned)(a.l.chunks * ((a.k + 63) / 64));
    if (a.dx != nullptr) {
      if (a.drop) outer_kernel<BF, NT, true, true><<<grid, kOuterThreads, 0, stream>>>(a, x);
      else outer_kernel<BF, NT, true, false><<<grid, kOuterThreads, 0, stream>>>(a, x);
    } else {
      if (a.drop) outer_kernel<BF, NT, false, true><<<grid, kOuterThreads, 0, stream>>>(a, x);
      else outer_kernel<BF, NT, false, false><<<grid, kOuterThreads, 0, stream>>>(a, x);
    }
  }
  if (a.da != nullptr || a.db != nullptr) {
    const int64_t items = (int64_t)a.adapters * a.r * ((a.da ? a.k : 0) + (a.db ? a.n : 0)) / 4;
    const unsigned grid = (unsigned)std::min<int64_t>((items + kThreads - 1) / kThreads, 1 << 16);
    reduce_kernel<BF><<<grid, kThreads, 0, stream>>>(a, share_a, share_b);
  }
  return hipGetLastError();
}
template <bool BF>
hipError_t launch_rank(const AdapterArgs& a, const BackwardWs& w, hipStream_t stream) {
  if (a.r <= 16) return launch_grad<BF, 1>(a, w, stream);
  if (a.r <= 32) return launch_grad<BF, 2>(a, w, stream);
  if (a.r <= 64) return launch_grad<BF, 4>(a, w, stream);
  return launch_grad<BF, 8>(a, w, stream);
}

}  // namespace

hipError_t launch_adapters_grad(const AdapterArgs& a, const BackwardWs& w, hipStream_t stream) {
  return a.bf16 ? launch_rank<true>(a, w, stream) : launch_rank<false>(a, w, stream);
}

}  // namespace dw4
