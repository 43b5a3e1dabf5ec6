// Gradients of the low-rank adapters (w4a16_adapters.hip): with g_t the output's gradient,
// h_t = A_a d(x_t) and dh_t = s_a B_a^T g_t,
//   dx_t = d'(A_a^T dh_t),  dA_a = sum of dh_t d(x_t)^T,  dB_a = s_a sum of g_t h_t^T.
//
// Four launches.  grad_b_kernel reads g once for both of its products: 32 rows by 256
// columns at a time, from registers for B^T g (rows as the matrix instruction's columns) and,
// turned around by way of LDS, for g h^T (rows as its reduction).  join_kernel sums the
// slabs' planes of dh.  grad_a_kernel reads x once, for dh x^T, and writes dx from the same
// tile.  reduce_kernel sums the chunks' shares of dA and dB in order: no float atomics.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "w4a16_adapters_device.h"

namespace dw4 {

namespace {

constexpr int kThreads = 256;
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

// The power of two that brings a chunk's values of each column r of h within fp16's range
// (for the lane's columns 16 t + lane % 16; bf16: none).
template <bool BF, int NT>
__device__ __forceinline__ void column_exponents(const float* h, int rows, int r, float* tmp, int (&e)[NT]) {
  if constexpr (BF) {
#pragma unroll
    for (int t = 0; t < NT; ++t) e[t] = 0;
  } else {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = min(t * 16 + c, r - 1);
      float m = 0.f;
      for (int i = wave * 4 + g; i < rows; i += 16) m = fmaxf(m, fabsf(h[(int64_t)i * r + col]));
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      __syncthreads();
      if (g == 0) tmp[wave * 16 + c] = m;
      __syncthreads();
      e[t] = range_exponent<BF>(fmaxf(fmaxf(tmp[c], tmp[16 + c]), fmaxf(tmp[32 + c], tmp[48 + c])));
    }
    __syncthreads();
  }
}

// Columns 16 t + lane % 16 of h, rows 8 (lane / 16) .. + 7 of a step (of which `rows` are
// there), as B operands.
template <bool BF>
__device__ __forceinline__ void column_operand(const float* h, int rows, int r, int t, int e, u4& hi, u4& lo) {
  const int lane = threadIdx.x & 63, g = lane >> 4, col = t * 16 + (lane & 15);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = 8 * g + j;
    const bool in = row < rows && col < r;
    v[j] = h[in ? row * r + col : 0];
    if (!in) v[j] = 0.f;
    if constexpr (!BF) v[j] = times_pow2(v[j], e);
  }
  split16<BF>(v, hi, lo);
}

// Chunk blockIdx.x's rows, columns 256 blockIdx.y on: planes of B^T g, and the chunk's g^T h.
template <bool BF, int NT>
__global__ void __launch_bounds__(kThreads) grad_b_kernel(AdapterArgs p, AdapterGradParts parts) {
  constexpr int kPitch = NT * 16 + 4;
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  float* const red = reinterpret_cast<float*>(sm);  // [4][kStep][kPitch]
  const int4 chunk = *(const int4*)(p.plan + p.l.chunk + 4 * blockIdx.x);
  const int ad = chunk.x;
  if (ad < 0 || ad >= p.adapters) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  uint16_t* const tile = reinterpret_cast<uint16_t*>(red + 4 * kStep * kPitch) + wave * kStep * kTurn;
  const int n0 = blockIdx.y * kSlab + wave * 64;
  const int32_t* order = p.plan + p.l.order + chunk.y;
  const float* h = p.h + (int64_t)chunk.y * p.r;
  float* plane = p.ws + ((int64_t)blockIdx.y * p.l.positions + chunk.y) * p.r;
  // B turned around: row r of the operand, eight columns n
  u4 bt[2][NT];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = n0 + 32 * j + 8 * g + 2 * e + i, r = t * 16 + c;
          const bool in = n < p.n && r < p.r;
          w[i] = p.b[in ? ((int64_t)ad * p.n + n) * p.r + r : 0];
          if (!in) w[i] = 0;
        }
        bt[j][t][e] = w[0] | w[1] << 16;
      }
  int ex[NT];
  column_exponents<BF, NT>(h, chunk.z, p.r, red, ex);
  f4 acc[4][NT] = {};
  for (int first = 0; first < chunk.z; first += kStep) {
    u4 y[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int at = first + t * 16 + c;
      const int row = at < chunk.z ? order[at] : -1;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + 32 * j + 8 * g;
        const bool in = row >= 0 && n < p.n;
        y[t][j] = *(const u4*)(p.g + (in ? row * p.ldg + n : 0));
        if (!in) y[t][j] = u4{};
        *(u4*)(tile + (t * 16 + c) * kTurn + 32 * j + 8 * g) = y[t][j];
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        f4 d = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) d = mfma16_of<BF>(bt[j][u], y[t][j], d);
        *(f4*)(red + (wave * kStep + t * 16 + c) * kPitch + u * 16 + 4 * g) = d;
      }
    __syncthreads();
    const int quads = p.r / 4;
    for (int i = threadIdx.x; i < kStep * quads; i += kThreads) {
      const int at = i / quads, q = i % quads * 4;
      f4 v = *(const f4*)(red + at * kPitch + q);
#pragma unroll
      for (int w = 1; w < 4; ++w) v += *(const f4*)(red + (w * kStep + at) * kPitch + q);
      if (first + at < chunk.z) *(f4*)(plane + (int64_t)(first + at) * p.r + q) = v;
    }
    u4 yt[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) yt[t] = turned(tile, t);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      u4 hi, lo;
      column_operand<BF>(h + (int64_t)first * p.r, chunk.z - first, p.r, u, ex[u], hi, lo);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        acc[t][u] = mfma16_of<BF>(yt[t], hi, acc[t][u]);
        acc[t][u] = mfma16_of<BF>(yt[t], lo, acc[t][u]);
      }
    }
    __syncthreads();
  }
  if (p.db == nullptr) return;
  float* share = p.ws + parts.db + (int64_t)blockIdx.x * p.n * p.r;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int r = u * 16 + c;
      if (r >= p.r) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + t * 16 + 4 * g + i;
        if (n < p.n) share[(int64_t)n * p.r + r] = BF ? acc[t][u][i] : times_pow2(acc[t][u][i], -ex[u]);
      }
    }
}

// dh = s_a (1 / kept share) times the sum of its planes.
__global__ void __launch_bounds__(kThreads) join_kernel(AdapterArgs p, AdapterGradParts parts, int slabs) {
  const int ad = p.plan[p.l.tile_adapter + blockIdx.x];
  if (ad < 0 || ad >= p.adapters) return;
  const float scale = p.scaling[ad] * p.keep_scale;
  const int32_t* order = p.plan + p.l.order + (int64_t)blockIdx.x * p.l.align;
  const int quads = p.r / 4;
  const int64_t first = (int64_t)blockIdx.x * p.l.align * p.r;
  for (int i = threadIdx.x; i < p.l.align * quads; i += kThreads) {
    f4 v = {};
    if (order[i / quads] >= 0) {
      for (int s = 0; s < slabs; ++s) v += *(const f4*)(p.ws + (int64_t)s * p.l.positions * p.r + first + 4 * i);
      v *= scale;
    }
    *(f4*)(p.ws + parts.dh + first + 4 * i) = v;
  }
}

// Chunk blockIdx.x's rows, columns 256 blockIdx.y on of x: dx, and the chunk's dh^T d(x).
template <bool BF, int NT, bool DROP>
__global__ void __launch_bounds__(kThreads) grad_a_kernel(AdapterArgs p, AdapterGradParts parts) {
  constexpr int kJ = NT == 1 ? 1 : NT / 2;
  __shared__ __attribute__((aligned(16))) uint16_t tiles[4][kStep * kTurn];
  __shared__ float tmp[64];
  const int4 chunk = *(const int4*)(p.plan + p.l.chunk + 4 * blockIdx.x);
  const int ad = chunk.x;
  if (ad < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int k0 = blockIdx.y * kSlab + wave * 64;
  const int32_t* order = p.plan + p.l.order + chunk.y;
  if (ad >= p.adapters) {  // rows without an adapter
    if (p.dx == nullptr) return;
    const int units = min(kSlab, p.k - blockIdx.y * kSlab) / 8;
    for (int i = threadIdx.x; i < chunk.z * units; i += kThreads)
      *(u4*)(p.dx + order[i / units] * p.lddx + blockIdx.y * kSlab + i % units * 8) = u4{};
    return;
  }
  uint16_t* const tile = tiles[wave];
  const float* dh = p.ws + parts.dh + (int64_t)chunk.y * p.r;
  // A turned around: the operand's row is a column of x, eight values of r
  u4 at[2][2][kJ];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int col = k0 + 32 * q + (c >> 2) * 8 + u * 4 + (c & 3);
            const int r = (NT == 1 ? (g & 1) * 8 : 32 * j + 8 * g) + 2 * e + i;
            const bool in = col < p.k && r < p.r;
            w[i] = p.a[in ? ((int64_t)ad * p.r + r) * p.k + col : 0];
            if (!in) w[i] = 0;
          }
          at[q][u][j][e] = w[0] | w[1] << 16;
        }
  const Philox philox(DROP ? p.seed : reinterpret_cast<const int64_t*>(p.plan));
  int ex[NT];
  column_exponents<BF, NT>(dh, chunk.z, p.r, tmp, ex);
  f4 acc[4][NT] = {};
  for (int first = 0; first < chunk.z; first += kStep) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int pos = first + t * 16 + c;
      const int row = pos < chunk.z ? order[pos] : -1;
      u4 keep[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = k0 + 32 * q + 8 * g;
        const bool in = row >= 0 && k < p.k;
        u4 v = *(const u4*)(p.x + (in ? row * p.ldx + k : 0));
        if constexpr (DROP) {
          keep[q] = philox.mask(k >> 3, row, p.drop);
          v &= keep[q];
        }
        if (!in) v = u4{};
        *(u4*)(tile + (t * 16 + c) * kTurn + 32 * q + 8 * g) = v;
      }
      if (p.dx == nullptr) continue;
      // the row's dh as a B operand
      float v[kJ][8], m = 0.f;
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int r = NT == 1 ? (g & 1) * 8 : 32 * j + 8 * g;
        const bool in = row >= 0 && r < p.r;
        const float* from = dh + (in ? (int64_t)pos * p.r + r : 0);
        const f4 a = *(const f4*)from, b = *(const f4*)(from + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[j][e] = in ? (e < 4 ? a[e] : b[e - 4]) : 0.f;
          if constexpr (!BF) m = fmaxf(m, fabsf(v[j][e]));
        }
      }
      int e = 0;
      if constexpr (!BF) {
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        e = range_exponent<BF>(m);
      }
      f4 d[2][2] = {};
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        if constexpr (!BF) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = times_pow2(v[j][i], e);
        }
        u4 hi, lo;
        split16<BF>(v[j], hi, lo);
        if (NT == 1 && g >= 2) hi = lo;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            d[q][u] = mfma16_of<BF>(at[q][u][j], hi, d[q][u]);
            if constexpr (NT > 1) d[q][u] = mfma16_of<BF>(at[q][u][j], lo, d[q][u]);
          }
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        u4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float lo = d[q][i >> 1][(i & 1) * 2], hi = d[q][i >> 1][(i & 1) * 2 + 1];
          if constexpr (!BF) {
            lo = times_pow2(lo, -e);
            hi = times_pow2(hi, -e);
          }
          o[i] = pack16<BF>(lo, hi);
        }
        if constexpr (DROP) o &= keep[q];
        const int k = k0 + 32 * q + 8 * g;
        if (row >= 0 && k < p.k) *(u4*)(p.dx + row * p.lddx + k) = o;
      }
    }
    if (p.da == nullptr) continue;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    u4 xt[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) xt[t] = turned(tile, t);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      u4 hi, lo;
      column_operand<BF>(dh + (int64_t)first * p.r, chunk.z - first, p.r, u, ex[u], hi, lo);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        acc[t][u] = mfma16_of<BF>(xt[t], hi, acc[t][u]);
        acc[t][u] = mfma16_of<BF>(xt[t], lo, acc[t][u]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if (p.da == nullptr) return;
  float* share = p.ws + parts.da + (int64_t)blockIdx.x * p.r * p.k;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int r = u * 16 + c, k = k0 + t * 16 + 4 * g;
      f4 v = acc[t][u];
      if constexpr (!BF) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = times_pow2(v[i], -ex[u]);
      }
      if (r < p.r && k < p.k) *(f4*)(share + (int64_t)r * p.k + k) = v;
    }
}

// dA and dB of each adapter: its chunks' shares summed in order; four elements a thread.
template <bool BF>
__global__ void __launch_bounds__(kThreads) reduce_kernel(AdapterArgs p, AdapterGradParts parts) {
  const int64_t each_a = p.da ? (int64_t)p.r * p.k / 4 : 0, each_b = p.db ? (int64_t)p.r * p.n / 4 : 0;
  const int64_t items = (each_a + each_b) * p.adapters;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < items; i += (int64_t)gridDim.x * kThreads) {
    const int ad = (int)(i / (each_a + each_b));
    const int64_t at = i - ad * (each_a + each_b);
    const bool is_a = at < each_a;
    const int64_t q = is_a ? at : at - each_a, each = is_a ? (int64_t)p.r * p.k / 4 : (int64_t)p.r * p.n / 4;
    const float* share = p.ws + (is_a ? parts.da : parts.db);
    const int c0 = p.plan[p.l.chunk_start + ad], c1 = p.plan[p.l.chunk_start + ad + 1];
    f4 v = {};
    for (int c = c0; c < c1; ++c) v += *(const f4*)(share + (c * each + q) * 4);
    if (!is_a) v *= p.scaling[ad] * p.keep_scale;
    *(uint2*)((is_a ? p.da : p.db) + (ad * each + q) * 4) = make_uint2(pack16<BF>(v[0], v[1]), pack16<BF>(v[2], v[3]));
  }
}

template <bool BF, int NT>
hipError_t launch_grad(const AdapterArgs& a, hipStream_t stream) {
  const AdapterGradParts parts = adapter_grad_parts(a.l, a.k, a.n, a.r);
  const int slabs = (a.n + kSlab - 1) / kSlab;
  constexpr size_t smem = 4 * kStep * (NT * 16 + 4) * sizeof(float) + 4 * kStep * kTurn * sizeof(uint16_t);
  if constexpr (smem > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&grad_b_kernel<BF, NT>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != hipSuccess) return e;
  }
  grad_b_kernel<BF, NT><<<dim3(a.l.chunks, slabs), kThreads, smem, stream>>>(a, parts);
  if (a.dx != nullptr || a.da != nullptr) {
    join_kernel<<<a.l.tiles, kThreads, 0, stream>>>(a, parts, slabs);
    const dim3 grid(a.l.chunks, (a.k + kSlab - 1) / kSlab);
    if (a.drop) grad_a_kernel<BF, NT, true><<<grid, kThreads, 0, stream>>>(a, parts);
    else grad_a_kernel<BF, NT, false><<<grid, kThreads, 0, stream>>>(a, parts);
  }
  if (a.da != nullptr || a.db != nullptr) {
    const int64_t items = (int64_t)a.adapters * a.r * ((a.da ? a.k : 0) + (a.db ? a.n : 0)) / 4;
    reduce_kernel<BF><<<(unsigned)std::min<int64_t>((items + kThreads - 1) / kThreads, 1 << 16), kThreads, 0, stream>>>(a, parts);
  }
  return hipGetLastError();
}
template <bool BF>
hipError_t launch_rank(const AdapterArgs& a, hipStream_t stream) {
  if (a.r <= 16) return launch_grad<BF, 1>(a, stream);
  if (a.r <= 32) return launch_grad<BF, 2>(a, stream);
  if (a.r <= 64) return launch_grad<BF, 4>(a, stream);
  return launch_grad<BF, 8>(a, stream);
}

}  // namespace

hipError_t launch_adapters_grad(const AdapterArgs& a, hipStream_t stream) {
  return a.bf16 ? launch_rank<true>(a, stream) : launch_rank<false>(a, stream);
}

}  // namespace dw4
