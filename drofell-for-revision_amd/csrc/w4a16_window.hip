// Windowed attention of few rows over a paged KV cache: decode steps, and up
// to 32 rows (new tokens x query heads) per kv head of short prompts and
// drafts.
//
//   out[i][h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max),
// over the tokens j <= i with j > i - window or j < sinks, positions i counted
// in the sequence.  Cache layout as in w4a16_attention.hip: a 16-byte unit of
// a key block is 8 dims of a token, one of a value block 8 tokens of a dim, the
// operands of both products as they lie.
//
// HBM-bound: the keys and values seen are read once, straight into operand
// registers, and only they: blocks before the window that hold no sink are not
// even looked up.  A workgroup takes one (sequence, kv head) and up to 32 rows
// of it as the columns of 32 x 32 x 16 products; its waves take steps of 32
// tokens round-robin, keep a running max and sum per row, and meet once in LDS.
// Probabilities enter p . v as two 16-bit parts (22 bits of fp16's 2^10 p, 16 of
// bf16's p): the products' time is hidden behind the stream, and so is a look at every
// value for NaN and infinities, which take a path of their own (48 streams 146.5 us without
// it, 146.8 with it).  Where there are
// too few (sequence, kv head) pairs for the CUs, the steps are split among
// workgroups, which leave max, sum and unnormalised fp32 outputs for
// window_join_kernel, in a fixed order (deterministic).
//
// Measured: 48 streams, window 4096 and 4 sinks, heads 32 on 8 of 128, bf16: 800 MB
// of cache in 144 us, 5.5 TB/s (a copy of 1 GiB reaches 5.2, reading alone 6.5).  One
// stream with window 512, where no load hides another (table, pointer, block, then
// the join in LDS): 7 to 10 us.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "w4a16_device.h"
#include "w4a16_window.h"
#include "w4a16_window_device.h"

namespace dw4 {

namespace {

template <int HS, int BS, bool BF, int W>
__global__ void __launch_bounds__(W * 64, W == 8 || HS <= 128 ? 2 : 1)
window_rows_kernel(WindowArgs a, int splits, int cols, float* __restrict__ ws_ml, float* __restrict__ ws_out) {
  constexpr int KD = HS / 16;         // 16-dim reduction steps of q . k
  constexpr int ND = (HS + 31) / 32;  // 32-dim tiles of p . v (the last may be half empty)
  constexpr int NB = 32 / BS;         // blocks of a step
  constexpr bool VTAIL = HS % 32 != 0;
  extern __shared__ __attribute__((aligned(16))) float sm[];

  int pair, split;
  if (!work_of(blockIdx.x, a.num_seqs * a.num_kv_heads, splits, pair, split)) return;
  const int seq = pair / a.num_kv_heads, kvh = pair % a.num_kv_heads;
  const int G = a.num_heads / a.num_kv_heads;
  int q0, q1;
  seq_rows(a.starts, seq, a.total_rows, q0, q1);
  const int n = min(q1 - q0, a.max_query);
  const int nrows = n * G;  // at most kWinRowsTile
  if (nrows <= 0) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, half = lane >> 5;
  const int len = a.lens[seq];
  const int cap = min(len, a.max_blocks * BS);  // a table shorter than the context ends it
  const int p0 = len - (q1 - q0);                // position of the first new token
  const Span span = Span::of<32>(p0, p0 + n - 1, cap, a.window, a.sinks);
  const int per = (span.steps + splits - 1) / splits;
  const int s0 = split * per, s1 = min(span.steps, s0 + per);
  const int nsw = s0 + wave < s1 ? (s1 - s0 - wave + W - 1) / W : 0;  // this wave's steps

  // row c (rows past the last repeat it; they are not stored)
  const int row = min(c, nrows - 1);
  const int pos = p0 + row / G;
  const int last = min(pos, cap - 1), before = a.window == 0 ? INT32_MIN : pos - a.window;

  // Lane l holds the addresses of block l % NB of the wave's step l / NB (of
  // 64 / NB), 0 for a block that the table lacks.
  uint64_t kp = 0, vp = 0;
  auto fetch = [&](int i0) {
    const int i = i0 + lane / NB;
    kp = vp = 0;
    if (i < nsw) {
      const int b = span.token<32>(s0 + wave + W * i) / BS + lane % NB;
      const int blk = b * BS < cap ? a.tables[(size_t)seq * a.max_blocks + b] : -1;
      if (blk >= 0 && blk < a.num_blocks) {
        const size_t head = (size_t)kvh * a.kv_head_stride * sizeof(uint16_t);
        kp = (uint64_t)a.kptr[blk] + head;
        vp = (uint64_t)a.vptr[blk] + head;
      }
    }
  };
  auto block_of = [&](uint64_t v, int l) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l);
    return ((uint64_t)hi << 32) | lo;
  };
  const int ktok = row_token(c);
  const uint32_t koff = (uint32_t)((half * BS + ktok % BS) * 16);
  h8 kreg[KD], vreg[ND][2];
  uint32_t held = 0, held_next = 0;  // bit b: block b of the step is there
  auto load_k = [&](int i) {
    const int l = i * NB % 64;
    if (l == 0) fetch(i);
    uint64_t base_k = block_of(kp, l);
    held_next = base_k != 0;
    if (NB == 2) {
      const uint64_t second = block_of(kp, l + 1);
      held_next |= (uint32_t)(second != 0) << 1;
      base_k = ktok < 16 ? base_k : second;
    }
    const unsigned char* kb = reinterpret_cast<const unsigned char*>(base_k) + koff;
#pragma unroll
    for (int j = 0; j < KD; ++j) kreg[j] = base_k == 0 ? h8{} : *(const h8*)(kb + j * (2 * BS * 16));
  };
  auto load_v = [&](int i) {
    const int l = i * NB % 64;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint64_t base_v = block_of(vp, NB == 2 ? l + s : l);
      const unsigned char* vb = reinterpret_cast<const unsigned char*>(base_v) + (c * BS + (BS == 32 ? 16 * s : 0) + 8 * half) * 2;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        if (base_v == 0 || (VTAIL && d * 32 + c >= HS)) vreg[d][s] = h8{};
        else vreg[d][s] = *(const h8*)(vb + d * (32 * BS * 2));
      }
    }
  };
  if (nsw > 0) {
    load_k(0);
    load_v(0);
  }
  held = held_next;
  h8 qreg[KD];  // B operand: column c is row c
  {
    const uint16_t* qp = a.q + (size_t)(q0 + row / G) * a.q_stride + (size_t)(kvh * G + row % G) * HS + 8 * half;
#pragma unroll
    for (int j = 0; j < KD; ++j) qreg[j] = *(const h8*)(qp + 16 * j);
  }

  float m = kNoMax, l = 0.f;  // of row c (l: this lane's tokens)
  f16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f16v{};
  for (int i = 0; i < nsw; ++i) {
    const int t = span.token<32>(s0 + wave + W * i);
    f16v s = {};
#pragma unroll
    for (int j = 0; j < KD; ++j) s = mfma32_of<BF>(kreg[j], qreg[j], s);
    // every row sees every token of the step?
    const bool full = held == (1u << NB) - 1 && t + 31 <= min(p0, cap - 1) &&
                      (a.window == 0 || t > p0 + n - 1 - a.window || t + 31 < a.sinks);
    uint32_t seen = 0xFFFF;  // bit e: score e
    if (!full) {
      seen = own_scores(seen_of(t, last, before, a.sinks), half);
      if constexpr (NB == 1) seen = held ? seen : 0u;
      else seen &= (held & 1 ? 0xFFu : 0u) | (held & 2 ? 0xFF00u : 0u);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = where_seen(seen, e, s[e], -INFINITY);
    }
    if (i + 1 < nsw) load_k(i + 1);
    held = held_next;
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = both_max(mx) * a.scale_log2;
    if (__any(mx > m + kLag)) {  // the maximum may lag kLag behind
      const float mn = fmaxf(m, mx);
      const float f = __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= f;
      m = mn;
    }
    const float shift = p_shift<BF>() - m;
    h8 hi[2], lo[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      u4 h, r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[8 * g + 2 * e], a.scale_log2, shift));
        const float y = __builtin_amdgcn_exp2f(fmaf(s[8 * g + 2 * e + 1], a.scale_log2, shift));
        l += x;
        l += y;
        h[e] = pack2<BF>(x, y);
        r[e] = pack2<BF>(x - unpack<BF>(h[e], 0), y - unpack<BF>(h[e], 1));
      }
      hi[g] = __builtin_bit_cast(h8, h);
      lo[g] = __builtin_bit_cast(h8, r);
    }
    // a value that some rows do not see (or that is behind the context) must not reach
    // them as 0 * inf, nor an infinity a row that sees it as inf - inf, by a negative
    // second part
    uint32_t bits = 0;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      add_nonfinite<BF>(vreg[d][0], bits);
      add_nonfinite<BF>(vreg[d][1], bits);
    }
    const bool odd = __any((bits & kNonfinite) != 0);
    if (odd) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        for (uint32_t sign = 0; sign <= 0x8000u; sign += 0x8000u) {
          const float inf = sign ? -INFINITY : INFINITY;
          f16v count = {};
#pragma unroll
          for (int g = 0; g < 2; ++g)
            count = mfma32_of<BF>(infinite_part<BF>(vreg[d][g], sign), ones_of<BF>(seen >> (8 * g)), count);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (count[e] > 0.f) o[d][e] += inf;
        }
        vreg[d][0] = finite_part<BF>(vreg[d][0]);
        vreg[d][1] = finite_part<BF>(vreg[d][1]);
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        o[d] = mfma32_of<BF>(vreg[d][g], hi[g], o[d]);
        o[d] = mfma32_of<BF>(vreg[d][g], lo[g], o[d]);
      }
    if (i + 1 < nsw) load_v(i + 1);
  }

  // ---- the waves' outputs, combined in wave order
  float* red = sm;                  // [waves][cols][HS]
  float* ml = red + W * cols * HS;  // [waves][cols][2]
  l = both_sum(l);
  if (c < nrows) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int dim = d * 32 + 2 * e + 4 * half;
        if (!VTAIL || dim < HS)
          *(f4*)(red + (wave * cols + c) * HS + dim) = f4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
      }
    if (half == 0) {
      ml[(wave * cols + c) * 2] = m;
      ml[(wave * cols + c) * 2 + 1] = l;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * HS; i += W * 64) {
    const int r = i / HS, d = i % HS;
    float gm = ml[r * 2];
#pragma unroll
    for (int w = 1; w < W; ++w) gm = fmaxf(gm, ml[(w * cols + r) * 2]);
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[(w * cols + r) * 2] - gm);
      sum += f * ml[(w * cols + r) * 2 + 1];
      acc += f * red[(w * cols + r) * HS + d];
    }
    const int token = q0 + r / G, head = kvh * G + r % G;
    if (splits == 1) {
      const float y = sum == 0.f ? acc : acc / sum;  // no visible token: zeros
      a.out[(size_t)token * a.o_stride + (size_t)head * HS + d] = (uint16_t)pack2<BF>(y, 0.f);
    } else {
      const size_t slot = ((size_t)token * a.num_heads + head) * splits + split;
      ws_out[slot * HS + d] = acc;
      if (d == 0) {
        ws_ml[2 * slot] = gm;
        ws_ml[2 * slot + 1] = sum;
      }
    }
  }
}

// The splits of each row joined in their order, a wave per (row, head).  Launch-bound: 4 to
// 5 us for the splits of 48 tokens with 32 heads as for those of 84.
template <int HS, bool BF>
__global__ void __launch_bounds__(256)
window_join_kernel(WindowArgs a, int splits, const float* __restrict__ ws_ml,
                   const float* __restrict__ ws_out) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int head = (int)(id % a.num_heads);
  const int i = (int)(id / a.num_heads % a.max_query);
  const int seq = (int)(id / a.num_heads / a.max_query);
  if (seq >= a.num_seqs) return;
  int q0, q1;
  seq_rows(a.starts, seq, a.total_rows, q0, q1);
  if (i >= q1 - q0) return;
  const size_t slot = ((size_t)(q0 + i) * a.num_heads + head) * splits;
  // max and sum of all splits: lane s holds split s (of 64 at a time)
  float gm = kNoMax;
  for (int s = lane; s < splits; s += 64) gm = fmaxf(gm, ws_ml[2 * (slot + s)]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) gm = fmaxf(gm, __shfl_xor(gm, off));
  constexpr int D = (HS + 63) / 64;
  float sum = 0.f, o[D] = {};
  for (int s0 = 0; s0 < splits; s0 += 8) {
    float v[8][D], f[8], ls[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool in = s0 + u < splits;
      const size_t at = slot + min(s0 + u, splits - 1);
      f[u] = in ? __builtin_amdgcn_exp2f(ws_ml[2 * at] - gm) : 0.f;
      ls[u] = ws_ml[2 * at + 1];
#pragma unroll
      for (int d = 0; d < D; ++d) v[u][d] = HS % 64 == 0 || lane + 64 * d < HS ? ws_out[at * HS + lane + 64 * d] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s0 + u < splits) {
        sum += f[u] * ls[u];
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] += f[u] * v[u][d];
      }
    }
  }
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (HS % 64 == 0 || lane + 64 * d < HS)
      a.out[(size_t)(q0 + i) * a.o_stride + (size_t)head * HS + lane + 64 * d] =
          (uint16_t)pack2<BF>(sum == 0.f ? o[d] : o[d] / sum, 0.f);
}

template <int HS, int BS, bool BF, int W>
hipError_t launch_rows_w(const WindowArgs& a, const WindowPlan& p, float* ws_ml, float* ws_out,
                         hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const int cols = (int)std::min<int64_t>(kWinRowsTile, (int64_t)a.max_query * (a.num_heads / a.num_kv_heads));
  const size_t smem = win_rows_smem(HS, cols, W);
  auto kern = &window_rows_kernel<HS, BS, BF, W>;
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(kern), win_rows_smem(HS, kWinRowsTile, W), done);
  if (e != hipSuccess) return e;
  kern<<<win_grid(a.num_seqs * a.num_kv_heads, p.splits), W * 64, smem, stream>>>(a, p.splits, cols, ws_ml, ws_out);
  return hipGetLastError();
}

template <int HS, bool BF>
hipError_t launch_rows_hs(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream) {
  float* ws_ml = ws;
  float* ws_out = ws + win_ml_floats(a.total_rows, a.num_heads, p.splits);
  hipError_t e = hipErrorInvalidValue;
  if (p.rows) {
    if (p.waves == 4)
      e = a.block_size == 16 ? launch_rows_w<HS, 16, BF, 4>(a, p, ws_ml, ws_out, stream)
                             : launch_rows_w<HS, 32, BF, 4>(a, p, ws_ml, ws_out, stream);
    if constexpr (HS <= 128)
      if (p.waves == 8)
        e = a.block_size == 16 ? launch_rows_w<HS, 16, BF, 8>(a, p, ws_ml, ws_out, stream)
                               : launch_rows_w<HS, 32, BF, 8>(a, p, ws_ml, ws_out, stream);
  } else {
    e = launch_window_tile<BF>(a, p, ws, stream);
  }
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t joins = (int64_t)a.num_seqs * a.max_query * a.num_heads;
  window_join_kernel<HS, BF><<<(unsigned)((joins + 3) / 4), 256, 0, stream>>>(a, p.splits, ws_ml, ws_out);
  return hipGetLastError();
}

}  // namespace

template <bool BF>
hipError_t launch_window_rows(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream) {
  switch (a.head_size) {
    case 64: return launch_rows_hs<64, BF>(a, p, ws, stream);
    case 80: return launch_rows_hs<80, BF>(a, p, ws, stream);
    case 96: return launch_rows_hs<96, BF>(a, p, ws, stream);
    case 112: return launch_rows_hs<112, BF>(a, p, ws, stream);
    case 128: return launch_rows_hs<128, BF>(a, p, ws, stream);
    case 256: return launch_rows_hs<256, BF>(a, p, ws, stream);
    default: return hipErrorInvalidValue;
  }
}
template hipError_t launch_window_rows<WINDOW_BF16>(const WindowArgs&, const WindowPlan&, float*, hipStream_t);

#if !WINDOW_BF16
hipError_t launch_window(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream) {
  return a.bf16 ? launch_window_rows<true>(a, p, ws, stream) : launch_window_rows<false>(a, p, ws, stream);
}

// Tokens that one row tile may see, in steps of bk: two more than they fill,
// for a window that starts inside a step and the sinks before it.
static int64_t window_steps(const WindowArgs& a, int max_context, int tile_rows, int bk) {
  const int G = a.num_heads / a.num_kv_heads;
  int64_t span = max_context;
  if (a.window != 0)
    span = std::min<int64_t>(span, (int64_t)a.window + std::min(a.max_query, (tile_rows + G - 1) / G + 1));
  const int64_t far = a.window != 0 ? std::min<int64_t>(a.sinks, max_context - span) : 0;
  return (span + bk - 1) / bk + (far + bk - 1) / bk;
}

// Splits over the tokens, for calls that leave CUs without a workgroup; g
// workgroups without splits, n steps of tokens each.
//
// Rows kernel (32-token steps): one 8-wave workgroup per CU, at least 12 steps in a
// part; not for contexts under 24 steps, nor for two parts unless they are long
// (100 steps), which the join's launch costs more than it gains.  Between one and
// two workgroups per CU, of which some CUs then have two and others one, long
// contexts go in two parts, or three where those fill two per CU better.  Measured (us,
// one part / these / more; heads 32 on 8 unless said): 1 x 300 tokens 6.7 / - / 7.5 (4
// parts), 1 x 3000 24.8 / 10.2 / 10.5 (16), 1 x 8000 58 / 17.8 / 19 (32), 4 x 3000 28.5
// / 17.0 / 17.4 (8), 16 x 3000 33.4 / - / 35.0 (2), 16 x 8000 118 / 95 / 98.5 (4), 8 x
// 600, 32 on 32, 15.8 / - / 22.4 (2), 40 x 4100 150 / 124 / 126 (4), 48 x 4100 155 / 145 /
// 150 (3), 12 x 3500 with 7 new tokens 36.3 / 31.9 / 39.1 (3).  More workgroups than CUs: four waves each (32 x
// 128 tokens, 32 on 32, 23.5 with eight, 16.5).
//
// Tile kernel (64-token steps): one workgroup per CU, or two where that leaves
// fewer than four parts of a long context (64 steps), at least three steps in a
// part and at most 16 parts below 128 steps.  Measured (us, one part / these /
// twice as many): 16 new tokens over 2000 42 / 14.2 / 18, over 8000 153 / 26.5 /
// 26.9; 200 over 8000 157 / 53 / 63; 600 over 2000 45 / - / 48.5, over 8000 158 / 107
// / 118; 4 x 200 over 700 23.5 / - / 38.6, over 8000 160 / 139 / 136.
WindowPlan plan_window(const WindowArgs& a, int max_context, int cus) {
  WindowPlan p;
  const int G = a.num_heads / a.num_kv_heads;
  const int64_t most = (int64_t)a.max_query * G;  // rows of a (sequence, kv head) pair
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  p.rows = a.block_size != 0 && most <= kWinRowsTile;
  const int tile_rows = p.rows ? kWinRowsTile : 4 * 32;
  p.tiles = (int)((most + tile_rows - 1) / tile_rows);
  const int64_t g = pairs * p.tiles;
  const int64_t n = window_steps(a, max_context, tile_rows, p.rows ? kWinRowsTokens : kWinTileTokens);
  if (p.rows && a.head_size <= 128 && g <= cus) p.waves = 8;
  if (a.block_size == 0 || g == 0) return p;
  int64_t s = cus / g;
  if (p.rows) {
    s = std::min(s, (n + 11) / 12);
    if (n < 24 || (s < 3 && n < 100)) s = 1;
    if (g > cus && g < 2 * cus && n >= 100) s = 3 * g <= 4 * cus ? 3 : 2;
  } else {
    if (n >= 64 && s < 4) s = 2 * cus / g;
    s = std::min({s, (n + 2) / 3, std::max<int64_t>(16, n / 8)});
  }
  p.splits = (int)std::max<int64_t>(1, s);
  return p;
}

size_t window_ws_bytes(const WindowPlan& p, int total_rows, int num_heads, int head_size) {
  if (p.splits == 1) return 0;
  return sizeof(float) * (win_ml_floats(total_rows, num_heads, p.splits) + (size_t)total_rows * num_heads * p.splits * head_size);
}
#endif

}  // namespace dw4
