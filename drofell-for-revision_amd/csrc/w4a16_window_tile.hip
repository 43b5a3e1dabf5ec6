// Windowed attention of many rows: prompts over a paged KV cache, and packed
// sequences whose keys and values are rows beside the queries (training).
//
// A workgroup takes one (sequence, kv head) and 128 rows of it (new tokens x
// query heads of the kv head, token by token, so that all heads of a group read
// a key once); its waves take 32 rows each, as the columns of 32 x 32 x 16
// products, and share steps of 64 tokens through LDS: while one step is worked
// on, the next is copied in (global_load_lds, two stages).
// Scores are formed transposed, S^T = K Q^T, so that a row's scores lie in one
// lane pair, and the probabilities are the B operand of O^T = V^T P^T as they
// stand (w4a16_window_device.h).
//   * cache blocks lie in LDS as in memory, keys [dims / 8][32 tokens][8], values
//     [dims][32 tokens] with the four 16-byte units of a row rotated against
//     bank conflicts;
//   * token rows lie as [token][dims], and values reach the second product
//     through LDS's transposing reads.
// Matrix-core and vector-ALU bound.  Probabilities enter p . v rounded to the
// value type (fp16: of 2^10 p), as the matrix cores take it: their errors are
// independent of each other, and add to the output's own rounding about as much
// again; the sum of the denominator is of the unrounded ones.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "w4a16_device.h"
#include "w4a16_window.h"
#include "w4a16_window_device.h"

namespace dw4 {

namespace {

constexpr int kBk = kWinTileTokens;

// BS: block size of the cache, 0 for token rows.
template <int HS, int BS, bool BF>
__global__ void __launch_bounds__(256, HS <= 128 ? 2 : 1)
window_tile_kernel(WindowArgs a, int tiles, int splits, int padded, float* __restrict__ ws_ml,
                   float* __restrict__ ws_out) {
  constexpr int KD = HS / 16;
  constexpr int ND = (HS + 31) / 32;
  constexpr bool VTAIL = HS % 32 != 0;
  constexpr int NB = BS == 0 ? 1 : kBk / BS;  // blocks of a step
  constexpr int STEPS = 64 / NB;              // steps whose block addresses the lanes hold
  constexpr int SUB = HS * 64;                // bytes of 32 tokens' keys (or values)
  constexpr int STAGE = 4 * SUB;              // keys of 64 tokens, then their values
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];

  if constexpr (BS == 0)
    zero_outside(a.out, a.o_stride, a.num_heads * HS, a.starts, a.num_seqs, a.total_rows, blockIdx.x, padded);
  const int id = xcd_order(blockIdx.x, padded);
  if (id >= a.num_seqs * a.num_kv_heads * tiles * splits) return;
  const int split = id % splits;
  const int tile = tiles - 1 - id / splits % tiles;  // the longest spans first
  const int pair = id / (splits * tiles);
  const int seq = pair / a.num_kv_heads, kvh = pair % a.num_kv_heads;
  const int G = a.num_heads / a.num_kv_heads;
  int q0, q1;
  seq_rows(a.starts, seq, a.total_rows, q0, q1);
  const int n = min(q1 - q0, a.max_query);
  const int rows = n * G, base = tile * 128;
  if (base >= rows) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, half = lane >> 5;
  const int len = BS == 0 ? q1 - q0 : a.lens[seq];
  const int cap = BS == 0 ? len : min(len, a.max_blocks * BS);
  const int p0 = len - (q1 - q0);
  const Span span = Span::of<kBk>(p0 + base / G, p0 + (min(base + 128, rows) - 1) / G, cap, a.window, a.sinks);
  const int per = (span.steps + splits - 1) / splits;
  const int s0 = split * per, s1 = min(span.steps, s0 + per);

  // this wave's rows; those past the last repeat it and are not stored
  const int wbase = base + 32 * wave;
  const int nrows = min(32, rows - wbase);
  const int row = min(wbase + c, rows - 1);
  const int pos = p0 + row / G;
  const int last = min(pos, cap - 1), before = a.window == 0 ? INT32_MIN : pos - a.window;
  const int wfirst = p0 + min(wbase, rows - 1) / G, wlast = p0 + min(wbase + 31, rows - 1) / G;

  // ---- the copies of one step into a stage
  uint64_t kp = 0, vp = 0;  // lane l: block l % NB of step l / NB (of STEPS), 0: not in the table
  auto fetch = [&](int s) {
    kp = vp = 0;
    if (s + lane / NB < s1) {
      const int b = span.token<kBk>(s + lane / NB) / (BS == 0 ? 1 : BS) + lane % NB;
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
  uint32_t held[2] = {(1u << NB) - 1, (1u << NB) - 1};  // by stage: the blocks that are there
  const uint32_t lds0 = lds_offset(lds);
  auto issue = [&](int s, int stage) {
    const uint32_t dst = lds0 + stage * STAGE;
    if constexpr (BS == 0) {
      const int t = span.token<kBk>(s);
      constexpr int UNITS = HS / 8, CHUNKS = kBk * UNITS / 64;
      for (int ch = wave; ch < CHUNKS; ch += 4) {
        const int u = ch * 64 + lane;
        const int r = u / UNITS, at = (u % UNITS) ^ swizzle<HS>(r);
        const int64_t token = q0 + min(t + r, cap - 1);
        const size_t col = (size_t)kvh * HS + at * 8;
        copy16(a.k + token * a.k_stride + col, dst + ch * 1024);
        copy16(a.v + token * a.v_stride + col, dst + 2 * SUB + ch * 1024);
      }
    } else {
      if ((s - s0) % STEPS == 0) fetch(s);
      const int l0 = (s - s0) % STEPS * NB;
      uint32_t there = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b) there |= (uint32_t)(block_of(kp, l0 + b) != 0) << b;
      held[stage] = there;
      constexpr int CHUNKS = SUB / 1024;  // of 64 units, per 32 tokens
      for (int ch = wave; ch < 2 * CHUNKS; ch += 4) {
        const int sub = ch / CHUNKS, u = ch % CHUNKS * 64 + lane;
        const int d = u >> 2, at = (u & 3) ^ ((d >> 2) & 3);  // value row and unit
        if constexpr (BS == 32) {
          const uint64_t kb = block_of(kp, l0 + sub), vb = block_of(vp, l0 + sub);
          if (kb != 0) {
            copy16((const void*)(kb + u * 16), dst + ch * 1024);
            copy16((const void*)(vb + d * 64 + at * 16), dst + 2 * SUB + ch * 1024);
          }
        } else {
          const uint64_t ka = block_of(kp, l0 + 2 * sub), kb = block_of(kp, l0 + 2 * sub + 1);
          const uint64_t va = block_of(vp, l0 + 2 * sub), vb = block_of(vp, l0 + 2 * sub + 1);
          const uint64_t k = u & 16 ? kb : ka, v = at & 2 ? vb : va;
          if (k != 0) copy16((const void*)(k + (u >> 5) * 256 + (u & 15) * 16), dst + ch * 1024);
          if (v != 0) copy16((const void*)(v + d * 32 + (at & 1) * 16), dst + 2 * SUB + ch * 1024);
        }
      }
    }
  };
  auto key = [&](const unsigned char* st, int sub, int kk) {
    if constexpr (BS == 0) return row_unit<HS>(st, 32 * sub + row_token(c), 2 * kk + half);
    else return *(const h8*)(st + sub * SUB + ((2 * kk + half) * 32 + row_token(c)) * 16);
  };
  auto value = [&](const unsigned char* st, int sub, int d, int s) {
    if constexpr (BS == 0) {
      return column_unit<HS>(st + 2 * SUB, 32 * sub + 16 * s, d);
    } else {
      const int dim = VTAIL ? min(32 * d + c, HS - 1) : 32 * d + c;
      return *(const h8*)(st + 2 * SUB + sub * SUB + dim * 64 + (((2 * s + half) ^ ((dim >> 2) & 3)) << 4));
    }
  };

  if (s0 < s1) issue(s0, 0);
  h8 qreg[KD];  // B operand: column c is this lane's row
  {
    const uint16_t* qp = a.q + (size_t)(q0 + row / G) * a.q_stride + (size_t)(kvh * G + row % G) * HS + 8 * half;
#pragma unroll
    for (int j = 0; j < KD; ++j) qreg[j] = *(const h8*)(qp + 16 * j);
  }
  float m = kNoMax, l = 0.f;  // of the row (l: this lane's tokens)
  f16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f16v{};

  for (int step = s0; step < s1; ++step) {
    const int stage = (step - s0) & 1;
    wait_copies();
    if (step + 1 < s1) issue(step + 1, stage ^ 1);
    const int t = span.token<kBk>(step);
    // does the wave see any of it, and all its rows all of it?
    if (nrows <= 0 || t > wlast || (a.window != 0 && t + kBk - 1 <= wfirst - a.window && t >= a.sinks)) continue;
    const bool full = held[stage] == (1u << NB) - 1 && t + kBk - 1 <= min(wfirst, cap - 1) &&
                      (a.window == 0 || t > wlast - a.window || t + kBk - 1 < a.sinks);
    const unsigned char* st = lds + stage * STAGE;
    f16v s[2] = {f16v{}, f16v{}};
#pragma unroll
    for (int j = 0; j < KD; ++j)
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = mfma32_of<BF>(key(st, b, j), qreg[j], s[b]);
    auto visible = [&](int b, int e) {  // of score e of the 32 tokens b
      const int in = 32 * b + 16 * (e >> 3) + 8 * half + (e & 7);
      const bool there = BS == 0 || ((held[stage] >> (BS == 32 ? b : 2 * b + (e >> 3))) & 1);
      return there && sees(t + in, last, before, a.sinks);
    };
    if (!full) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[b][e] = visible(b, e) ? s[b][e] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) mx = fmaxf(mx, s[e >> 4][e & 15]);
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
    h8 p[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = __builtin_amdgcn_exp2f(fmaf(s[b][8 * g + 2 * e], a.scale_log2, shift));
          const float z = __builtin_amdgcn_exp2f(fmaf(s[b][8 * g + 2 * e + 1], a.scale_log2, shift));
          l += y;
          l += z;
          x[e] = pack2<BF>(y, z);
        }
        p[b][g] = __builtin_bit_cast(h8, x);
      }
    if (full) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d] = mfma32_of<BF>(value(st, b, d, g), p[b][g], o[d]);
    } else {
      // a value that some rows do not see (or that no row does) must not reach
      // them as 0 * inf: where there is one, its part is added apart
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        h8 v[2][2];
        bool odd = false;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            v[b][g] = value(st, b, d, g);
            odd |= any_nonfinite<BF>(v[b][g]);
          }
        if (__any(odd)) {
          f16v up = {}, down = {};
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              u4 w;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t one = BF ? 0x3F80u : 0x3C00u;
                w[e] = (visible(b, 8 * g + 2 * e) ? one : 0u) | (visible(b, 8 * g + 2 * e + 1) ? one << 16 : 0u);
              }
              h8 pn, nn;
              split_nonfinite<BF>(v[b][g], pn, nn);
              up = mfma32_of<BF>(pn, __builtin_bit_cast(h8, w), up);
              down = mfma32_of<BF>(nn, __builtin_bit_cast(h8, w), down);
            }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (up[e] > 0.f) o[d][e] += INFINITY;
            if (down[e] > 0.f) o[d][e] -= INFINITY;
          }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int g = 0; g < 2; ++g) o[d] = mfma32_of<BF>(v[b][g], p[b][g], o[d]);
      }
    }
  }

  l = both_sum(l);
  if (c >= nrows) return;
  const int token = q0 + row / G, head = kvh * G + row % G;
  if (splits == 1) {
    const float f = l == 0.f ? 1.f : 1.f / l;  // no visible token: zeros
    uint16_t* op = a.out + (size_t)token * a.o_stride + (size_t)head * HS;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int dim = d * 32 + 2 * e + 4 * half;
        if (!VTAIL || dim < HS)
          *(uint2*)(op + dim) = make_uint2(pack2<BF>(o[d][e] * f, o[d][e + 1] * f),
                                           pack2<BF>(o[d][e + 2] * f, o[d][e + 3] * f));
      }
    if (a.lse != nullptr && half == 0)
      a.lse[(size_t)token * a.num_heads + head] = m + __builtin_amdgcn_logf(l) - p_shift<BF>();
  } else {
    const size_t slot = ((size_t)token * a.num_heads + head) * splits + split;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int dim = d * 32 + 2 * e + 4 * half;
        if (!VTAIL || dim < HS)
          *(f4*)(ws_out + slot * HS + dim) = f4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
      }
    if (half == 0) {
      ws_ml[2 * slot] = m;
      ws_ml[2 * slot + 1] = l;
    }
  }
}

template <int HS, int BS, bool BF>
hipError_t launch_tile_bs(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  auto kern = &window_tile_kernel<HS, BS, BF>;
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(kern), win_tile_smem(HS), done);
  if (e != hipSuccess) return e;
  const int total = a.num_seqs * a.num_kv_heads * p.tiles * p.splits, padded = (total + 7) / 8 * 8;
  kern<<<(unsigned)padded, 256, win_tile_smem(HS), stream>>>(
      a, p.tiles, p.splits, padded, ws, ws + 2 * (size_t)a.total_rows * a.num_heads * p.splits);
  return hipGetLastError();
}

template <int HS, bool BF>
hipError_t launch_tile_hs(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream) {
  if (a.block_size == 16) return launch_tile_bs<HS, 16, BF>(a, p, ws, stream);
  if (a.block_size == 32) return launch_tile_bs<HS, 32, BF>(a, p, ws, stream);
  return launch_tile_bs<HS, 0, BF>(a, p, ws, stream);
}

}  // namespace

template <bool BF>
hipError_t launch_window_tile(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream) {
  switch (a.head_size) {
    case 64: return launch_tile_hs<64, BF>(a, p, ws, stream);
    case 80: return launch_tile_hs<80, BF>(a, p, ws, stream);
    case 96: return launch_tile_hs<96, BF>(a, p, ws, stream);
    case 112: return launch_tile_hs<112, BF>(a, p, ws, stream);
    case 128: return launch_tile_hs<128, BF>(a, p, ws, stream);
    case 256: return launch_tile_hs<256, BF>(a, p, ws, stream);
    default: return hipErrorInvalidValue;
  }
}
template hipError_t launch_window_tile<WINDOW_BF16>(const WindowArgs&, const WindowPlan&, float*, hipStream_t);

}  // namespace dw4
