// Gradients of windowed attention over packed sequences (training).
//
// With P the probabilities, dO the output's gradient and c the scale:
//   delta_i = dO_i . O_i          dV_j = sum_i P_ij dO_i
//   dS_ij   = P_ij (dO_i . V_j - delta_i)
//   dQ_i = c sum_j dS_ij K_j      dK_j = c sum_i dS_ij Q_i
// P is formed again from the forward's log-sums.  Two kernels, seven products (nine,
// dS being in two parts) where one pass with atomic sums would need five, so that every sum has one
// order and results repeat bit for bit:
//   * window_dq_kernel: as the forward, 128 rows (tokens x query heads of a kv
//     head) of a workgroup, steps of 64 tokens through LDS; it writes delta too;
//   * window_dkv_kernel: 128 tokens of a workgroup, a wave's 32 as the columns
//     of its products, steps of 32 rows through LDS; the heads of a group are
//     rows like any others, so that shared heads' gradients add up in registers.
//     The tokens' values stay in LDS beside the steps, which leaves registers
//     for two waves per SIMD (1003 us when that was measured against one wave, with
//     steps of 64 rows and the values in registers, 1372 us; sizes as below).
// Both read a tile from LDS in both directions, rows in plain and columns in
// transposing reads.  Bound by matrix cores and vector ALU together, as the forward
// (busy 48 and 42 % of the cycles in dq, 44 and 34 % in dkv, whose copies cost 10 %:
// registers do not reach for issuing them among its products).  Measured, for
// sequences of 6000 and 4100 tokens, 32 heads of 128, window 2048, bf16 (0.155 TFLOP a
// product): dq 700 us for its four products (dS in two parts), dkv 955 us for its
// five, 0.89 and 0.81 PFLOP/s; fp16 756 and 1076 us.
//
// Roundings: P enters its product in 16 bits, as the matrix cores take it, with
// independent errors.  dS, whose errors would add up with those of delta, enters
// as two 16-bit parts, over operands that are in registers already, and delta
// sums the forward's output and what its rounding left off.  (With one part
// and the rounded output alone dq and dk were 1.7 times as far from float64 as their
// own rounding is.)  What is left of delta's error, from the forward's 16-bit
// probabilities, is seen in a row's dS, whose sum over the tokens is zero: dq takes
// the sum off again, by the probabilities of the row's last tokens, and dkv gets delta
// with it.  (Else keys that share a vector, 8 times what tells them apart, put dq 7
// times its rounding off; so it is 1.0 to 1.4 times, 1 to 2 % of the pass dearer.)
// fp16 holds neither small probabilities nor small or large gradients, so P goes in
// as 2^10 P and dS times a power of two per row (dq) or token (dkv) that follows the
// largest of what it is summed from (keep_in_range()); bf16 needs neither.
// A sequence's non-finite values may reach any gradient of that sequence.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "w4a16_device.h"
#include "w4a16_window.h"
#include "w4a16_window_device.h"

namespace dw4 {

namespace {

constexpr int kBk = kWinTileTokens;
constexpr int kGradTile = 128;  // rows of a dq workgroup, tokens of a dkv workgroup

// fp16: the factors dO . V - delta of a step (of this lane's column: a row in dq, a token in
// dkv) times a power of two that keeps the largest so far at MOST / 16 or above and at MOST
// or below, and with them the sums, as a softmax keeps its running maximum: nothing
// overflows, and nothing that counts beside the largest is lost, whatever the sizes of dO
// and V.  (The largest of the factors, not of dS = P times them, which a P <= 1 only makes
// smaller: it is known before the exponentials are.  A power of two from |dO| alone, which takes
// no step's time, overflowed at coherent values and lost small gradients beside large ones;
// this costs 2 % of fp16 training with heads of 128, 2 x 6000 tokens, 4 % with heads of 64, 3 %
// with heads of 256.)
constexpr float kFirstScale = 0x1p100f;
template <int MOST, int ND>
__device__ __forceinline__ void keep_in_range(float (&v)[16], float& scale, f16v (&sums)[ND], float& total) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(v[e]));
  if (__any(top * scale > (float)(1 << MOST))) {
    top = both_max(top);
    const float to = top * scale > (float)(1 << MOST) ? __builtin_amdgcn_ldexpf(1.f, MOST - 3 - __builtin_amdgcn_frexp_expf(top)) : scale;
    const float f = __builtin_amdgcn_ldexpf(to, 1 - __builtin_amdgcn_frexp_expf(scale));  // to / scale, powers of two
#pragma unroll
    for (int d = 0; d < ND; ++d) sums[d] *= f;
    total *= f;
    scale = to;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] *= scale;
}

// sum of x (y + z)
template <bool BF>
__device__ __forceinline__ void dot8(u4 x, u4 y, u4 z, float& sum) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int h = 0; h < 2; ++h) sum = fmaf(unpack<BF>(x[e], h), unpack<BF>(y[e], h) + unpack<BF>(z[e], h), sum);
}

// Eight values as an operand, and what its rounding leaves off as another.
template <bool BF>
__device__ __forceinline__ void two_parts(const float* v, h8& hi, h8& lo) {
  u4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = pack2<BF>(v[2 * e], v[2 * e + 1]);
    l[e] = pack2<BF>(v[2 * e] - unpack<BF>(h[e], 0), v[2 * e + 1] - unpack<BF>(h[e], 1));
  }
  hi = __builtin_bit_cast(h8, h);
  lo = __builtin_bit_cast(h8, l);
}

template <int HS, bool BF>
__global__ void __launch_bounds__(256, HS <= 128 ? 2 : 1)
window_dq_kernel(WindowGradArgs g, int tiles, float* __restrict__ delta) {
  constexpr int KD = HS / 16, ND = (HS + 31) / 32;
  constexpr bool VTAIL = HS % 32 != 0;
  constexpr int TILE = row_at<HS>(kBk), STAGE = 2 * TILE;  // keys, values
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const WindowArgs& a = g.f;
  zero_outside(g.dq, g.dq_stride, a.num_heads * HS, a.starts, a.num_seqs, a.total_rows, blockIdx.x, gridDim.x);
  int pair, tile;
  if (!work_of(blockIdx.x, a.num_seqs * a.num_kv_heads, tiles, pair, tile)) return;
  tile = tiles - 1 - tile;
  const int seq = pair / a.num_kv_heads, kvh = pair % a.num_kv_heads;
  const int G = a.num_heads / a.num_kv_heads;
  int q0, q1;
  seq_rows(a.starts, seq, a.total_rows, q0, q1);
  const int n = min(q1 - q0, a.max_query);
  const int rows = n * G, base = tile * kGradTile;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  zero_beyond(g.dq + (size_t)kvh * G * HS, g.dq_stride, G * HS, q0 + n, q1, tile, tiles);
  if (base >= rows) return;
  const int c = lane & 31, half = lane >> 5;
  const Span span = Span::of<kBk>(base / G, (min(base + kGradTile, rows) - 1) / G, n, a.window, a.sinks);
  const int wbase = base + 32 * wave;
  const int nrows = min(32, rows - wbase);
  const int row = min(wbase + c, rows - 1);
  const int pos = row / G, before = a.window == 0 ? INT32_MIN : pos - a.window;
  const int wfirst = min(wbase, rows - 1) / G, wlast = min(wbase + 31, rows - 1) / G;
  const int token = q0 + pos, head = kvh * G + row % G;

  const uint32_t lds0 = lds_offset(lds);
  const bool near = a.k_stride <= kNearRows && a.v_stride <= kNearRows;
  // a step's copies, PARTS per wave, go out among the products of the one before
  // (at once they would hold up the wave); the last tokens' in one go, bounded
  constexpr int UNITS = HS / 8, CHUNKS = kBk * UNITS / 64, PARTS = (CHUNKS + 3) / 4 * 2;
  uint64_t next_k = 0, next_v = 0;
  uint32_t next_dst = 0;
  auto part = [&](int i) {
    const int ch = wave + 4 * (i >> 1);
    if (CHUNKS % 4 != 0 && ch >= CHUNKS) return;
    const int u = ch * 64 + lane;
    const uint32_t r = u / UNITS, at = ((u % UNITS) ^ swizzle<HS>(r)) * 16;
    if (i & 1) copy16(next_v, r * (uint32_t)(a.v_stride * 2) + at, next_dst + TILE + chunk_at<HS>(ch));
    else copy16(next_k, r * (uint32_t)(a.k_stride * 2) + at, next_dst + chunk_at<HS>(ch));
  };
  auto next_step = [&](int s, int stage) {  // whether part() is to copy it
    next_dst = lds0 + stage * STAGE;
    const int t = span.token<kBk>(s);
    if (near && t + kBk <= n) {
      const size_t col = (size_t)kvh * HS;
      next_k = (uint64_t)(a.k + (size_t)(q0 + t) * a.k_stride + col);
      next_v = (uint64_t)(a.v + (size_t)(q0 + t) * a.v_stride + col);
      return true;
    }
    for (int ch = wave; ch < CHUNKS; ch += 4) {
      const int u = ch * 64 + lane;
      const int r = u / UNITS, at = (u % UNITS) ^ swizzle<HS>(r);
      const int64_t tok = q0 + min(t + r, n - 1);
      const size_t col = (size_t)kvh * HS + at * 8;
      copy16(a.k + tok * a.k_stride + col, next_dst + chunk_at<HS>(ch));
      copy16(a.v + tok * a.v_stride + col, next_dst + TILE + chunk_at<HS>(ch));
    }
    return false;
  };
  if (span.steps > 0 && next_step(0, 0)) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) part(i);
  }
  h8 qreg[KD], oreg[KD];  // B operands: this row of Q and of dO
  float dl = 0.f;
  {
    const size_t col = (size_t)head * HS + 8 * half;
    const uint16_t* qp = a.q + (size_t)token * a.q_stride + col;
    const uint16_t* dp = g.dout + (size_t)token * g.do_stride + col;
    const uint16_t* op = a.out + (size_t)token * a.o_stride + col;
    const uint16_t* rp = a.rest + (size_t)token * a.num_heads * HS + col;
#pragma unroll
    for (int j = 0; j < KD; ++j) {
      qreg[j] = *(const h8*)(qp + 16 * j);
      oreg[j] = *(const h8*)(dp + 16 * j);
      dot8<BF>(__builtin_bit_cast(u4, oreg[j]), *(const u4*)(op + 16 * j), *(const u4*)(rp + 16 * j), dl);
    }
  }
  dl = both_sum(dl);
  const float lse = a.lse[(size_t)token * a.num_heads + head];
  float gs = BF ? 1.f : kFirstScale, total = 0.f;  // total: of this lane's dS

  wait_loads();
  f16v dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = f16v{};
  for (int step = 0; step < span.steps; ++step) {
    wait_copies();
    bool copies = step + 1 < span.steps && next_step(step + 1, (step + 1) & 1);
    const int t = span.token<kBk>(step);
    const unsigned char* st = lds + (step & 1) * STAGE;
    for (int b = 0; b < 2; ++b) {
      const int tb = t + 32 * b;
      if (nrows <= 0 || tb > wlast || (a.window != 0 && tb + 31 <= wfirst - a.window && tb >= a.sinks)) continue;
      const bool full = tb + 31 < wfirst && (a.window == 0 || tb > wlast - a.window || tb + 31 < a.sinks);
      f16v s = {}, p = {};
      auto products = [&](auto with) {
        feed<2 * KD, 6>(
            [&](int i) { return row_unit<HS>(st + (i & 1) * TILE + row_at<HS>(32 * b), row_token(c), (i & ~1) + half); },
            [&](int i, h8 f) {
              if (i & 1) p = mfma32_of<BF>(f, oreg[i >> 1], p);
              else s = mfma32_of<BF>(f, qreg[i >> 1], s);
              if constexpr (decltype(with)::value) {
#pragma unroll
                for (int k = i * PARTS / (2 * KD); k < (i + 1) * PARTS / (2 * KD); ++k) part(k);
              }
            });
      };
      if (copies) products(std::true_type{});
      else products(std::false_type{});
      copies = false;
      float pr[16], ds[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        pr[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -lse));
        ds[e] = p[e] - dl;
      }
      if constexpr (!BF) keep_in_range<15>(ds, gs, dq, total);
#pragma unroll
      for (int e = 0; e < 16; ++e) ds[e] *= pr[e];
      if (!full) {
        const uint32_t seen = own_scores(seen_of(tb, pos, before, a.sinks), half);
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] = where_seen(seen, e, ds[e], 0.f);
      }
#pragma unroll
      for (int e = 0; e < 16; e += 4) total += (ds[e] + ds[e + 1]) + (ds[e + 2] + ds[e + 3]);
      // Some rows' own tokens, their last, are among these (`full` leaves them out): what all
      // their dS sum to is known.  (Not by parts of a softmax below 2^-40.)
      if (tb + 31 >= wfirst) {
        const uint32_t seen = own_scores(seen_of(tb, pos, before, a.sinks), half);
        float own = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) own += where_seen(seen, e, pr[e], 0.f);
        own = both_sum(own);
        const float left = both_sum(total), r = pos >= tb && pos < tb + 32 && own > 0x1p-40f ? left / own : 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] = fmaf(-r, where_seen(seen, e, pr[e], 0.f), ds[e]);
      }
      h8 hi[2], lo[2];
      two_parts<BF>(ds, hi[0], lo[0]);
      two_parts<BF>(ds + 8, hi[1], lo[1]);
      feed<2 * ND, 6>([&](int i) { return column_unit<HS>(st, 32 * b + 16 * (i / ND), i % ND); },
                      [&](int i, h8 f) {
                        dq[i % ND] = mfma32_of<BF>(f, hi[i / ND], dq[i % ND]);
                        dq[i % ND] = mfma32_of<BF>(f, lo[i / ND], dq[i % ND]);
                      });
    }
    if (copies) {  // the wave sees nothing of this step
#pragma unroll
      for (int i = 0; i < PARTS; ++i) part(i);
    }
  }
  total = both_sum(total);
  const int thread = thread_again(), col = thread & 31, hi = thread >> 5 & 1;
  if (col >= nrows) return;
  const int own = wbase + col, at = q0 + own / G, to = kvh * G + own % G;
  if (hi == 0) delta[(size_t)at * a.num_heads + to] = dl + total / gs;
  const float f = g.scale / gs;
  uint16_t* out = g.dq + (size_t)at * g.dq_stride + (size_t)to * HS;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int dim = d * 32 + 2 * e + 4 * hi;
      if (!VTAIL || dim < HS)
        *(uint2*)(out + dim) = make_uint2(pack2<BF>(dq[d][e] * f, dq[d][e + 1] * f),
                                          pack2<BF>(dq[d][e + 2] * f, dq[d][e + 3] * f));
    }
}

// Token of a row (row / G), by the magic ceil(2^32 / G).  The product's quotient is one
// too large for the last rows of far tokens (rows times the magic's excess, up to G - 1,
// pass 2^32: with 1023 heads from token 4120 on, with 77 from 764093), never more, which
// the product back tells.
__device__ __forceinline__ int token_of(int row, int G, uint32_t magic) {
  const int i = div_by_magic(row, magic);
  return i * G > row ? i - 1 : i;
}

// Floats of a workspace part, whole 16-byte units.
constexpr size_t grad_rows(size_t a, size_t b) { return (a * b + 3) / 4 * 4; }

// The row steps (of kDkvRows rows) of a tile of tokens are split into parts where
// that many workgroups are wanted: sink tiles, which a window does not bound, by
// `sink_parts`, the others by `parts`.  Items of a pair: the sink tiles' parts, then
// the other tiles'.
struct DkvPlan {
  int tiles, sink_tiles, parts, sink_parts;
  __host__ __device__ int items() const { return sink_tiles * sink_parts + (tiles - sink_tiles) * parts; }
  // Items of a pair that are parts, the first ones (sink_parts >= parts): they leave sums in the workspace.
  __host__ __device__ int partial_items() const { return parts > 1 ? items() : sink_parts > 1 ? sink_tiles * sink_parts : 0; }
};
constexpr int kDkvRows = 32;

template <int HS, bool BF>
__global__ void __launch_bounds__(256, HS <= 128 ? 2 : 1)
window_dkv_kernel(WindowGradArgs g, DkvPlan plan, uint32_t magic, const float* __restrict__ delta,
                  float* __restrict__ partial) {
  constexpr int KD = HS / 16, ND = (HS + 31) / 32;
  constexpr bool VTAIL = HS % 32 != 0;
  constexpr int AHEAD = HS <= 96 ? 3 : 2;  // operands in flight (registers)
  constexpr int TILE = row_at<HS>(kDkvRows);
  constexpr int STAGE = 2 * TILE + 3 * kDkvRows * 4;  // rows of Q and of dO, log-sums, deltas, positions
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  unsigned char* const vtile = lds + 2 * STAGE;  // the tokens' values [128][HS]
  const WindowArgs& a = g.f;
  zero_outside(g.dk, g.dk_stride, a.num_kv_heads * HS, a.starts, a.num_seqs, a.total_rows, blockIdx.x, gridDim.x);
  zero_outside(g.dv, g.dv_stride, a.num_kv_heads * HS, a.starts, a.num_seqs, a.total_rows, blockIdx.x, gridDim.x);
  int pair, item;
  if (!work_of(blockIdx.x, a.num_seqs * a.num_kv_heads, plan.items(), pair, item)) return;
  const int far = plan.sink_tiles * plan.sink_parts;
  const int parts = item < far ? plan.sink_parts : plan.parts;
  const int tile = item < far ? item / parts : plan.sink_tiles + (item - far) / parts;
  const int part = item < far ? item % parts : (item - far) % parts;
  const int seq = pair / a.num_kv_heads, kvh = pair % a.num_kv_heads;
  const int G = a.num_heads / a.num_kv_heads;
  int q0, q1;
  seq_rows(a.starts, seq, a.total_rows, q0, q1);
  const int n = min(q1 - q0, a.max_query);
  const int t0 = tile * kGradTile;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  zero_beyond(g.dk + (size_t)kvh * HS, g.dk_stride, HS, q0 + n, q1, item, plan.items());
  zero_beyond(g.dv + (size_t)kvh * HS, g.dv_stride, HS, q0 + n, q1, item, plan.items());
  if (t0 >= n) return;
  const int c = lane & 31, half = lane >> 5;
  // rows that see a token of the tile, and this part of them
  const int64_t reach = a.window == 0 || t0 < a.sinks ? n : (int64_t)t0 + kGradTile - 1 + a.window;
  const int r0 = t0 * G, r1 = (int)min<int64_t>(n, reach) * G;
  const int all = (r1 - r0 + kDkvRows - 1) / kDkvRows, per = (all + parts - 1) / parts;
  const int s0 = part * per, s1 = min(all, s0 + per);
  const int wa = t0 + 32 * wave, wb = min(wa + 31, n - 1);  // this wave's tokens
  const int tk = min(wa + c, n - 1);

  const uint32_t lds0 = lds_offset(lds);
  constexpr int UNITS = HS / 8;
  const int log_g = 31 - __builtin_clz(G);
  const bool near = kDkvRows % G == 0 && a.q_stride <= kNearRows && g.do_stride <= kNearRows;
  constexpr int CHUNKS = kDkvRows * UNITS / 64, TURNS = (CHUNKS + 3) / 4;
  // Whole tokens' rows (G divides a step's): uniform addresses that advance by the step,
  // and one offset per lane; a wave's turns are 256 units apart, whole rows where a row
  // is a power of two.
  const uint64_t q_first = (uint64_t)(a.q + (size_t)(q0 + t0) * a.q_stride + (size_t)kvh * G * HS);
  const uint64_t o_first = (uint64_t)(g.dout + (size_t)(q0 + t0) * g.do_stride + (size_t)kvh * G * HS);
  const uint64_t l_first = (uint64_t)((wave == 0 ? a.lse : delta) + (size_t)(q0 + t0) * a.num_heads + kvh * G);
  auto issue = [&](int s, int stage) {
    const uint32_t dst = lds0 + stage * STAGE;
    if (near && r0 + (s + 1) * kDkvRows <= r1) {
      const uint32_t tokens = (uint32_t)(s * kDkvRows) >> log_g, q2 = (uint32_t)(a.q_stride * 2), o2 = (uint32_t)(g.do_stride * 2);
      const uint64_t qb = q_first + (uint64_t)tokens * q2, ob = o_first + (uint64_t)tokens * o2;
      constexpr bool EVEN = 256 % UNITS == 0;
      const int l = BF || HS != 128 ? lane : thread_again() & 63;  // (fp16's powers of two leave no register for offsets)
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int ch = wave + 4 * i;
        if (CHUNKS % 4 != 0 && ch >= CHUNKS) break;
        const int u = (EVEN ? wave : ch) * 64 + l, rows = EVEN ? i * (256 / UNITS) : 0;
        const uint32_t r = u / UNITS, at = ((u % UNITS) ^ swizzle<HS>(r)) * 16 + (r & (G - 1)) * (HS * 2);
        const uint32_t on = (rows & (G - 1)) * (HS * 2), by = (uint32_t)rows >> log_g;
        copy16(qb + on + by * q2, (r >> log_g) * q2 + at, dst + chunk_at<HS>(ch));
        copy16(ob + on + by * o2, (r >> log_g) * o2 + at, dst + TILE + chunk_at<HS>(ch));
      }
      if (wave < 3 && l < kDkvRows) {
        const uint32_t off = ((l >> log_g) * a.num_heads + (l & (G - 1))) * 4;
        if (wave == 2) *(int*)(lds + stage * STAGE + 2 * TILE + 2 * kDkvRows * 4 + l * 4) = t0 + tokens + (l >> log_g);
        else copy4(l_first + 4 * (uint64_t)tokens * a.num_heads, off, dst + 2 * TILE + wave * kDkvRows * 4);
      }
      return;
    }
    for (int ch = wave; ch < CHUNKS; ch += 4) {
      const int u = ch * 64 + lane;
      const int r = u / UNITS, at = (u % UNITS) ^ swizzle<HS>(r);
      const int row = min(r0 + s * kDkvRows + r, r1 - 1), i = token_of(row, G, magic);
      const size_t col = (size_t)(kvh * G + row - i * G) * HS + at * 8;
      copy16(a.q + (size_t)(q0 + i) * a.q_stride + col, dst + chunk_at<HS>(ch));
      copy16(g.dout + (size_t)(q0 + i) * g.do_stride + col, dst + TILE + chunk_at<HS>(ch));
    }
    if (wave < 3 && lane < kDkvRows) {
      const int row = r0 + s * kDkvRows + lane, in = min(row, r1 - 1), i = token_of(in, G, magic);
      const size_t at = (size_t)(q0 + i) * a.num_heads + kvh * G + in - i * G;
      if (wave == 0) copy4(a.lse + at, dst + 2 * TILE);
      else if (wave == 1) copy4(delta + at, dst + 2 * TILE + kDkvRows * 4);
      else *(int*)(lds + stage * STAGE + 2 * TILE + 2 * kDkvRows * 4 + lane * 4) = row < r1 ? i : -1;
    }
  };
  if (s0 < s1) issue(s0, 0);
  for (int ch = wave; s0 < s1 && ch < kGradTile * UNITS / 64; ch += 4) {
    const int u = ch * 64 + lane;
    const int r = u / UNITS, at = (u % UNITS) ^ swizzle<HS>(r);
    copy16(a.v + (size_t)(q0 + min(t0 + r, n - 1)) * a.v_stride + (size_t)kvh * HS + at * 8,
           lds0 + 2 * STAGE + chunk_at<HS>(ch));
  }
  h8 kreg[KD];  // B operand: this token's key
  {
    const uint16_t* kp = a.k + (size_t)(q0 + tk) * a.k_stride + (size_t)kvh * HS + 8 * half;
#pragma unroll
    for (int j = 0; j < KD; ++j) kreg[j] = *(const h8*)(kp + 16 * j);
  }
  const float ps = p_shift<BF>();
  float gs = BF ? 1.f : kFirstScale;  // of 2^ps dS

  wait_loads();
  f16v dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f16v{};
  for (int step = s0; step < s1; ++step) {
    const int stage = (step - s0) & 1;
    wait_copies();
    if (step + 1 < s1) issue(step + 1, stage ^ 1);
    const unsigned char* st = lds + stage * STAGE;
    const int ra = r0 + step * kDkvRows;
    const int ia = token_of(ra, G, magic), ib = token_of(min(ra + kDkvRows, r1) - 1, G, magic);
    if (wa >= n || ib < wa || (a.window != 0 && ia - a.window >= wb && wa >= a.sinks)) continue;
    const bool full = ra + kDkvRows <= r1 && ia >= wb && (a.window == 0 || ib < wa + a.window || wb < a.sinks);
    f16v s = {}, p = {};
    struct Operands {
      h8 q, o, v;
    };
    feed<KD, AHEAD>(
        [&](int j) {
          return Operands{row_unit<HS>(st, row_token(c), 2 * j + half), row_unit<HS>(st + TILE, row_token(c), 2 * j + half),
                          row_unit<HS>(vtile + row_at<HS>(32 * wave), c, 2 * j + half)};
        },
        [&](int j, const Operands& f) {
          s = mfma32_of<BF>(f.q, kreg[j], s);
          p = mfma32_of<BF>(f.o, f.v, p);
        });
    h8 pw[2], hi[2], lo[2];
    float pr[16], ds[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float* ls = (const float*)(st + 2 * TILE) + 16 * (e / 8) + 8 * half + e % 8;  // of the lane's rows
      pr[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, ps - ls[0]));
      ds[e] = p[e] - ls[kDkvRows];
    }
    float none = 0.f;
    if constexpr (!BF) keep_in_range<5>(ds, gs, dk, none);
#pragma unroll
    for (int e = 0; e < 16; ++e) ds[e] *= pr[e];
    if (!full) {
      const int own = wa + (thread_again() & 31);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = ((const int*)(st + 2 * TILE))[2 * kDkvRows + 16 * (e / 8) + 8 * half + e % 8];
        const bool seen = sees(own, i, a.window == 0 ? INT32_MIN : i - a.window, i < 0 ? 0 : a.sinks);
        pr[e] = seen ? pr[e] : 0.f;
        ds[e] = seen ? ds[e] : 0.f;
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float* v = pr + 8 * x;
      pw[x] = __builtin_bit_cast(h8, u4{pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3]), pack2<BF>(v[4], v[5]), pack2<BF>(v[6], v[7])});
      two_parts<BF>(ds + 8 * x, hi[x], lo[x]);
    }
    feed<4 * ND, 6>(  // of each 16 rows and 32 dims: dO, then Q
        [&](int i) { return column_unit<HS>(st + (1 - (i & 1)) * TILE, 16 * (i / (2 * ND)), i / 2 % ND); },
        [&](int i, h8 f) {
          const int x = i / (2 * ND), d = i / 2 % ND;
          if (i & 1) {
            dk[d] = mfma32_of<BF>(f, hi[x], dk[d]);
            dk[d] = mfma32_of<BF>(f, lo[x], dk[d]);
          } else {
            dv[d] = mfma32_of<BF>(f, pw[x], dv[d]);
          }
        });
  }
  const int thread = HS <= 128 ? thread_again() : (int)threadIdx.x, col = thread & 31, hi = thread >> 5 & 1, token = wa + col;
  if (token >= n) return;
  const float fv = __builtin_amdgcn_exp2f(-ps), fk = g.scale * fv / gs;
  uint16_t* ok = g.dk + (size_t)(q0 + token) * g.dk_stride + (size_t)kvh * HS;
  uint16_t* ov = g.dv + (size_t)(q0 + token) * g.dv_stride + (size_t)kvh * HS;
  float* pk = partial + (((size_t)pair * plan.partial_items() + item) * kGradTile + 32 * wave + col) * (2 * HS);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int dim = d * 32 + 2 * e + 4 * hi;
      if (VTAIL && dim >= HS) continue;
      const f4 x = f4{dk[d][e], dk[d][e + 1], dk[d][e + 2], dk[d][e + 3]} * fk;
      const f4 y = f4{dv[d][e], dv[d][e + 1], dv[d][e + 2], dv[d][e + 3]} * fv;
      if (parts == 1) {
        *(uint2*)(ok + dim) = make_uint2(pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]));
        *(uint2*)(ov + dim) = make_uint2(pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3]));
      } else {
        *(f4*)(pk + dim) = x;
        *(f4*)(pk + HS + dim) = y;
      }
    }
}

// The parts of a tile summed in their order, four dims per thread.  Launch-bound where
// parts are made (few tiles): 4 us for five sequences of 333 tokens, 4 kv heads of 80.
template <int HS, bool BF>
__global__ void __launch_bounds__(256)
window_dkv_join_kernel(WindowGradArgs g, DkvPlan plan, int tiles, const float* __restrict__ partial) {
  const WindowArgs& a = g.f;
  constexpr int PER = kGradTile * (2 * HS / 4) / 256;  // workgroups of 256 units per tile
  const int chunk = blockIdx.x % PER, tile = blockIdx.x / PER % tiles, pair = blockIdx.x / PER / tiles;
  const int parts = tile < plan.sink_tiles ? plan.sink_parts : plan.parts;
  if (parts == 1) return;
  const int item = tile < plan.sink_tiles ? tile * parts : plan.sink_tiles * plan.sink_parts + (tile - plan.sink_tiles) * parts;
  const int seq = pair / a.num_kv_heads, kvh = pair % a.num_kv_heads;
  int q0, q1;
  seq_rows(a.starts, seq, a.total_rows, q0, q1);
  const int u = chunk * 256 + threadIdx.x, t = u / (2 * HS / 4), dim = u % (2 * HS / 4) * 4;
  const int token = tile * kGradTile + t;
  if (token >= min(q1 - q0, a.max_query)) return;
  const float* src = partial + (((size_t)pair * plan.partial_items() + item) * kGradTile + t) * (2 * HS) + dim;
  f4 sum = {};
  for (int p = 0; p < parts; ++p) sum += *(const f4*)(src + (size_t)p * kGradTile * (2 * HS));
  uint16_t* out = dim < HS ? g.dk + (size_t)(q0 + token) * g.dk_stride + (size_t)kvh * HS + dim
                           : g.dv + (size_t)(q0 + token) * g.dv_stride + (size_t)kvh * HS + dim - HS;
  *(uint2*)out = make_uint2(pack2<BF>(sum[0], sum[1]), pack2<BF>(sum[2], sum[3]));
}

// Tiles of tokens split into parts: all of them where they leave more than half
// of the CUs (two workgroups each) without one, down to eight steps a part; sink
// tiles, whose rows a window does not bound, to about twice a bounded tile's rows, or
// until their parts, which go first, fill every CU once: more would only cost workspace.
DkvPlan plan_dkv(const WindowArgs& a, int cus) {
  DkvPlan p = {};
  const int64_t G = a.num_heads / a.num_kv_heads, pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  p.tiles = (a.max_query + kGradTile - 1) / kGradTile;
  const int64_t bound = a.window == 0 ? a.max_query : std::min<int64_t>(a.max_query, (int64_t)a.window + kGradTile);
  const int64_t steps = (bound * G + kDkvRows - 1) / kDkvRows;
  p.parts = 1;
  if (pairs * p.tiles <= cus) p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(2 * cus / (pairs * p.tiles), steps / 8));
  p.sink_tiles = a.window == 0 ? 0 : (int)std::min<int64_t>(p.tiles, ((int64_t)a.sinks + kGradTile - 1) / kGradTile);
  p.sink_parts = p.parts;
  if (p.sink_tiles > 0 && a.max_query >= 3 * bound)
    p.sink_parts = (int)std::max<int64_t>(p.parts, std::min({(int64_t)64, a.max_query / (2 * bound) * p.parts, 2 * cus / (pairs * p.sink_tiles)}));
  return p;
}

template <int HS, bool BF>
hipError_t launch_grad_hs(const WindowGradArgs& g, float* ws, hipStream_t stream) {
  static std::atomic<uint64_t> done_q{0}, done_kv{0};
  const WindowArgs& a = g.f;
  const int G = a.num_heads / a.num_kv_heads;
  const size_t smem = 4 * row_at<HS>(kBk);
  const size_t smem_kv = 2 * (2 * row_at<HS>(kDkvRows) + 3 * kDkvRows * 4) + row_at<HS>(kGradTile);
  auto dq = &window_dq_kernel<HS, BF>;
  auto dkv = &window_dkv_kernel<HS, BF>;
  hipError_t e = allow_lds(reinterpret_cast<const void*>(dq), smem, done_q);
  if (e == hipSuccess) e = allow_lds(reinterpret_cast<const void*>(dkv), smem_kv, done_kv);
  if (e != hipSuccess) return e;
  const int pairs = a.num_seqs * a.num_kv_heads;
  const int row_tiles = (int)(((int64_t)a.max_query * G + kGradTile - 1) / kGradTile);
  const DkvPlan plan = plan_dkv(a, cu_count());
  float* delta = ws;
  float* partial = delta + grad_rows(a.total_rows, a.num_heads);
  dq<<<win_grid(pairs, row_tiles), 256, smem, stream>>>(g, row_tiles, delta);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t magic = G == 1 ? 0u : (uint32_t)((0x100000000ull + G - 1) / G);
  dkv<<<win_grid(pairs, plan.items()), 256, smem_kv, stream>>>(g, plan, magic, delta, partial);
  e = hipGetLastError();
  if (e != hipSuccess || plan.partial_items() == 0) return e;
  const int tiles = plan.parts > 1 ? plan.tiles : plan.sink_tiles;
  window_dkv_join_kernel<HS, BF><<<(unsigned)(pairs * tiles * (kGradTile * (2 * HS / 4) / 256)), 256, 0, stream>>>(
      g, plan, tiles, partial);
  return hipGetLastError();
}

}  // namespace

template <bool BF>
hipError_t launch_window_grad(const WindowGradArgs& g, float* ws, hipStream_t stream) {
  switch (g.f.head_size) {
    case 64: return launch_grad_hs<64, BF>(g, ws, stream);
    case 80: return launch_grad_hs<80, BF>(g, ws, stream);
    case 96: return launch_grad_hs<96, BF>(g, ws, stream);
    case 112: return launch_grad_hs<112, BF>(g, ws, stream);
    case 128: return launch_grad_hs<128, BF>(g, ws, stream);
    case 256: return launch_grad_hs<256, BF>(g, ws, stream);
    default: return hipErrorInvalidValue;
  }
}
template hipError_t launch_window_grad<WINDOW_BF16>(const WindowGradArgs&, float*, hipStream_t);

#if !WINDOW_BF16
size_t window_grad_ws_bytes(const WindowArgs& a) {
  const DkvPlan p = plan_dkv(a, cu_count());
  const size_t pairs = (size_t)a.num_seqs * a.num_kv_heads;
  return sizeof(float) * (grad_rows(a.total_rows, a.num_heads) + pairs * p.partial_items() * kGradTile * 2 * a.head_size);
}
#endif

}  // namespace dw4
