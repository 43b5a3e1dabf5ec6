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
//   * cache blocks lie in LDS as in memory, those of 32 tokens with the four
//     16-byte units of a dim's values rotated against bank conflicts;
//   * token rows lie as [token][dims], and values reach the second product
//     through LDS's transposing reads.
// Matrix cores and vector ALU bound it together, each busy for half of the cycles at
// the 1.8 to 1.9 GHz that the card holds under this load.  Measured: four prompts of
// 900 to 12000 tokens, window 4096, heads 32 on 8 of 128, bf16 (1.7 TFLOP) 1717 to 1800 us
// from box to box, 0.95 to 1.0 PFLOP/s (a 16384^3 library product 1.32 to 1.37); dense rows of
// 6000 and 4100 tokens, window 2048, 32 heads of 128 (0.31 TFLOP) 428 us, 0.72 PFLOP/s: its
// spans are half as long, and their masked steps, which issue their copies at once and
// read every value twice, weigh double.  Two workgroups of four waves per CU, so that one's
// softmax runs beside another's products: eight waves on one step's copies won 2.6 %
// on the prompts and lost 17 % on the dense rows, 64 rows a wave with one wave per SIMD took 11 % and
// 45 % longer, copies issued together instead of among the products 6 % longer.
//
// Probabilities enter p . v rounded to the
// value type (fp16: of 2^10 p), as the matrix cores take it: their errors are
// independent of each other, and add to the output's own rounding about as much
// again; the denominator sums the rounded ones, so that the weights add up to 1.
// Values of NaN and infinity reach the rows that see them and no others; where a step is
// seen whole an infinity whose probability rounds to zero (fp16: below 2^-35) gives NaN.

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

// BS: block size of the cache, 0 for token rows.
template <int HS, int BS, bool BF>
__global__ void __launch_bounds__(256, HS <= 128 ? 2 : 1)
window_tile_kernel(WindowArgs a, int tiles, int splits, float* __restrict__ ws_ml,
                   float* __restrict__ ws_out) {
  constexpr int KD = HS / 16;
  constexpr int ND = (HS + 31) / 32;
  constexpr bool VTAIL = HS % 32 != 0;
  constexpr int NB = BS == 0 ? 1 : kBk / BS;  // blocks of a step
  constexpr int STEPS = 64 / NB;              // steps whose block addresses the lanes hold
  constexpr int BB = HS * BS * 2;             // bytes of a block's keys (or values)
  constexpr int HALF = BS == 0 ? row_at<HS>(kBk) : kBk * HS * 2;
  constexpr int STAGE = 2 * HALF;             // keys of 64 tokens, then their values
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];

  if constexpr (BS == 0)
    zero_outside(a.out, a.o_stride, a.num_heads * HS, a.starts, a.num_seqs, a.total_rows, blockIdx.x, gridDim.x);
  int pair, item;
  if (!work_of(blockIdx.x, a.num_seqs * a.num_kv_heads, tiles * splits, pair, item)) return;
  const int split = item % splits;
  const int tile = tiles - 1 - item / splits;
  const int seq = pair / a.num_kv_heads, kvh = pair % a.num_kv_heads;
  const int G = a.num_heads / a.num_kv_heads;
  int q0, q1;
  seq_rows(a.starts, seq, a.total_rows, q0, q1);
  const int n = min(q1 - q0, a.max_query);
  const int rows = n * G, base = tile * 128;
  if (BS == 0) zero_beyond(a.out + (size_t)kvh * G * HS, a.o_stride, G * HS, q0 + n, q1, tile, tiles);
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
  const int wfirst = p0 + min(wbase, rows - 1) / G, wlast = p0 + min(wbase + 31, rows - 1) / G;

  // ---- the copies of one step into a stage
  const bool near = a.k_stride <= kNearRows && a.v_stride <= kNearRows;
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
  // A step's copies are PARTS per wave, keys and values in turn (part()), from
  // addresses that next_step() sets; steps with missing blocks and the last tokens of
  // a sequence, which need a bound each, go as a whole (slowly()).
  constexpr int UNITS = HS / 8, CHUNKS = BS == 0 ? kBk * UNITS / 64 : (BB + 1023) / 1024;
  constexpr int ITEMS = BS == 0 ? CHUNKS : NB * CHUNKS, PARTS = (ITEMS + 3) / 4 * 2;
  const uint64_t k_first = (uint64_t)(a.k + (size_t)q0 * a.k_stride + (size_t)kvh * HS);
  const uint64_t v_first = (uint64_t)(a.v + (size_t)q0 * a.v_stride + (size_t)kvh * HS);
  uint64_t next_k = 0, next_v = 0;  // token rows: their addresses
  int next_l = 0;                   // blocks: the lane that holds the first one's
  uint32_t next_dst = 0;
  auto next_step = [&](int s, int stage) {  // false: slowly()
    next_dst = lds0 + stage * STAGE;
    if constexpr (BS == 0) {
      const int t = span.token<kBk>(s);
      if (!near || t + kBk > cap) return false;
      next_k = k_first + (uint64_t)(uint32_t)t * (uint32_t)(a.k_stride * 2);
      next_v = v_first + (uint64_t)(uint32_t)t * (uint32_t)(a.v_stride * 2);
    } else {
      if ((s - s0) % STEPS == 0) {
        fetch(s);
        wait_loads();
      }
      next_l = (s - s0) % STEPS * NB;
      uint32_t there = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b) there |= (uint32_t)(block_of(kp, next_l + b) != 0) << b;
      held[stage] = there;
      return there == (1u << NB) - 1;
    }
    return true;
  };
  auto part = [&](int i, auto all) {  // all: no block of the step is missing
    const int it = wave + 4 * (i >> 1);
    const bool values = i & 1;
    if (ITEMS % 4 != 0 && it >= ITEMS) return;
    if constexpr (BS == 0) {
      // (256 units further are whole rows where a row is a power of two: one offset per lane)
      constexpr bool EVEN = 256 % UNITS == 0;
      const int u = (EVEN ? wave : it) * 64 + lane;
      const uint32_t r = u / UNITS, at = ((u % UNITS) ^ swizzle<HS>(r)) * 16;
      const uint32_t k2 = (uint32_t)(a.k_stride * 2), v2 = (uint32_t)(a.v_stride * 2), on = EVEN ? (i >> 1) * (256 / UNITS) : 0;
      if (values) copy16(next_v + on * v2, r * v2 + at, next_dst + HALF + chunk_at<HS>(it));
      else copy16(next_k + on * k2, r * k2 + at, next_dst + chunk_at<HS>(it));
    } else {
      // a block's keys as they lie; its values too, for 32-token blocks with the
      // four 16-byte units of a row rotated by dim / 4 (mod 4)
      const int b = it / CHUNKS, at = it % CHUNKS * 1024;
      const uint64_t p = block_of(values ? vp : kp, next_l + b);
      if (!decltype(all)::value && p == 0) return;
      if (BB % 1024 != 0 && at + lane * 16 >= BB) return;
      const uint32_t off = BS == 32 && values ? (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 4) & 3)) * 16) : lane * 16;
      copy16(p + at, off, next_dst + (values ? HALF : 0) + b * BB + at);
    }
  };
  auto slowly = [&](int s) {
    if constexpr (BS != 0) {
#pragma unroll
      for (int i = 0; i < PARTS; ++i) part(i, std::false_type{});
      return;
    }
    const int t = span.token<kBk>(s);
    for (int ch = wave; ch < CHUNKS; ch += 4) {
      const int u = ch * 64 + lane;
      const int r = u / UNITS, at = (u % UNITS) ^ swizzle<HS>(r);
      const int64_t token = q0 + min(t + r, cap - 1);
      const size_t col = (size_t)kvh * HS + at * 8;
      copy16(a.k + token * a.k_stride + col, next_dst + chunk_at<HS>(ch));
      copy16(a.v + token * a.v_stride + col, next_dst + HALF + chunk_at<HS>(ch));
    }
  };
  auto issue = [&](int s, int stage) {
    if (next_step(s, stage)) {
#pragma unroll
      for (int i = 0; i < PARTS; ++i) part(i, std::true_type{});
    } else {
      slowly(s);
    }
  };
  auto key = [&](const unsigned char* st, int sub, int kk) {
    const int t = row_token(c);  // of the 32 tokens `sub`
    if constexpr (BS == 0) return row_unit<HS>(st + row_at<HS>(32 * sub), t, 2 * kk + half);
    else return *(const h8*)(st + 32 / (BS + !BS) * sub * BB + t / (BS + !BS) * BB + ((2 * kk + half) * BS + t % (BS + !BS)) * 16);
  };
  auto value = [&](const unsigned char* st, int sub, int d, int s) {
    const int dim = VTAIL ? min(32 * d + c, HS - 1) : 32 * d + c;
    if constexpr (BS == 0) return column_unit<HS>(st + HALF, 32 * sub + 16 * s, d);
    else if constexpr (BS == 16) return *(const h8*)(st + HALF + (2 * sub + s) * BB + dim * 32 + half * 16);
    else return *(const h8*)(st + HALF + sub * BB + dim * 64 + (((2 * s + half) ^ ((dim >> 2) & 3)) << 4));
  };

  if (s0 < s1) issue(s0, 0);
  h8 qreg[KD];  // B operand: column c is this lane's row
  {
    const uint16_t* qp = a.q + (size_t)(q0 + row / G) * a.q_stride + (size_t)(kvh * G + row % G) * HS + 8 * half;
#pragma unroll
    for (int j = 0; j < KD; ++j) qreg[j] = *(const h8*)(qp + 16 * j);
  }
  wait_loads();
  float m = kNoMax, l[2] = {0.f, 0.f};  // of the row (l: this lane's tokens, in two parts)
  f16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f16v{};

  // the steps of which every row of the workgroup sees every token
  int f0 = s1, f1 = s0;
  {
    const int first = p0 + base / G, last_row = p0 + (min(base + 128, rows) - 1) / G;
    const int most = min(first, cap - 1) - (kBk - 1) - span.lo;  // of token(step) - lo
    const int least = a.window == 0 ? 0 : last_row - a.window + 1 - span.lo;
    if (most >= 0) {
      f0 = span.sink_steps + (max(least, 0) + kBk - 1) / kBk;
      f1 = span.sink_steps + most / kBk + 1;
    }
  }
  // with `copies`, the next step's go out among the products: at once they would
  // hold up the wave until the memory pipeline has taken them all
  auto scores = [&](const unsigned char* st, f16v (&s)[2], auto copies) {
    constexpr bool kCopies = decltype(copies)::value;
    feed<2 * KD, 8>([&](int i) { return key(st, i & 1, i >> 1); },
                    [&](int i, h8 f) {
                      s[i & 1] = mfma32_of<BF>(f, qreg[i >> 1], s[i & 1]);
                      if constexpr (kCopies) {
#pragma unroll
                        for (int c = i * PARTS / (2 * KD); c < (i + 1) * PARTS / (2 * KD); ++c) part(c, std::true_type{});
                      }
                    });
  };
  // the running maximum (it may lag kLag behind), and the probabilities
  auto probabilities = [&](f16v (&s)[2], h8 (&p)[2][2]) {
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) mx = fmaxf(mx, s[e >> 4][e & 15]);
    mx = both_max(mx) * a.scale_log2;
    if (__any(mx > m + kLag)) {
      const float mn = fmaxf(m, mx);
      const float f = __builtin_amdgcn_exp2f(m - mn);
      l[0] *= f;
      l[1] *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= f;
      m = mn;
    }
    const float shift = p_shift<BF>() - m;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = __builtin_amdgcn_exp2f(fmaf(s[b][8 * g + 2 * e], a.scale_log2, shift));
          const float z = __builtin_amdgcn_exp2f(fmaf(s[b][8 * g + 2 * e + 1], a.scale_log2, shift));
          x[e] = pack2<BF>(y, z);
          l[e & 1] = add_pair<BF>(x[e], l[e & 1]);
        }
        p[b][g] = __builtin_bit_cast(h8, x);
      }
  };
  auto whole = [&](int stage, bool more) {  // a step that every row sees
    const unsigned char* st = lds + stage * STAGE;
    f16v s[2] = {f16v{}, f16v{}};
    h8 p[2][2];
    if (more) scores(st, s, std::true_type{});
    else scores(st, s, std::false_type{});
    probabilities(s, p);
    feed<4 * ND, 8>(
        [&](int i) { return value(st, i / (2 * ND), i % ND, i / ND % 2); },
        [&](int i, h8 f) { o[i % ND] = mfma32_of<BF>(f, p[i / (2 * ND)][i / ND % 2], o[i % ND]); });
  };
  auto masked = [&](int step, int stage) {
    const int t = span.token<kBk>(step);
    if (nrows <= 0 || t > wlast || (a.window != 0 && t + kBk - 1 <= wfirst - a.window && t >= a.sinks)) return;
    const unsigned char* st = lds + stage * STAGE;
    int at = pos;  // (what follows from it holds no register across the steps)
    asm volatile("" : "+v"(at));
    const int last = min(at, cap - 1), before = a.window == 0 ? INT32_MIN : at - a.window;
    uint32_t seen = 0;  // bit 16 b + e: score e of the 32 tokens b
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t x = own_scores(seen_of(t + 32 * b, last, before, a.sinks), half);
      if constexpr (BS == 32) x = held[stage] >> b & 1 ? x : 0u;
      if constexpr (BS == 16) x &= (held[stage] >> (2 * b) & 1 ? 0xFFu : 0u) | (held[stage] >> (2 * b + 1) & 1 ? 0xFF00u : 0u);
      seen |= x << (16 * b);
    }
    f16v s[2] = {f16v{}, f16v{}};
    h8 p[2][2];
    scores(st, s, std::false_type{});
#pragma unroll
    for (int x = 0; x < 32; ++x) s[x >> 4][x & 15] = where_seen(seen, x, s[x >> 4][x & 15], -INFINITY);
    probabilities(s, p);
    // a value that some rows do not see (or that no row does) must not reach
    // them as 0 * inf: where there is one, its part is added apart
    uint32_t bits = 0;
    feed<4 * ND, 8>([&](int i) { return value(st, i / (2 * ND), i % ND, i / ND % 2); },
                    [&](int, h8 f) { add_nonfinite<BF>(f, bits); });
    const bool odd = __any((bits & kNonfinite) != 0);
    if (odd) {  // (a fragment at a time: scheduled together they take registers from the usual steps)
      for (uint32_t sign = 0; sign <= 0x8000u; sign += 0x8000u) {
        const float inf = sign ? -INFINITY : INFINITY;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          f16v count = {};
#pragma unroll
          for (int x = 0; x < 4; ++x)
            count = mfma32_of<BF>(infinite_part<BF>(value(st, x >> 1, d, x & 1), sign), ones_of<BF>(seen >> (8 * x)), count);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (count[e] > 0.f) o[d][e] += inf;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4 * ND; ++i) {
        o[i % ND] = mfma32_of<BF>(finite_part<BF>(value(st, i / (2 * ND), i % ND, i / ND % 2)), p[i / (2 * ND)][i / ND % 2], o[i % ND]);
        __builtin_amdgcn_sched_barrier(0);
      }
      return;
    }
    feed<4 * ND, 8>([&](int i) { return value(st, i / (2 * ND), i % ND, i / ND % 2); },
                    [&](int i, h8 f) { o[i % ND] = mfma32_of<BF>(f, p[i / (2 * ND)][i / ND % 2], o[i % ND]); });
  };
  int stage = 0, step = s0;
  auto is_whole = [&]() { return step >= f0 && step < f1 && held[stage] == (1u << NB) - 1; };
  while (step < s1) {
    wait_copies();
    wait_loads();  // (registers that the masked steps put aside: none may be waited for in the loop)
    while (is_whole()) {
      const bool more = step + 1 < s1, parts = more && next_step(step + 1, stage ^ 1);
      if (more && !parts) slowly(step + 1);
      whole(stage, parts);
      stage ^= 1;
      if (++step == s1) break;
      wait_copies();
    }
    if (step == s1) break;
    if (step + 1 < s1) issue(step + 1, stage ^ 1);
    masked(step, stage);
    stage ^= 1;
    ++step;
  }

  const float sum = both_sum(l[0] + l[1]);
  const int thread = thread_again(), col = thread & 31, hi = thread >> 5 & 1;
  if (col >= nrows) return;
  const int own = wbase + col, token = q0 + own / G, head = kvh * G + own % G;
  if (splits == 1) {
    const float f = sum == 0.f ? 1.f : 1.f / sum;  // no visible token: zeros
    uint16_t* op = a.out + (size_t)token * a.o_stride + (size_t)head * HS;
    uint16_t* rp = a.rest + ((size_t)token * a.num_heads + head) * HS;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int dim = d * 32 + 2 * e + 4 * hi;
        if (VTAIL && dim >= HS) continue;
        float y[4];
        uint32_t x[2], r[2];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = o[d][e + k] * f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          x[k] = pack2<BF>(y[2 * k], y[2 * k + 1]);
          r[k] = pack2<BF>(y[2 * k] - unpack<BF>(x[k], 0), y[2 * k + 1] - unpack<BF>(x[k], 1));
        }
        *(uint2*)(op + dim) = make_uint2(x[0], x[1]);
        if (BS == 0 && a.rest != nullptr) *(uint2*)(rp + dim) = make_uint2(r[0], r[1]);
      }
    if (a.lse != nullptr && hi == 0)
      a.lse[(size_t)token * a.num_heads + head] = m + __builtin_amdgcn_logf(sum) - p_shift<BF>();
  } else {
    const size_t slot = ((size_t)token * a.num_heads + head) * splits + split;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int dim = d * 32 + 2 * e + 4 * hi;
        if (!VTAIL || dim < HS)
          *(f4*)(ws_out + slot * HS + dim) = f4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
      }
    if (hi == 0) {
      ws_ml[2 * slot] = m;
      ws_ml[2 * slot + 1] = sum;
    }
  }
}

template <int HS, int BS, bool BF>
hipError_t launch_tile_bs(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  auto kern = &window_tile_kernel<HS, BS, BF>;
  constexpr size_t smem = BS == 0 ? 4 * row_at<HS>(kBk) : 4 * kBk * HS * 2;
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(kern), smem, done);
  if (e != hipSuccess) return e;
  kern<<<win_grid(a.num_seqs * a.num_kv_heads, p.tiles * p.splits), 256, smem, stream>>>(
      a, p.tiles, p.splits, ws, ws + win_ml_floats(a.total_rows, a.num_heads, p.splits));
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
