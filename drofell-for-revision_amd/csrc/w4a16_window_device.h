// Device helpers of the windowed-attention kernels.
//
// All of them work on 32 x 32 x 16 matrix instructions, with the scores'
// columns one row of the softmax each: lane l holds column l % 32, and register
// i the token (of 32) 16 (i / 8) + 8 (l / 32) + i % 8.  The instruction itself
// puts row 8 (i / 4) + 4 (l / 32) + i % 4 there; the A operand's rows are
// loaded in the order row_token() for it, and then a lane's eight scores
// i / 8 == s are those of the eight consecutive tokens that the B operand of the
// next product wants of it (reduction step s): probabilities go from one
// product to the next without leaving their lane.
#pragma once

#include "w4a16_device.h"

namespace dw4 {

constexpr float kNoMax = -3.4028234663852886e38f;  // running maximum of a row that saw no token
// exp2 offset of fp16 probabilities: those down to 2^-24 of the largest keep
// all of fp16's bits (a running maximum may lag kLag behind: 2^10 * 2^4 < 65504)
template <bool BF>
__device__ __forceinline__ constexpr float p_shift() { return BF ? 0.f : 10.f; }
constexpr float kLag = 4.f;

__device__ __forceinline__ int row_token(int r) {  // token (of 32) of the A operand's row r
  return (r & 16) | ((r & 4) << 1) | ((r & 8) >> 1) | (r & 3);
}

// max / sum over the two lanes of a column
__device__ __forceinline__ float both_max(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)x[0]), __builtin_bit_cast(float, (uint32_t)x[1]));
}
__device__ __forceinline__ float both_sum(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)x[0]) + __builtin_bit_cast(float, (uint32_t)x[1]);
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF) return pack_bf16(lo, hi);
  else return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
}
template <bool BF>
__device__ __forceinline__ float unpack(uint32_t u, int hi) {
  if constexpr (BF) return __builtin_bit_cast(float, hi ? u & 0xFFFF0000u : u << 16);
  else return (float)as_h2(u)[hi];
}
// sum + both halves of a packed pair (v_dot2 with ones: exact products, fp32 sum)
template <bool BF>
__device__ __forceinline__ float add_pair(uint32_t u, float sum) {
  if constexpr (BF) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, u), __builtin_bit_cast(bf2, kOnesBf16), sum, false);
  } else {
    return __builtin_amdgcn_fdot2(as_h2(u), h2{(_Float16)1.f, (_Float16)1.f}, sum, false);
  }
}

// Which tokens a tile of rows at positions first..last sees, in steps of BK
// tokens that start at multiples of BK: the steps over the sinks that lie
// before the window, then those of the window.
struct Span {
  int lo, sink_steps, steps;
  template <int BK>
  __device__ __forceinline__ static Span of(int first, int last, int cap, int window, int sinks) {
    Span s;
    const int hi = min(last + 1, cap);
    s.lo = (window == 0 ? 0 : max(0, first - window + 1)) & ~(BK - 1);
    s.sink_steps = (max(min(min(sinks, s.lo), hi), 0) + BK - 1) / BK;
    s.steps = s.sink_steps + (hi > s.lo ? (hi - s.lo + BK - 1) / BK : 0);
    return s;
  }
  template <int BK>
  __device__ __forceinline__ int token(int step) const {
    return step < sink_steps ? step * BK : lo + (step - sink_steps) * BK;
  }
};

// Row range of a sequence, kept within the tensor whatever the starts hold.
__device__ __forceinline__ void seq_rows(const int32_t* starts, int seq, int total, int& q0, int& q1) {
  q0 = seq;
  q1 = seq + 1;
  if (starts != nullptr) {
    q0 = min(max(starts[seq], 0), total);
    q1 = min(max(starts[seq + 1], q0), total);
  }
}

// Rows of a result that belong to no sequence (before the first, behind the
// last) become zeros, spread over the workgroups of the launch; usually none.
__device__ __forceinline__ void zero_outside(uint16_t* x, int64_t stride, int width, const int32_t* starts,
                                             int num_seqs, int total, int wg, int wgs) {
  const int head = min(max(starts[0], 0), total), tail = min(max(starts[num_seqs], head), total);
  const int n = head + total - tail;
  for (int i = wg; i < n; i += wgs) {
    const int64_t row = i < head ? i : tail + i - head;
    for (int d = threadIdx.x * 8; d < width; d += blockDim.x * 8) *(u4*)(x + row * stride + d) = u4{};
  }
}

// The rows of a sequence longer than the call said, beyond what it works on (first .. end - 1,
// usually none), become zeros: those of a pair's columns by its workgroups in turn.
__device__ __forceinline__ void zero_beyond(uint16_t* x, int64_t stride, int width, int first, int end, int item, int items) {
  for (int64_t row = (int64_t)first + item; row < end; row += items)
    for (int d = threadIdx.x * 8; d < width; d += blockDim.x * 8) *(u4*)(x + row * stride + d) = u4{};
}

// Workgroup b's (sequence, kv head) pair and its item of `items` (row tiles,
// longest spans first, x splits), false where there is none.  Workgroups go
// round-robin to the eight XCDs, each with an L2 of its own: kWinUnit
// neighbouring items, which read the same keys and values, go to one XCD, and
// the units of all pairs in turn over the XCDs, so that long and short
// sequences spread evenly.  (Pairs in one run per XCD: four prompts of 3500 to
// 12000 tokens took 1.4 times as long, the longest one's XCDs being last.)
__device__ __forceinline__ bool work_of(int b, int pairs, int items, int& pair, int& item) {
  const int unit = min(items, kWinUnit), slot = b >> 3;
  const int u = (b & 7) + 8 * (slot / unit);
  pair = u % pairs;
  item = u / pairs * unit + slot % unit;
  return item < items;
}

// Sets bit 15 or 31 of a word of `bits` if an element of x is not finite (the
// exponent's carry; other bits of `bits` mean nothing).
template <bool BF>
__device__ __forceinline__ void add_nonfinite(h8 x, uint32_t& bits) {
  constexpr uint32_t kExp = BF ? 0x7F807F80u : 0x7C007C00u, kLow = BF ? 0x00800080u : 0x04000400u;
  const u4 v = __builtin_bit_cast(u4, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) bits |= (v[e] & kExp) + kLow;
}
constexpr uint32_t kNonfinite = 0x80008000u;

// x without its non-finite elements.
template <bool BF>
__device__ __forceinline__ h8 finite_part(h8 x) {
  constexpr uint32_t kExp = BF ? 0x7F80u : 0x7C00u;
  u4 v = __builtin_bit_cast(u4, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = (v[e] & kExp) == kExp ? 0u : v[e] & 0xFFFFu;
    const uint32_t hi = (v[e] & (kExp << 16)) == kExp << 16 ? 0u : v[e] & 0xFFFF0000u;
    v[e] = lo | hi;
  }
  return __builtin_bit_cast(h8, v);
}
// 1 where x is NaN or the infinity of this sign bit, else 0.
template <bool BF>
__device__ __forceinline__ h8 infinite_part(h8 x, uint32_t sign) {
  constexpr uint32_t kExp = BF ? 0x7F80u : 0x7C00u, kOne = BF ? 0x3F80u : 0x3C00u;
  u4 v = __builtin_bit_cast(u4, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = v[e] & 0xFFFFu, hi = v[e] >> 16, other = kExp | (sign ^ 0x8000u);
    v[e] = ((lo & kExp) == kExp && lo != other ? kOne : 0u) | ((hi & kExp) == kExp && hi != other ? kOne << 16 : 0u);
  }
  return __builtin_bit_cast(h8, v);
}
// Eight ones and zeros as an operand, from the bits of a mask.
template <bool BF>
__device__ __forceinline__ h8 ones_of(uint32_t bits) {
  constexpr uint32_t kOne = BF ? 0x3F80u : 0x3C00u;
  u4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (bits >> (2 * e) & 1 ? kOne : 0u) | (bits >> (2 * e + 1) & 1 ? kOne << 16 : 0u);
  return __builtin_bit_cast(h8, v);
}

// Whether a row sees token j: not after `last` (the row's position, and within
// the cache), and after `before` or a sink.
__device__ __forceinline__ bool sees(int j, int last, int before, int sinks) {
  return j <= last && (j > before || j < sinks);
}
// The n lowest of 32 bits (none for n <= 0).
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
// Bit e: whether a row sees token t + e, of 32.
__device__ __forceinline__ uint32_t seen_of(int t, int last, int before, int sinks) {
  // before - t may pass the 32-bit range below (no window: every token is after it)
  const int b = before < t ? -1 : before - t;
  return low_bits(last - t + 1) & (~low_bits(b + 1) | low_bits(sinks - t));
}
// Of 32 tokens' bits (per row) the lane's own scores' (register i: token
// 16 (i / 8) + 8 (lane / 32) + i % 8), in bits 0 .. 15.
__device__ __forceinline__ uint32_t own_scores(uint32_t seen, int half) {
  const uint32_t x = seen >> (8 * half);
  return (x & 0xFFu) | ((x >> 8) & 0xFF00u);
}
// v where bit i of `seen` is set, else `other`.
__device__ __forceinline__ float where_seen(uint32_t seen, int i, float v, float other) {
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)seen, i, 1);
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & m) | (__builtin_bit_cast(uint32_t, other) & ~m));
}

// global -> LDS copy of 16 / 4 bytes per active lane, to lds + lane * 16 / 4 (a
// wave-uniform base).  In assembly, so that the compiler does not make every
// later LDS read wait for it; the kernels wait themselves (wait_copies()).
typedef __attribute__((address_space(3))) const void lds_cvoid;
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(lds_cvoid*)p;
}
__device__ __forceinline__ void copy16(const void* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds) : "memory");
}
__device__ __forceinline__ void copy4(const void* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "s"(lds) : "memory");
}
// The same from a wave-uniform address and an offset per lane, whose 64-bit
// sum then takes no vector ALU.
__device__ __forceinline__ void copy16(uint64_t g, uint32_t lane_offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               ::"v"(lane_offset), "s"(g), "s"(lds) : "memory");
}
__device__ __forceinline__ void copy4(uint64_t g, uint32_t lane_offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               ::"v"(lane_offset), "s"(g), "s"(lds) : "memory");
}
// Rows at most so far apart (elements) that 128 of them lie within 32-bit offsets.
constexpr int64_t kNearRows = 1 << 23;
// Every copy of this workgroup has landed and every wave has left the stage before.
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Every load of this wave has landed, to the compiler's knowledge too (a load
// into registers used in a loop would make it wait in every round of it).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); }

// threadIdx.x once more: what is computed from it holds no register before.
__device__ __forceinline__ int thread_again() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// N operands, each loaded (from LDS) AHEAD uses before its use.  The loads and
// the matrix instructions keep this order; vector-ALU work may move among them.
template <int N, int AHEAD, typename Load, typename Use>
__device__ __forceinline__ void feed(Load&& load, Use&& use) {
  constexpr int kMoves = 0x2 | 0x4 | 0x400;  // vector ALU, scalar ALU, transcendental
  decltype(load(0)) f[N];
#pragma unroll
  for (int i = 0; i < (AHEAD < N ? AHEAD : N); ++i) f[i] = load(i);
  __builtin_amdgcn_sched_barrier(kMoves);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + AHEAD < N) f[i + AHEAD] = load(i + AHEAD);
    __builtin_amdgcn_sched_barrier(kMoves);
    use(i, f[i]);
    __builtin_amdgcn_sched_barrier(kMoves);
  }
}

// Row-major tiles in LDS ([row][HS], as the tensors have them), laid out so that
// both reads, a unit of 32 rows (row_unit) and four rows by 32 dims (column_unit),
// spread over the banks, and so that few addresses differ by more than a constant:
//   * HS 128 and 256: 16-byte unit u of row r stands at unit u ^ 4 (r % 4), and
//     every four rows 16 bytes further;
//   * HS 64: at unit u ^ (2 (r & 2) + r / 4 % 4);
//   * HS 80, 96 and 112: as it is, the rows' own stride does it.
template <int HS>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (HS % 128 == 0) return (r & 3) << 2;
  else if constexpr (HS == 64) return ((r & 2) << 1) | ((r >> 2) & 3);
  else return 0;
}
template <int HS>
__host__ __device__ constexpr int row_at(int r) {
  return HS % 128 == 0 ? (r >> 2) * (8 * HS + 16) + (r & 3) * (2 * HS) : r * (2 * HS);
}
template <int HS>  // of 64 units (1 KiB), as a copy instruction writes them
__device__ __forceinline__ int chunk_at(int ch) {
  return ch * 1024 + (HS % 128 == 0 ? ch / (HS / 128) * 16 : 0);
}
// A operand: unit `unit` of row r.
template <int HS>
__device__ __forceinline__ h8 row_unit(const unsigned char* tile, int r, int unit) {
  return *(const h8*)(tile + row_at<HS>(r) + ((unit ^ swizzle<HS>(r)) << 4));
}
// A operand of the transposed tile: dims 32 dt + lane % 32 (below HS), rows
// r0 + 8 (lane / 32) .. + 7, by two transposing reads.  Lane l of 16 gives the
// address of four dims of row l / 4 and receives dim l of the four rows.
template <int HS>
__device__ __forceinline__ h8 column_unit(const unsigned char* tile, int r0, int dt) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 lds_s4;
  const int lane = threadIdx.x & 63;
  int d = dt * 32 + (lane & 16);
  if (HS % 32 != 0) d = min(d, HS - 16);
  d += 4 * (lane & 3);
  const int r = ((lane >> 5) << 3) + ((lane >> 2) & 3);
  tile += row_at<HS>(r0);  // r0 is a multiple of 16
  s4 x[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned char* at = tile + row_at<HS>(r + 4 * h) + ((((d >> 3) ^ swizzle<HS>(r + 4 * h)) << 4) | ((d & 7) << 1));
    x[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
  }
  typedef short s8 __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(h8, (s8)__builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

}  // namespace dw4
