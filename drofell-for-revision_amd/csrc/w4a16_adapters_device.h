// Device helpers of the low-rank adapters' kernels.
#pragma once

#include "w4a16_adapters.h"
#include "w4a16_device.h"

namespace dw4 {

// Dropout's generator: Philox 4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011) of the counter (column / 8, row,
// offset) under the seed; its 128 bits are eight elements' 16.  An element is kept
// if its 16 bits are at least `drop`.
struct Philox {
  uint32_t key0, key1, off0, off1;
  __device__ __forceinline__ explicit Philox(const int64_t* seed) {
    const uint64_t s = (uint64_t)seed[0], o = (uint64_t)seed[1];
    key0 = (uint32_t)s;
    key1 = (uint32_t)(s >> 32);
    off0 = (uint32_t)o;
    off1 = (uint32_t)(o >> 32);
  }
  __device__ __forceinline__ u4 operator()(uint32_t unit, uint32_t row) const {
    uint32_t c0 = unit, c1 = row, c2 = off0, c3 = off1, k0 = key0, k1 = key1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
      c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
      c1 = (uint32_t)b;
      c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
      c3 = (uint32_t)a;
      k0 += 0x9E3779B9u;
      k1 += 0xBB67AE85u;
    }
    return u4{c0, c1, c2, c3};
  }
  // Eight elements' bits where they are kept: all ones, else zeros.
  __device__ __forceinline__ u4 mask(uint32_t unit, uint32_t row, uint32_t drop) const {
    u4 w = (*this)(unit, row);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = ((w[e] & 0xFFFFu) >= drop ? 0xFFFFu : 0u) | ((w[e] >> 16) >= drop ? 0xFFFF0000u : 0u);
    return w;
  }
};

// Rows in memory and rows as operands.  A 16 x 16 x 32 operand holds four 16-byte units of 16
// rows (lane 16 g + c: unit g of row c), so that a load in that layout takes 64 bytes of
// each row, half a line.  Loads and stores take 128 instead: of a pair, the first instruction has
// rows 0 .. 7 and the second rows 8 .. 15, lane 16 g + c unit g (c below 8) or 4 + g (else) of
// row c % 8.  exchange() turns such a pair into the operands of units g and 4 + g of row c, and
// back: two moves a register within each 16 lanes.  Measured, 10240 rows of 16 KiB copied by tiles
// of 64 rows: 3.4 TB/s by 64 bytes a row, 4.6 by 128 or 256.
__device__ __forceinline__ void exchange(u4& p, u4& q) {
  constexpr int kRotate8 = 0x128;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int a = (int)p[e], b = (int)q[e];
    p[e] = (uint32_t)__builtin_amdgcn_update_dpp(a, b, kRotate8, 0xF, 0xC, false);  // lanes 8 .. 15: b of 0 .. 7
    q[e] = (uint32_t)__builtin_amdgcn_update_dpp(b, a, kRotate8, 0xF, 0x3, false);  // lanes 0 .. 7: a of 8 .. 15
  }
}
// The item (of `items`) that workgroup b of at least as many works on, or -1.  Workgroups go round-robin
// to the eight XCDs, each with an L2 of its own: neighbouring items, which read the same
// weights, go to one, equally many to each.
__device__ __forceinline__ int item_of_xcd(int b, int items) {
  const int each = items / 8, more = items % 8, xcd = b & 7, slot = b >> 3;
  return slot < each + (xcd < more) ? xcd * each + min(xcd, more) + slot : -1;
}
// A load of what is read once: past the caches' usual places, which the weights then keep. Measured,
// 10175 rows of 11008 against rank 16: 53.7 us with plain loads, 43.3 with these; the sum with
// the projection's output 59.7 and 45.8.
__device__ __forceinline__ u4 stream_load(const uint16_t* p) { return __builtin_nontemporal_load((const u4*)p); }
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// The lane's unit (of eight) in the memory layout.
__device__ __forceinline__ int line_unit() {
  const int lane = threadIdx.x & 63;
  return (lane >> 4) + ((lane & 8) >> 1);
}

template <bool BF>
__device__ __forceinline__ f4 mfma16_of(u4 a, u4 b, f4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF) return pack_bf16(lo, hi);
  else return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
}
template <bool BF>
__device__ __forceinline__ float unpack16(uint32_t u, int hi) {
  if constexpr (BF) return __builtin_bit_cast(float, hi ? u & 0xFFFF0000u : u << 16);
  else return (float)as_h2(u)[hi];
}

// Values that go into a product as 16-bit operands without losing what they hold
// in 32 bits: a first part, rounded, and the rest, rounded again (17 bits in bf16, 22 in
// fp16, for two products instead of one).  An infinite first part has no rest.
template <bool BF>
__device__ __forceinline__ void split16(float v0, float v1, uint32_t& hi, uint32_t& lo) {
  hi = pack16<BF>(v0, v1);
  const float a = unpack16<BF>(hi, 0), b = unpack16<BF>(hi, 1);
  lo = pack16<BF>(isinf(a) ? 0.f : v0 - a, isinf(b) ? 0.f : v1 - b);
}
template <bool BF>
__device__ __forceinline__ void split16(const float (&v)[8], u4& hi, u4& lo) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t x, y;
    split16<BF>(v[2 * e], v[2 * e + 1], x, y);
    hi[e] = x;
    lo[e] = y;
  }
}
// fp16's range is small: its operands are brought to below 2^14 by the power of two that
// this gives for their largest magnitude, and the product back by its inverse.  bf16 needs none.
template <bool BF>
__device__ __forceinline__ int range_exponent(float largest) {
  if (BF || !(largest > 0.f) || isinf(largest)) return 0;
  return min(13 - ilogbf(largest), 120);
}
__device__ __forceinline__ float times_pow2(float v, int e) { return __builtin_ldexpf(v, e); }
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }  // |e| below 127

}  // namespace dw4
