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
// rows, lane 16 g + c unit g of row c: loaded in that layout, neighbouring lanes touch different rows, half a
// line of each, one 16-byte access after the other.  Loads and stores take whole lines in consecutive lanes
// instead, a pair of instructions 16 rows of 128 bytes (lane l: unit l % 8 of rows l / 8 and 8 + l / 8), and
// 2 KiB of LDS of the wave's own turn the pair into the operands of units g and 4 + g of row c, and
// back; the units' places are exchanged by row so that the accesses spread over the banks.  Measured: 10240
// rows of 16 KiB copied by tiles of 64 rows 3.4 TB/s by 64 bytes a row, 4.6 by 128 or 256; 10175 rows
// of 11008 against rank 16 43.4 us with the lanes of a row 16 apart, 40.4 in consecutive lanes.
__device__ __forceinline__ void to_operands(u4& p, u4& q, u4* own) {
  const int lane = threadIdx.x & 63, r = lane >> 3, u = lane & 7, g = lane >> 4, c = lane & 15;
  own[r * 8 + (u ^ r)] = p;
  own[(8 + r) * 8 + (u ^ r)] = q;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  p = own[c * 8 + (g ^ (c & 7))];
  q = own[c * 8 + ((4 + g) ^ (c & 7))];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
__device__ __forceinline__ void from_operands(u4& p, u4& q, u4* own) {
  const int lane = threadIdx.x & 63, r = lane >> 3, u = lane & 7, g = lane >> 4, c = lane & 15;
  own[c * 8 + (g ^ (c & 7))] = p;
  own[c * 8 + ((4 + g) ^ (c & 7))] = q;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  p = own[r * 8 + (u ^ r)];
  q = own[(8 + r) * 8 + (u ^ r)];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

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
// An infinite value's product with a first part is what the sum comes to, infinite or NaN; its product with a
// second part of zero, or of the other sign, would make the sum NaN in any case.  What a second part is multiplied
// with where infinities are about: the finite values, zeros for the others.
template <bool BF>
__device__ __forceinline__ u4 finite_only(u4 v) {
  constexpr uint32_t kExp = BF ? 0x7F80u : 0x7C00u;
  asm volatile("" : "+v"(v));  // made where it is used: kept for several products it took 60 registers
#pragma unroll
  for (int e = 0; e < 4; ++e)
    v[e] = ((v[e] & kExp) == kExp ? 0u : v[e] & 0xFFFFu) | ((v[e] & (kExp << 16)) == kExp << 16 ? 0u : v[e] & 0xFFFF0000u);
  return v;
}
// Adds to `bits` whether a value of v is not finite (the exponent's carry into bits 15 and 31; other bits mean nothing).
template <bool BF>
__device__ __forceinline__ void add_nonfinite(u4 v, uint32_t& bits) {
  constexpr uint32_t kExp = BF ? 0x7F807F80u : 0x7C007C00u, kLow = BF ? 0x00800080u : 0x04000400u;
#pragma unroll
  for (int e = 0; e < 4; ++e) bits |= (v[e] & kExp) + kLow;
}
// Whether a lane of the wave holds NaN in v (infinities of both signs count too).
__device__ __forceinline__ bool nan_among(const f4 (&v)[4]) {
  const f4 s = v[0] + v[1] + v[2] + v[3];
  const float x = (s[0] + s[1]) + (s[2] + s[3]);
  return __ballot(x != x) != 0;
}
// fp16's range is small: its operands are brought to below 2^14 by the power of two that
// this gives for their largest finite magnitude, and the product back by its inverse.  bf16 needs none.
template <bool BF>
__device__ __forceinline__ int range_exponent(float largest) {
  if (BF || !(largest > 0.f)) return 0;
  return min(13 - ilogbf(largest), 120);
}
__device__ __forceinline__ float finite_magnitude(float v) { return isfinite(v) ? fabsf(v) : 0.f; }
__device__ __forceinline__ float times_pow2(float v, int e) { return __builtin_ldexpf(v, e); }
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }  // |e| below 127

}  // namespace dw4
