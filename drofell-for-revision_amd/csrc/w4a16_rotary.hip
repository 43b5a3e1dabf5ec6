// Rotary positions: the pairs of a head's first rotary_size dims turned by position times
// the pair's frequency,
//   a' = m (a cos - b sin),  b' = m (b cos + a sin),
// with (a, b) the dims (i, i + rotary_size / 2), or (2 i, 2 i + 1) interleaved; and the
// same with the keys, and the values as they are, going to their cache slots.
//
// A frequency comes as a 64-bit fraction of a turn, so that its product with a position
// wraps around at whole turns without rounding: angles are as exact at position 2^30 as at 2 (the fraction's
// own rounding, 2^-65 of a turn, reaches fp32's beyond position 2^38).
//
// Bound by memory: every element is read and written once.  A thread holds the sines and
// cosines of eight pairs (four, interleaved) of a row and turns them in one head after the other.
// Measured on several cards: 7907 rows of 32 + 32 heads of 128 (bf16) 49 to 52 us for 259 MB, 5.0 to 5.3 TB/s; 11678
// rows of 32 + 8 heads into the cache 57 to 63 us for 289 MB, 4.6 to 5.0; a decode step of 48 rows 6.1 to 6.3, one launch.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "w4a16_adapters_device.h"
#include "w4a16_rotary.h"

namespace dw4 {

namespace {

constexpr int kThreads = 256;

// What a thread works on within a head: VEC: a unit of eight pairs (two units of eight dims,
// or interleaved one unit of four pairs), then units of eight dims that pass; else a pair, then a dim.
template <bool VEC, bool IL>
struct Turn {
  static constexpr int kPairs = VEC ? (IL ? 4 : 8) : 1;
  float cs[kPairs], sn[kPairs];
  int at, other;  // first dims; other < 0: passes
  __device__ __forceinline__ static int units(int hd, int rd) {
    return VEC ? (IL ? rd / 8 : rd / 16) + (hd - rd) / 8 : rd / 2 + (hd - rd);
  }
  __device__ __forceinline__ void set(const RotaryArgs& p, int row, int unit) {
    const int rd = p.rotary_size, turning = rd / 2 / kPairs;
    if (unit >= turning) {
      at = rd + (unit - turning) * (VEC ? 8 : 1);
      other = -1;
      return;
    }
    const int pair = unit * kPairs;
    at = IL ? 2 * pair : pair;
    other = IL ? at : at + rd / 2;
    const int64_t pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[row]
                                      : static_cast<const int32_t*>(p.positions)[row];
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      const uint64_t turns = (uint64_t)p.turns[pair + e] * (uint64_t)pos + (1u << 31);
      const float half_turns = (float)(int32_t)(turns >> 32) * 0x1p-31f;
      float s, c;
      sincospif(half_turns, &s, &c);
      cs[e] = c * p.magnitude;
      sn[e] = (p.inverse ? -s : s) * p.magnitude;
    }
  }
  // STREAM: the source is read once
  template <bool BF, bool STREAM>
  __device__ __forceinline__ void apply(const uint16_t* src, uint16_t* dst) const {
    if constexpr (!VEC) {
      if (other < 0) {
        dst[at] = src[at];
        return;
      }
      const int j = IL ? at + 1 : other;
      const float a = unpack16<BF>(src[at], 0), b = unpack16<BF>(src[j], 0);
      dst[at] = (uint16_t)pack16<BF>(a * cs[0] - b * sn[0], 0.f);
      dst[j] = (uint16_t)pack16<BF>(b * cs[0] + a * sn[0], 0.f);
    } else {
      const u4 x = STREAM ? stream_load(src + at) : *(const u4*)(src + at);
      if (other < 0) {
        *(u4*)(dst + at) = x;
      } else if constexpr (IL) {
        u4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = unpack16<BF>(x[e], 0), b = unpack16<BF>(x[e], 1);
          o[e] = pack16<BF>(a * cs[e] - b * sn[e], b * cs[e] + a * sn[e]);
        }
        *(u4*)(dst + at) = o;
      } else {
        const u4 y = STREAM ? stream_load(src + other) : *(const u4*)(src + other);
        u4 o, q;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float r[2], s[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float a = unpack16<BF>(x[e], i), b = unpack16<BF>(y[e], i);
            r[i] = a * cs[2 * e + i] - b * sn[2 * e + i];
            s[i] = b * cs[2 * e + i] + a * sn[2 * e + i];
          }
          o[e] = pack16<BF>(r[0], r[1]);
          q[e] = pack16<BF>(s[0], s[1]);
        }
        *(u4*)(dst + at) = o;
        *(u4*)(dst + other) = q;
      }
    }
  }
};

// Heads [first, end) of all (the query heads, then the keys' where they are asked for).
template <bool BF, bool VEC, bool IL>
__device__ __forceinline__ void rotate_heads(const RotaryArgs& p, int64_t item, int first, int end) {
  const int units = Turn<VEC, IL>::units(p.head_size, p.rotary_size);
  const int64_t row64 = item / units;
  if (row64 >= p.rows) return;
  const int row = (int)row64;
  Turn<VEC, IL> turn;
  turn.set(p, row, (int)(item - row64 * units));
  for (int h = first; h < end; ++h) {
    const bool is_q = h < p.heads;
    const int64_t hh = (int64_t)(is_q ? h : h - p.heads) * p.head_size;
    turn.template apply<BF, true>((is_q ? p.q + row * p.q_stride : p.k + row * p.k_stride) + hh,
                            (is_q ? p.q_out + row * p.qo_stride : p.k_out + row * p.ko_stride) + hh);
  }
}

template <bool BF, bool VEC, bool IL>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs p, int each) {
  const int all = p.heads + p.kv_heads, first = blockIdx.y * each;
  rotate_heads<BF, VEC, IL>(p, (int64_t)blockIdx.x * kThreads + threadIdx.x, first, min(first + each, all));
}

// Tokens a workgroup of the cache's part: `tile` of them (at most kTile), and up to seven behind
// them, which complete a run of eight slots.
constexpr int kTile = 32, kHalo = 7;

// Workgroups [0, q_groups) turn query heads; the others one kv head of a tile of tokens:
// keys turned in LDS and stored as 16-byte units, eight tokens x 8 units a wave; values
// turned around in LDS, so that eight tokens in consecutive slots from a multiple of 8 on
// move as one 16-byte unit per dim (such a run belongs to the tile of its first token),
// the others as 2-byte elements.
template <bool BF, bool VEC, bool IL>
__global__ void __launch_bounds__(kThreads) rotary_cache_kernel(RotaryArgs p, int each, int q_groups, int q_blocks, int tile) {
  extern __shared__ __attribute__((aligned(16))) uint16_t sm[];
  __shared__ int64_t slot_s[kHalo + kTile + kHalo];  // of tokens t0 - 7 on; -1: none
  __shared__ int run_s[kTile], single_s[kTile];      // tokens at which a run of eight starts; by themselves
  __shared__ int count_s[2];
  const int hd = p.head_size, tid = threadIdx.x;
  if ((int)blockIdx.x < q_groups * q_blocks) {
    const int first = (int)blockIdx.x / q_blocks * each;
    rotate_heads<BF, VEC, IL>(p, (int64_t)((int)blockIdx.x % q_blocks) * kThreads + tid, first, min(first + each, p.heads));
    return;
  }
  const int wg = blockIdx.x - q_groups * q_blocks;
  const int head = wg % p.kv_heads, t0 = wg / p.kv_heads * tile;
  const int kpitch = hd + 8, vpitch = hd + 2;
  uint16_t* const ktile = sm;                   // [tile][kpitch]
  uint16_t* const vtile = sm + tile * kpitch;   // [tile + kHalo][vpitch]
  const int64_t limit = (int64_t)p.num_blocks * p.block_size;
  if (tid < tile + 2 * kHalo) {
    const int t = t0 - kHalo + tid;
    int64_t s = t >= 0 && t < p.rows ? p.slots[t] : -1;
    if (s < 0 || s >= limit) s = -1;
    slot_s[tid] = s;
  }
  // keys
  const int units = Turn<VEC, IL>::units(hd, p.rotary_size);
  for (int i = tid; i < tile * units; i += kThreads) {
    const int t = i / units;
    if (t0 + t >= p.rows) break;
    Turn<VEC, IL> turn;
    turn.set(p, t0 + t, i - t * units);
    turn.template apply<BF, true>(p.k + (t0 + t) * p.k_stride + (int64_t)head * hd, ktile + t * kpitch);
  }
  __syncthreads();
  if (tid < 64) {  // the first wave lists both
    int run = 0;
    if (tid < tile && slot_s[kHalo + tid] >= 0) {
      const int64_t s = slot_s[kHalo + tid], from = s & ~(int64_t)7;
      const int at = kHalo + tid - (int)(s & 7);  // the run's first token, if it is one
      bool whole = ((uint64_t)p.vptr[s / p.block_size] & 15) == 0;
      for (int e = 0; e < 8; ++e) whole = whole && slot_s[at + e] == from + e;
      run = !whole ? 2 : at == kHalo + tid ? 1 : 0;
    }
    const uint64_t runs = __ballot(run == 1), singles = __ballot(run == 2), before = (1ull << tid) - 1;
    if (run == 1) run_s[__popcll(runs & before)] = tid;
    if (run == 2) single_s[__popcll(singles & before)] = tid;
    if (tid == 0) {
      count_s[0] = __popcll(runs);
      count_s[1] = __popcll(singles);
    }
  }
  // values: of the tile, and of the tokens behind it that its last run needs
  const int nu = hd / 8;
  for (int i = tid; i < (tile + kHalo) * nu; i += kThreads) {
    const int t = i / nu, u = i - t * nu;
    if (t0 + t >= p.rows) break;
    const u4 v = *(const u4*)(p.v + (t0 + t) * p.v_stride + (int64_t)head * hd + u * 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) *(uint32_t*)(vtile + t * vpitch + u * 8 + 2 * e) = v[e];
  }
  __syncthreads();
  const int bs = p.block_size;
  for (int i = tid; i < tile * nu; i += kThreads) {
    // eight tokens by eight units a wave, where there are so many
    const int t = i % tile, u = i / tile;
    const int64_t s = slot_s[kHalo + t];
    if (s < 0) continue;
    uint16_t* unit = reinterpret_cast<uint16_t*>(p.kptr[s / bs]) + (int64_t)head * p.kv_head_stride + (u * bs + (int)(s % bs)) * 8;
    const u4 v = *(const u4*)(ktile + t * kpitch + u * 8);
    if ((reinterpret_cast<uintptr_t>(unit) & 15) == 0) {
      *(u4*)unit = v;
    } else {
      for (int e = 0; e < 8; ++e) unit[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  }
  auto place = [&](int t, int d) {
    const int64_t s = slot_s[kHalo + t];
    return reinterpret_cast<uint16_t*>(p.vptr[s / bs]) + (int64_t)head * p.kv_head_stride + d * bs + (int)(s % bs);
  };
  const int runs = count_s[0], singles = count_s[1];
  for (int i = tid; i < runs * (hd / 2); i += kThreads) {
    const int t = run_s[i % runs], d = i / runs * 2;
    uint16_t* dst = place(t, d);
    const uint16_t* src = vtile + t * vpitch + d;
    u4 lo, hi;  // eight tokens of the even and of the odd dim
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t a = *(const uint32_t*)(src + 2 * e * vpitch), b = *(const uint32_t*)(src + (2 * e + 1) * vpitch);
      lo[e] = (a & 0xFFFFu) | (b << 16);
      hi[e] = (a >> 16) | (b & 0xFFFF0000u);
    }
    *(u4*)dst = lo;
    *(u4*)(dst + bs) = hi;
  }
  for (int i = tid; i < singles * (hd / 2); i += kThreads) {
    const int t = single_s[i % singles], d = i / singles * 2;
    uint16_t* dst = place(t, d);
    const uint32_t v = *(const uint32_t*)(vtile + t * vpitch + d);
    dst[0] = (uint16_t)v;
    dst[bs] = (uint16_t)(v >> 16);
  }
}

// Whether 16-byte units of rows can be turned as they stand.
bool whole_units(const RotaryArgs& a) { return a.rotary_size % (a.interleaved ? 8 : 16) == 0; }
int host_units(const RotaryArgs& a) {
  const int hd = a.head_size, rd = a.rotary_size;
  if (!whole_units(a)) return rd / 2 + (hd - rd);
  return (a.interleaved ? rd / 8 : rd / 16) + (hd - rd) / 8;
}

// Heads a thread turns: as many as leave `want` waves, since each group of heads takes the sines anew.
int heads_each(const RotaryArgs& a, int heads, int want) {
  const int64_t waves = ((int64_t)a.rows * host_units(a) + 63) / 64;
  const int64_t groups = std::max<int64_t>(1, std::min<int64_t>(heads, (want + waves - 1) / waves));
  return (int)((heads + groups - 1) / groups);
}

template <bool BF, bool VEC, bool IL>
hipError_t launch_plain(const RotaryArgs& a, hipStream_t stream) {
  const int all = a.heads + a.kv_heads, each = heads_each(a, all, 16384);
  const int64_t blocks = ((int64_t)a.rows * host_units(a) + kThreads - 1) / kThreads;
  rotary_kernel<BF, VEC, IL><<<dim3((unsigned)blocks, (all + each - 1) / each), kThreads, 0, stream>>>(a, each);
  return hipGetLastError();
}
template <bool BF, bool VEC, bool IL>
hipError_t launch_cache(const RotaryArgs& a, hipStream_t stream) {
  const int each = heads_each(a, a.heads, 4096);
  const int64_t q_blocks = ((int64_t)a.rows * host_units(a) + kThreads - 1) / kThreads;
  const int q_groups = (a.heads + each - 1) / each;
  // Tiles of 32 rows write whole lines of the value cache; of 8 where those would leave fewer than two
  // workgroups per CU.  Measured, heads of 128: 48 rows of 8 kv heads 5.3 us by 8 and 8.3 by 32, 1024 of 8
  // 11.1 and 11.6, 512 of 32 12.3 and 11.4, 2048 of 8 16.6 and 14.1, 4096 of 32 66.5 and 45.9.  Heads above
  // 256 halve the tile: LDS, 37 KiB at heads of 256.
  const bool few = (int64_t)a.rows / kTile * a.kv_heads < 512;
  const int tile = few ? kTile / 4 : a.head_size > 256 ? kTile / 2 : kTile;
  const int64_t kv = (int64_t)((a.rows + tile - 1) / tile) * a.kv_heads;
  const size_t smem = 2 * ((size_t)tile * (a.head_size + 8) + (size_t)(tile + kHalo) * (a.head_size + 2));
  rotary_cache_kernel<BF, VEC, IL>
      <<<(unsigned)(q_blocks * q_groups + kv), kThreads, smem, stream>>>(a, each, q_groups, (int)q_blocks, tile);
  return hipGetLastError();
}

template <typename F>
hipError_t by_form(const RotaryArgs& a, F&& f) {
  const int form = a.bf16 * 4 + whole_units(a) * 2 + a.interleaved;
  return f(form);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream) {
  using Launch = hipError_t (*)(const RotaryArgs&, hipStream_t);
  static constexpr Launch kForms[8] = {
      &launch_plain<false, false, false>, &launch_plain<false, false, true>, &launch_plain<false, true, false>,
      &launch_plain<false, true, true>,   &launch_plain<true, false, false>, &launch_plain<true, false, true>,
      &launch_plain<true, true, false>,   &launch_plain<true, true, true>};
  return by_form(a, [&](int i) { return kForms[i](a, stream); });
}
hipError_t launch_rotary_cache(const RotaryArgs& a, hipStream_t stream) {
  using Launch = hipError_t (*)(const RotaryArgs&, hipStream_t);
  static constexpr Launch kForms[8] = {
      &launch_cache<false, false, false>, &launch_cache<false, false, true>, &launch_cache<false, true, false>,
      &launch_cache<false, true, true>,   &launch_cache<true, false, false>, &launch_cache<true, false, true>,
      &launch_cache<true, true, false>,   &launch_cache<true, true, true>};
  return by_form(a, [&](int i) { return kForms[i](a, stream); });
}

}  // namespace dw4
