// The cache-block pool: blocks copied, given to rows that grow, shared by forked
// rows, given back and moved together, with tables, lengths and reference counts
// on the device throughout, so that no step of a serving loop waits for the host.
//
// A pool's state is a table of block numbers per row (-1: none), the rows'
// lengths and, per block, how many table entries hold it (0: free).  Every call
// reads one state and writes another.  Which block goes where is fixed by the
// state alone: free blocks are handed out from the lowest number up, in the
// order of rows; counts are integer sums.
//
// Each of extend, fork and compact is two launches.  In the first, one workgroup of
// 1024 threads reads the counts (each wave a run of them, ranks by ballot after one
// scan over the waves' sums) and lists the blocks to hand out or to move, while others copy
// the state's unchanged parts.  The second applies the lists to the tables and counts
// and, where blocks' contents move, copies them in every layer: 16-byte units,
// 16 KiB of one block at a time per workgroup, as many workgroups as stay
// resident, so that the number of blocks need not be known to the host.
// Bound by memory where contents move, else by the launches.  Measured: 150 blocks of
// 32 tokens, 32 heads of 128, copied in 3 layers 96 us, 4.9 TB/s read and written (a 1 GiB
// copy 5.1); 2000 blocks of 8 heads compacted in 4 layers 105 us after a plan of 8; the plans
// of fork (1200 blocks) 6 us, of extend (30000 blocks) 15, their second launches 4.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "w4a16_blocks.h"
#include "w4a16_device.h"

namespace dw4 {

namespace {

constexpr int kPlanThreads = 1024, kThreads = 256;
constexpr int kItem = kThreads * 4 * 16;  // bytes that a workgroup copies at a time

// Exclusive sum over the workgroup's threads (kPlanThreads), and the total.
__device__ __forceinline__ int64_t scan(int64_t v, int64_t* tmp, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    const int64_t t = tmp[w];
    if (w < wave) before += t;
    total += t;
  }
  return before + x - v;
}

__device__ __forceinline__ int up(int64_t tokens, int bs) { return (int)min<int64_t>((tokens + bs - 1) / bs, INT_MAX); }

__device__ __forceinline__ bool is_block(const PoolArgs& a, int e) { return e >= 0 && e < a.num_blocks; }

// The counts in ascending order of blocks: each wave takes one run of them, 256 at
// a time; f(first, counts, which): lane l has the counts of blocks first + l + 64 e, e
// = 0 .. 3, and bit e of `which` says that there is such a block.
template <typename F>
__device__ __forceinline__ void sweep(const int32_t* __restrict__ refs, int n, F&& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int run = (n + 256 * (kPlanThreads / 64) - 1) / (256 * (kPlanThreads / 64)) * 256;
  const int to = min(n, (wave + 1) * run);
#pragma unroll 4
  for (int p = wave * run; p < to; p += 256) {
    int v[4], which = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = p + 64 * e + lane;
      which |= (at < to) << e;
      v[e] = at < to ? refs[at] : 0;
    }
    f(p, v, which);
  }
}
// How many blocks of the pool are free (LIVE: held), and of those before the wave's run.
template <bool LIVE>
__device__ __forceinline__ int64_t count_blocks(const int32_t* __restrict__ refs, int n, int64_t* tmp, int64_t& total) {
  int64_t own = 0;
  sweep(refs, n, [&](int, const int (&v)[4], int which) {
#pragma unroll
    for (int e = 0; e < 4; ++e) own += (which >> e & 1) && (LIVE ? v[e] > 0 : v[e] == 0);
  });
  const int64_t before = scan(own, tmp, total);
  return __shfl(before, 0);  // of the wave's first lane
}
// f(rank, block) of every free (LIVE: held) block, by its rank among them.
template <bool LIVE, typename F>
__device__ __forceinline__ void rank_blocks(const int32_t* __restrict__ refs, int n, int64_t before, F&& f) {
  const int lane = threadIdx.x & 63;
  sweep(refs, n, [&](int p, const int (&v)[4], int which) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = (which >> e & 1) && (LIVE ? v[e] > 0 : v[e] == 0);
      const uint64_t all = __ballot(in);
      if (in) f(before + __popcll(all & ((1ull << lane) - 1)), p + 64 * e + lane);
      before += __popcll(all);
    }
  });
}

// The workgroups beside the planning one copy n ints.
__device__ __forceinline__ void copy_ints(int32_t* dst, const int32_t* src, int64_t n) {
  for (int64_t i = (int64_t)(blockIdx.x - 1) * kPlanThreads + threadIdx.x; i < n;
       i += (int64_t)(gridDim.x - 1) * kPlanThreads)
    dst[i] = src[i];
}

__device__ __forceinline__ int clamp_int(int64_t v) { return (int)min<int64_t>(v, INT_MAX); }

// ---- contents

// Items of kItem bytes of the pairs' keys and values in every layer, by `wg` of `wgs` workgroups.
__device__ __forceinline__ void copy_pairs(const PoolArgs& a, const int32_t* pairs, int count, int64_t wg, int64_t wgs) {
  const int chunks = (int)((a.part_bytes + kItem - 1) / kItem);
  const int64_t items = (int64_t)count * a.layers * 2 * chunks;
  for (int64_t i = wg; i < items; i += wgs) {
    const int chunk = (int)(i % chunks);
    const int64_t j = i / chunks;
    const int part = (int)(j % (2 * a.layers));
    const int64_t k = j / (2 * a.layers);
    const int src = pairs[2 * k], dst = pairs[2 * k + 1];
    if (!is_block(a, src) || !is_block(a, dst) || src == dst) continue;
    const int64_t* table = reinterpret_cast<const int64_t*>((part & 1 ? a.value_tables : a.key_tables)[part >> 1]);
    const unsigned char* from = reinterpret_cast<const unsigned char*>(table[src]) + (int64_t)chunk * kItem;
    unsigned char* to = reinterpret_cast<unsigned char*>(table[dst]) + (int64_t)chunk * kItem;
    const int64_t left = a.part_bytes - (int64_t)chunk * kItem;
    u4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = (u * kThreads + threadIdx.x) * 16;
      if (at < left) v[u] = *(const u4*)(from + at);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = (u * kThreads + threadIdx.x) * 16;
      if (at < left) *(u4*)(to + at) = v[u];
    }
  }
}

__global__ void __launch_bounds__(kThreads) copy_blocks_kernel(PoolArgs a, int count, const int32_t* __restrict__ pairs) {
  copy_pairs(a, pairs, count, blockIdx.x, gridDim.x);
}

// ---- extend: workspace [head][offset per row][blocks handed out]

__global__ void __launch_bounds__(kPlanThreads) extend_plan_kernel(PoolArgs a) {
  if (blockIdx.x > 0) {
    copy_ints(a.refs_out, a.refs, a.num_blocks);
    copy_ints(a.tables_out, a.tables, (int64_t)a.rows * a.max_blocks);
    return;
  }
  __shared__ int64_t tmp[kPlanThreads / 64];
  int32_t* offset = a.ws + kPoolHead;
  int32_t* list = offset + a.rows;
  int64_t need = 0, wide = 0, total;
  for (int r0 = 0; r0 < a.rows; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    int64_t n = 0;
    if (r < a.rows) {
      const int64_t len = max(a.lens[r], 0);
      const int want = up(len + max(a.by_row[r], 0), a.block_size);
      n = want - up(len, a.block_size);
      wide += max(want - a.max_blocks, 0);
    }
    const int64_t before = scan(n, tmp, total);
    if (r < a.rows) offset[r] = clamp_int(need + before);
    need += total;
  }
  scan(wide, tmp, total);
  const int64_t beyond = total;
  const int64_t before = count_blocks<false>(a.refs, a.num_blocks, tmp, total);
  if (before < need)
    rank_blocks<false>(a.refs, a.num_blocks, before, [&](int64_t k, int p) {
      if (k < need) list[k] = p;
    });
  if (threadIdx.x == 0) a.shortage[0] = clamp_int(max<int64_t>(need - total, 0) + beyond);
}

__global__ void __launch_bounds__(kThreads) extend_apply_kernel(PoolArgs a) {
  const int r = blockIdx.x;
  const int32_t* offset = a.ws + kPoolHead;
  const int32_t* list = offset + a.rows;
  const int len = a.lens[r], add = max(a.by_row[r], 0);
  const bool ok = a.shortage[0] == 0;
  if (threadIdx.x == 0) a.lens_out[r] = ok ? len + add : len;
  if (!ok) return;
  const int have = up(max(len, 0), a.block_size), want = up((int64_t)max(len, 0) + add, a.block_size);
  for (int b = have + threadIdx.x; b < want; b += kThreads) {
    const int p = list[offset[r] + b - have];
    a.tables_out[(int64_t)r * a.max_blocks + b] = p;
    a.refs_out[p] = 1;
  }
}

// ---- the slots of rows' last tokens: every workgroup sums up the rows' new tokens
// (a few thousand integers from L2, so that one launch does) and maps as many tokens as it has threads, each
// to its row by bisection.  Bound by its launch and three dependent loads: 48 rows of one token 3.6 us, 300
// rows of 128 5.3 us.

__global__ void __launch_bounds__(kPlanThreads) token_slots_kernel(SlotArgs a) {
  extern __shared__ int start[];  // [rows + 1]
  __shared__ int64_t tmp[kPlanThreads / 64];
  int64_t sum = 0, total;
  for (int r0 = 0; r0 < a.rows; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    const int64_t n = r < a.rows ? max(min(a.new_tokens[r], a.lens[r]), 0) : 0;
    const int64_t before = scan(n, tmp, total);
    if (r < a.rows) start[r] = clamp_int(sum + before);
    sum += total;
  }
  const int64_t excess = max<int64_t>(sum - a.num_tokens, 0);
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int r = threadIdx.x; r <= a.rows; r += kPlanThreads)
      a.starts[r] = excess > 0 ? 0 : r < a.rows ? start[r] : (int)sum;
    if (threadIdx.x == 0) a.excess[0] = clamp_int(excess);
  }
  const int t = blockIdx.x * kPlanThreads + threadIdx.x;
  if (t >= a.num_tokens) return;
  int row = -1, pos = 0;
  int64_t slot = -1;
  if (excess == 0 && t < sum) {
    int lo = 0, hi = a.rows - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    row = lo;
    const int len = a.lens[row];
    pos = len - max(min(a.new_tokens[row], len), 0) + t - start[row];
    const int at = pos / a.block_size;
    if (at < a.max_blocks) {
      const int block = a.tables[(int64_t)row * a.max_blocks + at];
      if (block >= 0 && block < a.num_blocks) slot = (int64_t)block * a.block_size + pos % a.block_size;
    }
  }
  a.positions[t] = pos;
  a.slots[t] = slot;
  a.row_of[t] = row;
}

// ---- fork: workspace [head][fresh block per row][rows that need one][pairs]

__device__ __forceinline__ int parent_of(const PoolArgs& a, int r) {
  const int p = a.by_row[r];
  return p >= 0 && p < a.rows ? p : -1;
}

// A row's half-filled last block, -1 if it has none.
__device__ __forceinline__ int last_block(const PoolArgs& a, int row, int& at) {
  const int len = a.lens[row];
  at = len / a.block_size;
  if (len <= 0 || len % a.block_size == 0 || at >= a.max_blocks) return -1;
  const int e = a.tables[(int64_t)row * a.max_blocks + at];
  return is_block(a, e) ? e : -1;
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(PoolArgs a) {
  if (blockIdx.x > 0) {
    copy_ints(a.refs_out, a.refs, a.num_blocks);
    return;
  }
  extern __shared__ int first[];  // [rows] the first row that continues each parent
  __shared__ int64_t tmp[kPlanThreads / 64];
  int32_t* fresh = a.ws + kPoolHead;
  int32_t* needy = fresh + a.rows;
  int32_t* pairs = needy + a.rows;
  for (int r = threadIdx.x; r < a.rows; r += kPlanThreads) first[r] = INT_MAX;
  __syncthreads();
  for (int r = threadIdx.x; r < a.rows; r += kPlanThreads) {
    const int p = parent_of(a, r);
    if (p >= 0) atomicMin(&first[p], r);
  }
  __syncthreads();
  int64_t need = 0, total;
  for (int r0 = 0; r0 < a.rows; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    bool copy = false;
    if (r < a.rows) {
      const int p = parent_of(a, r);
      int at;
      const int e = p >= 0 ? last_block(a, p, at) : -1;
      copy = e >= 0 && (first[p] != r || a.refs[e] > 1);
      fresh[r] = -1;
    }
    const int64_t before = scan(copy, tmp, total);
    if (copy) needy[need + before] = r;
    need += total;
  }
  // (its barriers also publish needy and fresh)
  const int64_t before = count_blocks<false>(a.refs, a.num_blocks, tmp, total);
  if (before < need)
    rank_blocks<false>(a.refs, a.num_blocks, before, [&](int64_t k, int p) {
      if (k >= need) return;
      const int r = needy[k];
      int at;
      pairs[2 * k] = last_block(a, parent_of(a, r), at);
      pairs[2 * k + 1] = p;
      fresh[r] = p;
    });
  if (threadIdx.x == 0) {
    a.shortage[0] = clamp_int(max<int64_t>(need - total, 0));
    a.ws[0] = need > total ? 0 : (int)need;
  }
}

// Workgroups 0 .. rows - 1: a row's table, length and counts; the others: contents.
__global__ void __launch_bounds__(kThreads) fork_apply_kernel(PoolArgs a) {
  const int32_t* fresh = a.ws + kPoolHead;
  if ((int)blockIdx.x >= a.rows) {
    copy_pairs(a, fresh + 2 * a.rows, a.ws[0], blockIdx.x - a.rows, gridDim.x - a.rows);
    return;
  }
  const int r = blockIdx.x;
  const bool ok = a.shortage[0] == 0;
  const int p = ok ? parent_of(a, r) : r;
  const int len = p >= 0 ? a.lens[p] : 0, got = ok ? fresh[r] : -1;
  if (threadIdx.x == 0) a.lens_out[r] = len;
  for (int b = threadIdx.x; b < a.max_blocks; b += kThreads) {
    const int old = a.tables[(int64_t)r * a.max_blocks + b];
    int e = p >= 0 ? a.tables[(int64_t)p * a.max_blocks + b] : -1;
    if (got >= 0 && b == len / a.block_size) e = got;
    a.tables_out[(int64_t)r * a.max_blocks + b] = e;
    if (e == old) continue;
    if (is_block(a, e)) atomicAdd(&a.refs_out[e], 1);
    if (is_block(a, old)) atomicSub(&a.refs_out[old], 1);
  }
}

// ---- free

__global__ void __launch_bounds__(kThreads) copy_ints_kernel(int32_t* __restrict__ dst, const int32_t* __restrict__ src,
                                                             int n, int32_t* __restrict__ zero) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < n) dst[i] = src[i];
  if (i == 0) zero[0] = 0;
}

__global__ void __launch_bounds__(kThreads) free_kernel(PoolArgs a) {
  const int r = blockIdx.x;
  const int len = a.lens[r];
  const bool over = a.finished != nullptr && a.finished[r] != 0;
  // the next token, at position len, sees the tokens after len - window
  const int64_t gone = a.window == 0 ? 0 : (int64_t)len - a.window + 1;
  if (threadIdx.x == 0) a.lens_out[r] = over ? 0 : len;
  for (int b = threadIdx.x; b < a.max_blocks; b += kThreads) {
    int e = a.tables[(int64_t)r * a.max_blocks + b];
    const int64_t t = (int64_t)b * a.block_size;
    if (over || (t + a.block_size <= gone && t >= a.sinks)) {
      if (is_block(a, e)) atomicSub(&a.refs_out[e], 1);
      e = -1;
    }
    a.tables_out[(int64_t)r * a.max_blocks + b] = e;
  }
}

// ---- compact: workspace [head][moved: per block where it goes / comes from][pairs]

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(PoolArgs a) {
  __shared__ int64_t tmp[kPlanThreads / 64];
  int32_t* moved = a.ws + kPoolHead;
  int32_t* pairs = moved + a.num_blocks;
  int64_t live, below, count;
  const int64_t held = count_blocks<true>(a.refs, a.num_blocks, tmp, live);
  // holes below `live` and live blocks from there on: as many of one as of the other
  int64_t own = 0;
  sweep(a.refs, a.num_blocks, [&](int p, const int (&v)[4], int which) {
#pragma unroll
    for (int e = 0; e < 4; ++e) own += (which >> e & 1) && v[e] > 0 && p + 64 * e + (int)(threadIdx.x & 63) < live;
  });
  scan(own, tmp, below);
  count = live - below;
  rank_blocks<true>(a.refs, a.num_blocks, held, [&](int64_t k, int p) {
    if (p >= live) pairs[2 * (k - below)] = p;
  });
  // a hole's rank: the blocks before it less the live ones among them
  const int lane = threadIdx.x & 63;
  int64_t before = held;
  sweep(a.refs, a.num_blocks, [&](int p, const int (&v)[4], int which) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is_live = (which >> e & 1) && v[e] > 0;
      const uint64_t all = __ballot(is_live);
      const int64_t at = p + 64 * e + lane;
      if ((which >> e & 1) && !is_live && at < live) pairs[2 * (at - before - __popcll(all & ((1ull << lane) - 1))) + 1] = (int)at;
      before += __popcll(all);
    }
  });
  __syncthreads();
  for (int64_t k = threadIdx.x; k < count; k += kPlanThreads) {
    moved[pairs[2 * k]] = pairs[2 * k + 1];
    moved[pairs[2 * k + 1]] = pairs[2 * k];
  }
  if (threadIdx.x == 0) {
    a.ws[0] = (int)count;
    a.ws[1] = a.live[0] = (int)live;
    a.shortage[0] = 0;
  }
}

// Workgroups 0 .. heads - 1: tables and counts; the others: contents.
__global__ void __launch_bounds__(kThreads) compact_apply_kernel(PoolArgs a, int heads) {
  const int32_t* moved = a.ws + kPoolHead;
  if ((int)blockIdx.x >= heads) {
    copy_pairs(a, moved + a.num_blocks, a.ws[0], blockIdx.x - heads, gridDim.x - heads);
    return;
  }
  const int live = a.ws[1];
  const int64_t entries = (int64_t)a.rows * a.max_blocks, n = entries + a.num_blocks + a.rows;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)heads * kThreads) {
    if (i < entries) {
      const int e = a.tables[i];
      a.tables_out[i] = is_block(a, e) && e >= live && a.refs[e] > 0 ? moved[e] : e;
    } else if (i < entries + a.num_blocks) {
      const int p = (int)(i - entries), c = a.refs[p];
      a.refs_out[p] = p >= live ? (c > 0 ? 0 : c) : c > 0 ? c : a.refs[moved[p]];
    } else {
      a.lens_out[i - entries - a.num_blocks] = a.lens[i - entries - a.num_blocks];
    }
  }
}

// Workgroups that copy contents: enough to fill the card several times over,
// no more than there are items.
int copy_groups(const PoolArgs& a, int64_t most_pairs, int cus) {
  const int64_t chunks = (a.part_bytes + kItem - 1) / kItem;
  return (int)std::min<int64_t>(most_pairs * a.layers * 2 * chunks, (int64_t)cus * 8);
}

unsigned plan_groups(int64_t ints) { return (unsigned)(1 + std::min<int64_t>(64, (ints + kPlanThreads - 1) / kPlanThreads)); }

}  // namespace

hipError_t launch_token_slots(const SlotArgs& a, hipStream_t stream) {
  const unsigned grid = std::max(1u, ((unsigned)a.num_tokens + kPlanThreads - 1) / kPlanThreads);
  token_slots_kernel<<<grid, kPlanThreads, sizeof(int) * ((size_t)a.rows + 1), stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_copy_blocks(const PoolArgs& a, int count, const int32_t* pairs, int cus, hipStream_t stream) {
  copy_blocks_kernel<<<(unsigned)copy_groups(a, count, cus), kThreads, 0, stream>>>(a, count, pairs);
  return hipGetLastError();
}

hipError_t launch_extend_blocks(const PoolArgs& a, hipStream_t stream) {
  extend_plan_kernel<<<plan_groups((int64_t)a.rows * a.max_blocks + a.num_blocks), kPlanThreads, 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.rows == 0) return e;
  extend_apply_kernel<<<(unsigned)a.rows, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_fork_blocks(const PoolArgs& a, int cus, hipStream_t stream) {
  fork_plan_kernel<<<plan_groups(a.num_blocks), kPlanThreads, sizeof(int) * (size_t)a.rows, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.rows == 0) return e;
  fork_apply_kernel<<<(unsigned)(a.rows + copy_groups(a, a.rows, cus)), kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_free_blocks(const PoolArgs& a, hipStream_t stream) {
  copy_ints_kernel<<<(unsigned)std::max(1, (a.num_blocks + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
      a.refs_out, a.refs, a.num_blocks, a.shortage);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.rows == 0) return e;
  free_kernel<<<(unsigned)a.rows, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_compact_blocks(const PoolArgs& a, int cus, hipStream_t stream) {
  compact_plan_kernel<<<1, kPlanThreads, 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.rows + a.num_blocks == 0) return e;
  const int64_t ints = (int64_t)a.rows * a.max_blocks + a.num_blocks + a.rows;
  const int heads = (int)std::min<int64_t>(256, (ints + kThreads - 1) / kThreads);
  compact_apply_kernel<<<(unsigned)(heads + copy_groups(a, a.num_blocks / 2, cus)), kThreads, 0, stream>>>(a, heads);
  return hipGetLastError();
}

}  // namespace dw4
