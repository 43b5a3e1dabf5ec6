// Internal interface of the rotary-position kernels (w4a16_rotary.hip) for the C ABI
// (w4a16_capi_adapters.hip).  Not installed; the public ABI is include/drofell_w4a16.h.
#pragma once

#include "w4a16_internal.h"

namespace dw4 {

struct RotaryArgs {
  bool bf16, interleaved, inverse, positions64;
  int rows, heads, kv_heads, head_size, rotary_size;
  const uint16_t* q;
  int64_t q_stride;
  const uint16_t* k;
  int64_t k_stride;
  uint16_t* q_out;
  int64_t qo_stride;
  uint16_t* k_out;          // not with a cache
  int64_t ko_stride;
  const void* positions;    // int32, or int64
  const int64_t* turns;     // [rotary_size / 2]: turns per position, times 2^64
  float magnitude;
  // cache
  const uint16_t* v;
  int64_t v_stride;
  const int64_t* slots;
  const int64_t* kptr;
  const int64_t* vptr;
  int num_blocks, block_size, kv_head_stride;
};

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream);
hipError_t launch_rotary_cache(const RotaryArgs& a, hipStream_t stream);

}  // namespace dw4
