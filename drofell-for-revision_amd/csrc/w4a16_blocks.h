// Internal interface of the cache-block pool's kernels (w4a16_blocks.hip) for
// the C ABI (w4a16_capi_window.hip).  Not installed; the public ABI is
// include/drofell_w4a16.h.
#pragma once

#include "w4a16_internal.h"

namespace dw4 {

struct PoolArgs {
  // the layers' blocks: addresses of each layer's pointer tables (device)
  int layers;
  const int64_t* key_tables;
  const int64_t* value_tables;
  int64_t part_bytes;  // of a block's keys, and of its values
  int num_blocks, rows, max_blocks, block_size;
  const int32_t* tables;  // [rows][max_blocks]
  const int32_t* lens;
  const int32_t* refs;  // [num_blocks]
  int32_t* tables_out;
  int32_t* lens_out;
  int32_t* refs_out;
  int32_t* shortage;
  const int32_t* by_row;    // extend: tokens to add; fork: parents
  const uint8_t* finished;  // free: rows that end, or null
  int window, sinks;        // free
  int32_t* live;            // compact
  int32_t* ws;
};
// Workspace: ints of the lists that a call's first kernel leaves for its second.
constexpr int kPoolHead = 16;  // [0]: blocks to copy, [1]: live blocks
inline size_t pool_ws_ints(int rows, int num_blocks) {
  return (size_t)kPoolHead + 4 * (size_t)rows + 4 * (size_t)num_blocks + 16;
}
constexpr int kPoolMaxRows = 8192;   // a fork keeps one LDS word per row

// Positions and cache slots of rows' last tokens.
struct SlotArgs {
  int rows, max_blocks, num_blocks, block_size, num_tokens;
  const int32_t* tables;  // [rows][max_blocks]
  const int32_t* lens;
  const int32_t* new_tokens;  // [rows]
  int32_t* starts;            // [rows + 1]
  int32_t* positions;         // [num_tokens]
  int64_t* slots;
  int32_t* row_of;
  int32_t* excess;            // [1]
};
constexpr int kSlotMaxRows = 8192;  // each workgroup keeps the rows' starts in LDS

hipError_t launch_token_slots(const SlotArgs& a, hipStream_t stream);
hipError_t launch_copy_blocks(const PoolArgs& a, int count, const int32_t* pairs, int cus, hipStream_t stream);
hipError_t launch_extend_blocks(const PoolArgs& a, hipStream_t stream);
hipError_t launch_fork_blocks(const PoolArgs& a, int cus, hipStream_t stream);
hipError_t launch_free_blocks(const PoolArgs& a, hipStream_t stream);
hipError_t launch_compact_blocks(const PoolArgs& a, int cus, hipStream_t stream);

}  // namespace dw4
