// Internal interface of the windowed-attention kernels (w4a16_window*.hip) for
// the C ABI (w4a16_capi_window.hip).  Not installed; the public ABI is
// include/drofell_w4a16.h.
#pragma once

#include "w4a16_internal.h"

namespace dw4 {

// The token at position i of a sequence sees the tokens j <= i with j > i -
// window (window 0: all of them), and those with j < sinks.
struct WindowArgs {
  bool bf16;
  int num_seqs, num_heads, num_kv_heads, head_size;
  const uint16_t* q;  // [rows][num_heads][head_size], q_stride per row
  int64_t q_stride;
  uint16_t* out;
  int64_t o_stride;
  const int32_t* starts;  // [num_seqs + 1] first row of each sequence, null: row s alone
  int total_rows, max_query;
  float scale_log2;  // scale * log2(e): logits in base 2
  int window, sinks;
  // keys and values in cache blocks (block_size 16 or 32) ...
  int block_size, num_blocks;
  const int64_t* kptr;
  const int64_t* vptr;
  int kv_head_stride;
  const int32_t* tables;  // [num_seqs][max_blocks]
  int max_blocks;
  const int32_t* lens;
  // ... or (block_size 0) as rows beside the queries
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_stride, v_stride;
  float* lse;      // [rows][num_heads] log2 of the softmax's sum, or null
  uint16_t* rest;  // [rows][num_heads][head_size] what rounding the output left off, or null
};

// rows: the kernel whose waves share 32 rows and split the tokens; else the
// one whose waves take 32 rows each and share the tokens.
struct WindowPlan {
  bool rows = true;
  int waves = 4;   // per workgroup
  int tiles = 1;   // row tiles per (sequence, kv head)
  int splits = 1;  // parts of the tokens, joined by a second launch
};
constexpr int kWinRowsTile = 32;    // rows of a wave's MFMA columns
constexpr int kWinRowsTokens = 32;  // tokens of a step of the rows kernel
constexpr int kWinTileTokens = 64;  // tokens of a step of the tile kernels
constexpr int kWinMaxWindow = 1 << 30;
// Workgroups that share an XCD (work_of in w4a16_window_device.h), and the grid for them.
constexpr int kWinUnit = 8;
inline unsigned win_grid(int pairs, int items) {
  const int64_t unit = items < kWinUnit ? items : kWinUnit;
  const int64_t units = (items + unit - 1) / unit * pairs;
  return (unsigned)((units + 7) / 8 * 8 * unit);
}

inline size_t win_rows_smem(int hs, int cols, int waves) {
  return sizeof(float) * (size_t)waves * cols * (hs + 2);
}

WindowPlan plan_window(const WindowArgs& a, int max_context, int cus);
// Floats of a split call's maxima and sums, whole 16-byte units; the outputs follow.
inline size_t win_ml_floats(int total_rows, int num_heads, int splits) {
  return (2 * (size_t)total_rows * num_heads * splits + 3) / 4 * 4;
}
size_t window_ws_bytes(const WindowPlan& p, int total_rows, int num_heads, int head_size);
hipError_t launch_window(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream);
// The kernels by storage: rows kernel (blocks), tile kernel (blocks or rows).
template <bool BF>
hipError_t launch_window_rows(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream);
template <bool BF>
hipError_t launch_window_tile(const WindowArgs& a, const WindowPlan& p, float* ws, hipStream_t stream);

// Gradients of the row form.
struct WindowGradArgs {
  WindowArgs f;  // q, k, v, out (read), lse (read)
  const uint16_t* dout;
  int64_t do_stride;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  int64_t dq_stride, dk_stride, dv_stride;
  float scale;
};
size_t window_grad_ws_bytes(const WindowArgs& a);
template <bool BF>
hipError_t launch_window_grad(const WindowGradArgs& a, float* ws, hipStream_t stream);

}  // namespace dw4
