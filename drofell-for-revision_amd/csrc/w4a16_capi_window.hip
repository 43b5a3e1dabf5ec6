// C ABI of the windowed attention and of the cache-block pool (declared in
// include/drofell_w4a16.h): validation and dispatch.  Every entry point returns
// a status code; nothing throws across the ABI.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "drofell_w4a16.h"
#include "w4a16_blocks.h"
#include "w4a16_internal.h"
#include "w4a16_window.h"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int status_of(hipError_t e) { return e == hipSuccess ? DW4_OK : DW4_ERR_LAUNCH; }

int check_window(int dtype, int num_seqs, int num_heads, int num_kv_heads, int head_size, int total_rows,
                 int max_query, int window, int sinks) {
  if (dtype != DW4_F16 && dtype != DW4_BF16) return DW4_ERR_UNSUPPORTED;
  if (num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || total_rows < 0 || max_query < 0 || window < 0 || sinks < 0)
    return DW4_ERR_INVALID_ARG;
  if (num_heads % num_kv_heads != 0) return DW4_ERR_UNSUPPORTED;
  if (head_size != 64 && head_size != 80 && head_size != 96 && head_size != 112 && head_size != 128 && head_size != 256)
    return DW4_ERR_UNSUPPORTED;
  // rows of (token, head) and workgroups are counted in 32 bits
  const int64_t G = num_heads / num_kv_heads;
  if (G > 1024 || (int64_t)total_rows * num_heads > (int64_t)1 << 26) return DW4_ERR_UNSUPPORTED;
  max_query = max_query < total_rows ? max_query : total_rows;  // (a bound that the caller may have taken wide)
  const int64_t tiles = (max_query * G + 31) / 32 + 1;
  if ((int64_t)num_seqs * num_kv_heads > INT32_MAX / 4 || (int64_t)num_seqs * num_kv_heads * tiles > INT32_MAX / 4 ||
      (int64_t)num_seqs * max_query * num_heads > INT32_MAX)
    return DW4_ERR_UNSUPPORTED;
  return DW4_OK;
}

bool good_scale(float s) { return s > 0.f && std::isfinite(s); }

dw4::WindowArgs window_args(int dtype, int num_seqs, int num_heads, int num_kv_heads, int head_size, int total_rows,
                            int max_query, float scale, int window, int sinks) {
  dw4::WindowArgs a = {};
  a.bf16 = dtype == DW4_BF16;
  a.num_seqs = num_seqs;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_size = head_size;
  a.total_rows = total_rows;
  a.max_query = max_query < total_rows ? max_query : total_rows;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = window < dw4::kWinMaxWindow ? window : 0;  // no context is longer
  a.sinks = sinks;
  return a;
}

}  // namespace

extern "C" {

int dw4_window_attention_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_size, int block_size,
                                        int total_rows, int max_query_len, int window, int sinks, int max_context_len,
                                        size_t* workspace_bytes) {
  const int st = check_window(DW4_F16, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_query_len, window, sinks);
  if (st != DW4_OK) return st;
  if (block_size != 16 && block_size != 32) return DW4_ERR_UNSUPPORTED;
  if (workspace_bytes == nullptr || max_context_len < 0) return DW4_ERR_INVALID_ARG;
  dw4::WindowArgs a = window_args(DW4_F16, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_query_len, 1.f,
                                  window, sinks);
  a.block_size = block_size;
  *workspace_bytes = 0;
  if (num_seqs > 0 && a.max_query > 0)
    *workspace_bytes = dw4::window_ws_bytes(dw4::plan_window(a, max_context_len, dw4::cu_count()), total_rows, num_heads, head_size);
  return DW4_OK;
}

int dw4_window_attention(int dtype, int num_seqs, int num_heads, int num_kv_heads, int head_size, int block_size,
                         int num_blocks, const uint16_t* query, int64_t q_stride, uint16_t* out, int64_t o_stride,
                         const int32_t* query_starts, int total_rows, int max_query_len, const int64_t* key_block_ptrs,
                         const int64_t* value_block_ptrs, int kv_head_stride, float scale, int window, int sinks,
                         const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens,
                         int max_context_len, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_window(dtype, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_query_len, window, sinks);
  if (st != DW4_OK) return st;
  if (block_size != 16 && block_size != 32) return DW4_ERR_UNSUPPORTED;
  if (!good_scale(scale) || max_context_len < 0 || max_blocks_per_seq < 0 || num_blocks < 0) return DW4_ERR_INVALID_ARG;
  if (query_starts == nullptr && (total_rows != num_seqs || max_query_len != 1)) return DW4_ERR_INVALID_ARG;
  if (num_seqs == 0 || total_rows == 0 || max_query_len == 0) return DW4_OK;
  if (!query || !out || !context_lens) return DW4_ERR_INVALID_ARG;
  if ((num_blocks > 0 && (!key_block_ptrs || !value_block_ptrs)) || (max_blocks_per_seq > 0 && !block_tables))
    return DW4_ERR_INVALID_ARG;
  const int64_t row = (int64_t)num_heads * head_size;
  if (q_stride < row || o_stride < row || kv_head_stride < block_size * head_size ||
      (int64_t)max_blocks_per_seq * block_size < max_context_len || (int64_t)max_blocks_per_seq * block_size > dw4::kWinMaxWindow)
    return DW4_ERR_INVALID_ARG;
  if (!aligned16(query) || !aligned16(out) || q_stride % 8 != 0 || o_stride % 8 != 0 || kv_head_stride % 8 != 0)
    return DW4_ERR_MISALIGNED;
  dw4::WindowArgs a = window_args(dtype, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_query_len, scale,
                                  window, sinks);
  a.block_size = block_size;
  const dw4::WindowPlan p = dw4::plan_window(a, max_context_len, dw4::cu_count());
  const size_t need = dw4::window_ws_bytes(p, total_rows, num_heads, head_size);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return DW4_ERR_WORKSPACE;
  if (need > 0 && !aligned16(workspace)) return DW4_ERR_MISALIGNED;
  a.q = query;
  a.q_stride = q_stride;
  a.out = out;
  a.o_stride = o_stride;
  a.starts = query_starts;
  a.num_blocks = num_blocks;
  a.kptr = key_block_ptrs;
  a.vptr = value_block_ptrs;
  a.kv_head_stride = kv_head_stride;
  a.tables = block_tables;
  a.max_blocks = max_blocks_per_seq;
  a.lens = context_lens;
  return status_of(dw4::launch_window(a, p, static_cast<float*>(workspace), static_cast<hipStream_t>(stream)));
}

static int dense_args(int dtype, int num_seqs, int num_heads, int num_kv_heads, int head_size, const uint16_t* q,
                      int64_t q_stride, const uint16_t* k, int64_t k_stride, const uint16_t* v, int64_t v_stride,
                      const uint16_t* out, int64_t o_stride, const int32_t* seq_starts, int total_rows, int max_seq_len,
                      float scale, int window, int sinks, dw4::WindowArgs& a) {
  const int st = check_window(dtype, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_seq_len, window, sinks);
  if (st != DW4_OK) return st;
  if (!good_scale(scale)) return DW4_ERR_INVALID_ARG;
  if (num_seqs == 0 || total_rows == 0 || max_seq_len == 0) return DW4_OK;
  if (!q || !k || !v || !out || !seq_starts) return DW4_ERR_INVALID_ARG;
  const int64_t row = (int64_t)num_heads * head_size, kv = (int64_t)num_kv_heads * head_size;
  if (q_stride < row || o_stride < row || k_stride < kv || v_stride < kv) return DW4_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || q_stride % 8 != 0 || k_stride % 8 != 0 ||
      v_stride % 8 != 0 || o_stride % 8 != 0)
    return DW4_ERR_MISALIGNED;
  a = window_args(dtype, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_seq_len, scale, window, sinks);
  a.q = q;
  a.q_stride = q_stride;
  a.k = k;
  a.k_stride = k_stride;
  a.v = v;
  a.v_stride = v_stride;
  a.out = const_cast<uint16_t*>(out);
  a.o_stride = o_stride;
  a.starts = seq_starts;
  return DW4_OK;
}

int dw4_window_attention_dense(int dtype, int num_seqs, int num_heads, int num_kv_heads, int head_size,
                               const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
                               const uint16_t* v, int64_t v_stride, uint16_t* out, int64_t o_stride, float* lse, uint16_t* out_rest,
                               const int32_t* seq_starts, int total_rows, int max_seq_len, float scale, int window,
                               int sinks, void* stream) {
  dw4::WindowArgs a = {};
  const int st = dense_args(dtype, num_seqs, num_heads, num_kv_heads, head_size, q, q_stride, k, k_stride, v, v_stride, out,
                            o_stride, seq_starts, total_rows, max_seq_len, scale, window, sinks, a);
  if (st != DW4_OK || a.q == nullptr) return st;
  if ((lse == nullptr) != (out_rest == nullptr)) return DW4_ERR_INVALID_ARG;
  if (!aligned16(out_rest)) return DW4_ERR_MISALIGNED;
  a.lse = lse;
  a.rest = out_rest;
  return status_of(dw4::launch_window(a, dw4::plan_window(a, a.max_query, dw4::cu_count()), nullptr,
                                      static_cast<hipStream_t>(stream)));
}

int dw4_window_attention_dense_backward_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_size,
                                                       int total_rows, int max_seq_len, int window, int sinks,
                                                       size_t* workspace_bytes) {
  const int st = check_window(DW4_F16, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_seq_len, window, sinks);
  if (st != DW4_OK) return st;
  if (workspace_bytes == nullptr) return DW4_ERR_INVALID_ARG;
  *workspace_bytes = 0;
  if (num_seqs > 0 && total_rows > 0 && max_seq_len > 0)
    *workspace_bytes = dw4::window_grad_ws_bytes(
        window_args(DW4_F16, num_seqs, num_heads, num_kv_heads, head_size, total_rows, max_seq_len, 1.f, window, sinks));
  return DW4_OK;
}

int dw4_window_attention_dense_backward(int dtype, int num_seqs, int num_heads, int num_kv_heads, int head_size,
                                        const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
                                        const uint16_t* v, int64_t v_stride, const uint16_t* out, int64_t o_stride,
                                        const float* lse, const uint16_t* out_rest, const uint16_t* dout, int64_t do_stride, uint16_t* dq,
                                        int64_t dq_stride, uint16_t* dk, int64_t dk_stride, uint16_t* dv,
                                        int64_t dv_stride, const int32_t* seq_starts, int total_rows, int max_seq_len,
                                        float scale, int window, int sinks, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  dw4::WindowGradArgs g = {};
  const int st = dense_args(dtype, num_seqs, num_heads, num_kv_heads, head_size, q, q_stride, k, k_stride, v, v_stride, out,
                            o_stride, seq_starts, total_rows, max_seq_len, scale, window, sinks, g.f);
  if (st != DW4_OK || g.f.q == nullptr) return st;
  if (!lse || !out_rest || !dout || !dq || !dk || !dv) return DW4_ERR_INVALID_ARG;
  const int64_t row = (int64_t)num_heads * head_size, kv = (int64_t)num_kv_heads * head_size;
  if (do_stride < row || dq_stride < row || dk_stride < kv || dv_stride < kv) return DW4_ERR_INVALID_ARG;
  if (!aligned16(out_rest) || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || do_stride % 8 != 0 || dq_stride % 8 != 0 ||
      dk_stride % 8 != 0 || dv_stride % 8 != 0)
    return DW4_ERR_MISALIGNED;
  const size_t need = dw4::window_grad_ws_bytes(g.f);
  if (workspace == nullptr || workspace_bytes < need) return DW4_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DW4_ERR_MISALIGNED;
  g.f.lse = const_cast<float*>(lse);
  g.f.rest = const_cast<uint16_t*>(out_rest);
  g.dout = dout;
  g.do_stride = do_stride;
  g.dq = dq;
  g.dk = dk;
  g.dv = dv;
  g.dq_stride = dq_stride;
  g.dk_stride = dk_stride;
  g.dv_stride = dv_stride;
  g.scale = scale;
  auto launch = g.f.bf16 ? &dw4::launch_window_grad<true> : &dw4::launch_window_grad<false>;
  return status_of(launch(g, static_cast<float*>(workspace), static_cast<hipStream_t>(stream)));
}

// ---- the block pool

int dw4_blocks_workspace_size(int num_rows, int num_blocks, size_t* workspace_bytes) {
  if (num_rows < 0 || num_blocks < 0 || workspace_bytes == nullptr) return DW4_ERR_INVALID_ARG;
  *workspace_bytes = sizeof(int32_t) * dw4::pool_ws_ints(num_rows, num_blocks);
  return DW4_OK;
}

static int pool_layers(dw4::PoolArgs& a, int num_layers, const int64_t* kp, const int64_t* vp, int num_blocks,
                       int64_t part_bytes) {
  if (num_layers < 0 || num_blocks < 0 || part_bytes < 0) return DW4_ERR_INVALID_ARG;
  if (num_layers > 0 && (!kp || !vp || part_bytes == 0)) return DW4_ERR_INVALID_ARG;
  if (part_bytes % 16 != 0) return DW4_ERR_MISALIGNED;
  a.layers = num_layers;
  a.key_tables = kp;
  a.value_tables = vp;
  a.num_blocks = num_blocks;
  a.part_bytes = part_bytes;
  return DW4_OK;
}

static int pool_state(dw4::PoolArgs& a, int num_rows, int max_blocks, int num_blocks, const int32_t* tables,
                      const int32_t* lens, const int32_t* refs, int32_t* tables_out, int32_t* lens_out, int32_t* refs_out,
                      int32_t* shortage) {
  if (num_rows < 0 || max_blocks < 0 || num_blocks < 0 || !shortage) return DW4_ERR_INVALID_ARG;
  if (num_rows > 0 && (!lens || !lens_out || lens == lens_out)) return DW4_ERR_INVALID_ARG;
  if (num_rows > 0 && max_blocks > 0 && (!tables || !tables_out || tables == tables_out)) return DW4_ERR_INVALID_ARG;
  if (num_blocks > 0 && (!refs || !refs_out || refs == refs_out)) return DW4_ERR_INVALID_ARG;
  if (num_blocks > 1 << 28 || num_rows > 1 << 24) return DW4_ERR_UNSUPPORTED;
  a.rows = num_rows;
  a.max_blocks = max_blocks;
  a.num_blocks = num_blocks;
  a.tables = tables;
  a.lens = lens;
  a.refs = refs;
  a.tables_out = tables_out;
  a.lens_out = lens_out;
  a.refs_out = refs_out;
  a.shortage = shortage;
  return DW4_OK;
}

static int pool_workspace(dw4::PoolArgs& a, void* workspace, size_t workspace_bytes) {
  if (workspace == nullptr || workspace_bytes < sizeof(int32_t) * dw4::pool_ws_ints(a.rows, a.num_blocks))
    return DW4_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DW4_ERR_MISALIGNED;
  a.ws = static_cast<int32_t*>(workspace);
  return DW4_OK;
}

static bool good_block(int block_size) { return block_size == 16 || block_size == 32; }

int dw4_copy_blocks(int num_layers, const int64_t* layer_key_ptrs, const int64_t* layer_value_ptrs, int num_blocks,
                    int64_t part_bytes, int count, const int32_t* pairs, void* stream) {
  dw4::PoolArgs a = {};
  const int st = pool_layers(a, num_layers, layer_key_ptrs, layer_value_ptrs, num_blocks, part_bytes);
  if (st != DW4_OK) return st;
  if (count < 0 || (count > 0 && !pairs)) return DW4_ERR_INVALID_ARG;
  if (count == 0 || num_layers == 0) return DW4_OK;
  return status_of(dw4::launch_copy_blocks(a, count, pairs, dw4::cu_count(), static_cast<hipStream_t>(stream)));
}

int dw4_extend_blocks(int num_rows, int max_blocks, int num_blocks, int block_size, const int32_t* tables,
                      const int32_t* lens, const int32_t* refs, const int32_t* add, int32_t* tables_out, int32_t* lens_out,
                      int32_t* refs_out, int32_t* shortage, void* workspace, size_t workspace_bytes, void* stream) {
  dw4::PoolArgs a = {};
  int st = pool_state(a, num_rows, max_blocks, num_blocks, tables, lens, refs, tables_out, lens_out, refs_out, shortage);
  if (st != DW4_OK) return st;
  if (!good_block(block_size)) return DW4_ERR_UNSUPPORTED;
  if (num_rows > 0 && !add) return DW4_ERR_INVALID_ARG;
  if ((st = pool_workspace(a, workspace, workspace_bytes)) != DW4_OK) return st;
  a.block_size = block_size;
  a.by_row = add;
  return status_of(dw4::launch_extend_blocks(a, static_cast<hipStream_t>(stream)));
}

int dw4_fork_blocks(int num_layers, const int64_t* layer_key_ptrs, const int64_t* layer_value_ptrs, int64_t part_bytes,
                    int num_rows, int max_blocks, int num_blocks, int block_size, const int32_t* tables,
                    const int32_t* lens, const int32_t* refs, const int32_t* parents, int32_t* tables_out,
                    int32_t* lens_out, int32_t* refs_out, int32_t* shortage, void* workspace, size_t workspace_bytes,
                    void* stream) {
  dw4::PoolArgs a = {};
  int st = pool_state(a, num_rows, max_blocks, num_blocks, tables, lens, refs, tables_out, lens_out, refs_out, shortage);
  if (st == DW4_OK) st = pool_layers(a, num_layers, layer_key_ptrs, layer_value_ptrs, num_blocks, part_bytes);
  if (st != DW4_OK) return st;
  if (!good_block(block_size) || num_rows > dw4::kPoolMaxRows) return DW4_ERR_UNSUPPORTED;
  if (num_rows > 0 && !parents) return DW4_ERR_INVALID_ARG;
  if ((st = pool_workspace(a, workspace, workspace_bytes)) != DW4_OK) return st;
  a.block_size = block_size;
  a.by_row = parents;
  return status_of(dw4::launch_fork_blocks(a, dw4::cu_count(), static_cast<hipStream_t>(stream)));
}

int dw4_free_blocks(int num_rows, int max_blocks, int num_blocks, int block_size, const int32_t* tables,
                    const int32_t* lens, const int32_t* refs, const uint8_t* finished, int window, int sinks,
                    int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int32_t* shortage, void* stream) {
  dw4::PoolArgs a = {};
  const int st = pool_state(a, num_rows, max_blocks, num_blocks, tables, lens, refs, tables_out, lens_out, refs_out, shortage);
  if (st != DW4_OK) return st;
  if (!good_block(block_size)) return DW4_ERR_UNSUPPORTED;
  if (window < 0 || sinks < 0) return DW4_ERR_INVALID_ARG;
  a.block_size = block_size;
  a.finished = finished;
  a.window = window;
  a.sinks = sinks;
  return status_of(dw4::launch_free_blocks(a, static_cast<hipStream_t>(stream)));
}

int dw4_compact_blocks(int num_layers, const int64_t* layer_key_ptrs, const int64_t* layer_value_ptrs, int64_t part_bytes,
                       int num_rows, int max_blocks, int num_blocks, const int32_t* tables, const int32_t* lens,
                       const int32_t* refs, int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int32_t* shortage,
                       int32_t* live, void* workspace, size_t workspace_bytes, void* stream) {
  dw4::PoolArgs a = {};
  int st = pool_state(a, num_rows, max_blocks, num_blocks, tables, lens, refs, tables_out, lens_out, refs_out, shortage);
  if (st == DW4_OK) st = pool_layers(a, num_layers, layer_key_ptrs, layer_value_ptrs, num_blocks, part_bytes);
  if (st != DW4_OK) return st;
  if (!live) return DW4_ERR_INVALID_ARG;
  if ((st = pool_workspace(a, workspace, workspace_bytes)) != DW4_OK) return st;
  a.live = live;
  return status_of(dw4::launch_compact_blocks(a, dw4::cu_count(), static_cast<hipStream_t>(stream)));
}

}  // extern "C"
