// C ABI of the low-rank adapters, dropout, rotary positions and slot maps (declared in
// include/drofell_w4a16.h): validation and dispatch.  Every entry point returns a
// status code; nothing throws across the ABI.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "drofell_w4a16.h"
#include "w4a16_adapters.h"
#include "w4a16_blocks.h"
#include "w4a16_internal.h"
#include "w4a16_rotary.h"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int status_of(hipError_t e) { return e == hipSuccess ? DW4_OK : DW4_ERR_LAUNCH; }

int check_rows(int rows, int adapters) {
  if (rows < 0 || adapters < 0) return DW4_ERR_INVALID_ARG;
  if (rows > dw4::kAdapterMaxRows || adapters > dw4::kAdapterMaxCount) return DW4_ERR_UNSUPPORTED;
  return DW4_OK;
}

int check_shape(int rows, int adapters, int k, int n, int rank) {
  const int st = check_rows(rows, adapters);
  if (st != DW4_OK) return st;
  if (k <= 0 || n <= 0 || rank <= 0) return DW4_ERR_INVALID_ARG;
  if (k % 8 != 0 || n % 8 != 0 || rank % 8 != 0 || rank > dw4::kAdapterMaxRank) return DW4_ERR_UNSUPPORTED;
  if (k > 1 << 20 || n > 1 << 20) return DW4_ERR_UNSUPPORTED;
  return DW4_OK;
}

// A launch counts its threads, 256 a workgroup, in 32 bits.
int check_grad(int rows, int adapters, int k, int n, int rank) {
  const dw4::AdapterLayout l = dw4::adapter_layout(rows, adapters);
  return dw4::grad_workgroups(l, k, n, rank, adapters) < (int64_t)1 << 24 ? DW4_OK : DW4_ERR_UNSUPPORTED;
}

// A matrix [rows][width] of 16-bit values that kernels read or write in 16-byte units.
int check_matrix(const void* p, int64_t stride, int rows, int width) {
  if (p == nullptr) return DW4_ERR_INVALID_ARG;
  if (rows > 1 && stride < width) return DW4_ERR_INVALID_ARG;
  if (!aligned16(p) || (rows > 1 && stride % 8 != 0)) return DW4_ERR_MISALIGNED;
  return DW4_OK;
}

int check_drop(int drop, const int64_t* seed) {
  if (drop < 0 || drop > 65536) return DW4_ERR_INVALID_ARG;
  if (drop > 0 && seed == nullptr) return DW4_ERR_INVALID_ARG;
  return DW4_OK;
}
float keep_scale(int drop) { return drop < 65536 ? 65536.f / (float)(65536 - drop) : 0.f; }

#define DW4_TRY(expr)              \
  do {                             \
    const int st_ = (expr);        \
    if (st_ != DW4_OK) return st_; \
  } while (0)

dw4::AdapterArgs adapter_args(int dtype, int rows, int k, int n, int rank, int adapters, const uint16_t* x, int64_t ldx,
                              const uint16_t* a, const uint16_t* b, const float* scaling, const int32_t* plan, int drop,
                              const int64_t* seed, void* h, void* ws) {
  dw4::AdapterArgs p = {};
  p.l = dw4::adapter_layout(rows, adapters);
  p.bf16 = dtype == DW4_BF16;
  p.k = k;
  p.n = n;
  p.r = rank;
  p.adapters = adapters;
  p.plan = plan;
  p.x = x;
  p.ldx = ldx;
  p.a = a;
  p.b = b;
  p.scaling = scaling;
  p.drop = drop;
  p.seed = seed;
  p.keep_scale = keep_scale(drop);
  p.h = h;
  p.ws = static_cast<unsigned char*>(ws);
  return p;
}

bool good_dtype(int dtype) { return dtype == DW4_F16 || dtype == DW4_BF16; }

int check_rotary(int dtype, int rows, int heads, int kv_heads, int head_size, int rotary_size, int form, float magnitude) {
  if (!good_dtype(dtype)) return DW4_ERR_UNSUPPORTED;
  if (form & ~(DW4_ROTARY_INTERLEAVED | DW4_ROTARY_POSITIONS64)) return DW4_ERR_INVALID_ARG;
  if (rows < 0 || heads < 0 || kv_heads < 0 || head_size <= 0 || rotary_size <= 0 || rotary_size > head_size ||
      !std::isfinite(magnitude))
    return DW4_ERR_INVALID_ARG;
  if (head_size % 8 != 0 || head_size > 512 || rotary_size % 2 != 0) return DW4_ERR_UNSUPPORTED;
  // a launch counts its threads in 32 bits, up to one a dim of every row
  if (rows > 1 << 22 || heads > 1 << 14 || kv_heads > 1 << 14 || (int64_t)rows * (heads + kv_heads) > (int64_t)1 << 27)
    return DW4_ERR_UNSUPPORTED;
  return DW4_OK;
}

}  // namespace

extern "C" {

int dw4_adapter_plan_size(int num_rows, int num_adapters, size_t* plan_bytes) {
  DW4_TRY(check_rows(num_rows, num_adapters));
  if (plan_bytes == nullptr) return DW4_ERR_INVALID_ARG;
  *plan_bytes = num_rows ? sizeof(int32_t) * (size_t)dw4::adapter_layout(num_rows, num_adapters).ints : 0;
  return DW4_OK;
}

int dw4_adapter_plan(int num_rows, int num_adapters, const int32_t* adapters, int32_t* plan, size_t plan_bytes, void* stream) {
  DW4_TRY(check_rows(num_rows, num_adapters));
  if (num_rows == 0) return DW4_OK;
  if (adapters == nullptr || plan == nullptr) return DW4_ERR_INVALID_ARG;
  const dw4::AdapterLayout l = dw4::adapter_layout(num_rows, num_adapters);
  if (plan_bytes < sizeof(int32_t) * (size_t)l.ints) return DW4_ERR_WORKSPACE;
  if (!aligned16(plan)) return DW4_ERR_MISALIGNED;
  return status_of(dw4::launch_adapter_plan(l, num_rows, num_adapters, adapters, plan, static_cast<hipStream_t>(stream)));
}

int dw4_adapters_workspace_size(int num_rows, int num_adapters, int k, int n, int rank, int backward, size_t* workspace_bytes,
                                size_t* h_bytes) {
  DW4_TRY(check_shape(num_rows, num_adapters, k, n, rank));
  if (workspace_bytes == nullptr) return DW4_ERR_INVALID_ARG;
  if (backward) DW4_TRY(check_grad(num_rows, num_adapters, k, n, rank));
  const dw4::AdapterLayout l = dw4::adapter_layout(num_rows, num_adapters);
  if (h_bytes != nullptr) *h_bytes = num_rows ? dw4::col_pack_bytes(l, rank) : 0;
  *workspace_bytes = 0;
  if (num_rows > 0)
    *workspace_bytes = backward ? dw4::backward_ws(l, k, n, rank, num_adapters, dw4::cu_count()).bytes
                                : dw4::forward_ws(l, k, rank, dw4::cu_count()).bytes;
  return DW4_OK;
}

int dw4_adapters(int dtype, int num_rows, int num_adapters, int k, int n, int rank, const uint16_t* x, int64_t ldx,
                 const uint16_t* base, int64_t ldb, uint16_t* out, int64_t ldo, const uint16_t* a, const uint16_t* b,
                 const float* scaling, const int32_t* plan, int drop, const int64_t* seed, void* h, void* workspace,
                 size_t workspace_bytes, void* stream) {
  if (!good_dtype(dtype)) return DW4_ERR_UNSUPPORTED;
  DW4_TRY(check_shape(num_rows, num_adapters, k, n, rank));
  DW4_TRY(check_drop(drop, seed));
  if (num_rows == 0) return DW4_OK;
  if (plan == nullptr || (num_adapters > 0 && (a == nullptr || b == nullptr || scaling == nullptr))) return DW4_ERR_INVALID_ARG;
  DW4_TRY(check_matrix(x, ldx, num_rows, k));
  DW4_TRY(check_matrix(base, ldb, num_rows, n));
  DW4_TRY(check_matrix(out, ldo, num_rows, n));
  if (out == base && ldo != ldb && num_rows > 1) return DW4_ERR_INVALID_ARG;
  if (!aligned16(a) || !aligned16(b) || !aligned16(h) || !aligned16(plan)) return DW4_ERR_MISALIGNED;
  dw4::AdapterArgs p = adapter_args(dtype, num_rows, k, n, rank, num_adapters, x, ldx, a, b, scaling, plan, drop, seed, h, workspace);
  p.base = base;
  p.ldb = ldb;
  p.out = out;
  p.ldo = ldo;
  const dw4::ForwardWs w = dw4::forward_ws(p.l, k, rank, dw4::cu_count());
  if (workspace == nullptr || workspace_bytes < w.bytes) return DW4_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DW4_ERR_MISALIGNED;
  return status_of(dw4::launch_adapters(p, w, static_cast<hipStream_t>(stream)));
}

int dw4_adapters_backward(int dtype, int num_rows, int num_adapters, int k, int n, int rank, const uint16_t* x, int64_t ldx,
                          const uint16_t* dout, int64_t ldd, const uint16_t* a, const uint16_t* b, const float* scaling,
                          const int32_t* plan, int drop, const int64_t* seed, const void* h, uint16_t* dx, int64_t lddx,
                          uint16_t* da, uint16_t* db, void* workspace, size_t workspace_bytes, void* stream) {
  if (!good_dtype(dtype)) return DW4_ERR_UNSUPPORTED;
  DW4_TRY(check_shape(num_rows, num_adapters, k, n, rank));
  DW4_TRY(check_drop(drop, seed));
  if (num_rows == 0) return DW4_ERR_INVALID_ARG;  // nothing to reduce: the caller's zeros
  DW4_TRY(check_grad(num_rows, num_adapters, k, n, rank));
  if (plan == nullptr || h == nullptr || (num_adapters > 0 && (a == nullptr || b == nullptr || scaling == nullptr)))
    return DW4_ERR_INVALID_ARG;
  DW4_TRY(check_matrix(x, ldx, num_rows, k));
  DW4_TRY(check_matrix(dout, ldd, num_rows, n));
  if (dx != nullptr) DW4_TRY(check_matrix(dx, lddx, num_rows, k));
  if (!aligned16(a) || !aligned16(b) || !aligned16(h) || !aligned16(plan) || !aligned16(da) || !aligned16(db))
    return DW4_ERR_MISALIGNED;
  if (dx == nullptr && da == nullptr && db == nullptr) return DW4_OK;
  dw4::AdapterArgs p = adapter_args(dtype, num_rows, k, n, rank, num_adapters, x, ldx, a, b, scaling, plan, drop, seed,
                                    const_cast<void*>(h), workspace);
  p.g = dout;
  p.ldg = ldd;
  p.dx = dx;
  p.lddx = lddx;
  p.da = num_adapters ? da : nullptr;
  p.db = num_adapters ? db : nullptr;
  const dw4::BackwardWs w = dw4::backward_ws(p.l, k, n, rank, num_adapters, dw4::cu_count());
  if (workspace == nullptr || workspace_bytes < w.bytes) return DW4_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DW4_ERR_MISALIGNED;
  return status_of(dw4::launch_adapters_grad(p, w, static_cast<hipStream_t>(stream)));
}

int dw4_dropout(int dtype, int num_rows, int cols, const uint16_t* x, int64_t ldx, uint16_t* y, int64_t ldy, int drop,
                const int64_t* seed, void* stream) {
  if (!good_dtype(dtype)) return DW4_ERR_UNSUPPORTED;
  if (num_rows < 0 || cols < 0 || seed == nullptr) return DW4_ERR_INVALID_ARG;
  if (cols > 1 << 30) return DW4_ERR_UNSUPPORTED;
  DW4_TRY(check_drop(drop, seed));
  if (num_rows == 0 || cols == 0) return DW4_OK;
  if (x == nullptr || y == nullptr || (num_rows > 1 && (ldx < cols || ldy < cols))) return DW4_ERR_INVALID_ARG;
  return status_of(dw4::launch_dropout(dtype == DW4_BF16, num_rows, cols, x, ldx, y, ldy, drop, keep_scale(drop), seed,
                                       static_cast<hipStream_t>(stream)));
}

int dw4_rotary(int dtype, int num_rows, int num_heads, int num_kv_heads, int head_size, int rotary_size, int form,
               int inverse, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride, uint16_t* q_out,
               int64_t qo_stride, uint16_t* k_out, int64_t ko_stride, const void* positions, const int64_t* turns,
               float magnitude, void* stream) {
  DW4_TRY(check_rotary(dtype, num_rows, num_heads, num_kv_heads, head_size, rotary_size, form, magnitude));
  if (num_rows == 0 || num_heads + num_kv_heads == 0) return DW4_OK;
  if (positions == nullptr || turns == nullptr) return DW4_ERR_INVALID_ARG;
  if (num_heads > 0) {
    DW4_TRY(check_matrix(q, q_stride, num_rows, num_heads * head_size));
    DW4_TRY(check_matrix(q_out, qo_stride, num_rows, num_heads * head_size));
  }
  if (num_kv_heads > 0) {
    DW4_TRY(check_matrix(k, k_stride, num_rows, num_kv_heads * head_size));
    DW4_TRY(check_matrix(k_out, ko_stride, num_rows, num_kv_heads * head_size));
  }
  dw4::RotaryArgs a = {};
  a.bf16 = dtype == DW4_BF16;
  a.interleaved = (form & DW4_ROTARY_INTERLEAVED) != 0;
  a.positions64 = (form & DW4_ROTARY_POSITIONS64) != 0;
  a.inverse = inverse != 0;
  a.rows = num_rows;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.head_size = head_size;
  a.rotary_size = rotary_size;
  a.q = q;
  a.q_stride = q_stride;
  a.k = k;
  a.k_stride = k_stride;
  a.q_out = q_out;
  a.qo_stride = qo_stride;
  a.k_out = k_out;
  a.ko_stride = ko_stride;
  a.positions = positions;
  a.turns = turns;
  a.magnitude = magnitude;
  return status_of(dw4::launch_rotary(a, static_cast<hipStream_t>(stream)));
}

int dw4_rotary_and_cache(int dtype, int num_rows, int num_heads, int num_kv_heads, int head_size, int rotary_size,
                         int form, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
                         const uint16_t* v, int64_t v_stride, uint16_t* q_out, int64_t qo_stride, const void* positions,
                         const int64_t* turns, float magnitude, const int64_t* slots, int num_blocks, int block_size,
                         const int64_t* key_block_ptrs, const int64_t* value_block_ptrs, int kv_head_stride, void* stream) {
  DW4_TRY(check_rotary(dtype, num_rows, num_heads, num_kv_heads, head_size, rotary_size, form, magnitude));
  if (block_size != 16 && block_size != 32) return DW4_ERR_UNSUPPORTED;
  if (num_blocks < 0 || num_kv_heads == 0 || num_heads == 0 || kv_head_stride < head_size * block_size) return DW4_ERR_INVALID_ARG;
  if (num_rows == 0) return DW4_OK;
  if (positions == nullptr || turns == nullptr || slots == nullptr) return DW4_ERR_INVALID_ARG;
  if (num_blocks > 0 && (key_block_ptrs == nullptr || value_block_ptrs == nullptr)) return DW4_ERR_INVALID_ARG;
  DW4_TRY(check_matrix(q, q_stride, num_rows, num_heads * head_size));
  DW4_TRY(check_matrix(q_out, qo_stride, num_rows, num_heads * head_size));
  DW4_TRY(check_matrix(k, k_stride, num_rows, num_kv_heads * head_size));
  DW4_TRY(check_matrix(v, v_stride, num_rows, num_kv_heads * head_size));
  if (kv_head_stride % 8 != 0) return DW4_ERR_MISALIGNED;
  dw4::RotaryArgs a = {};
  a.bf16 = dtype == DW4_BF16;
  a.interleaved = (form & DW4_ROTARY_INTERLEAVED) != 0;
  a.positions64 = (form & DW4_ROTARY_POSITIONS64) != 0;
  a.rows = num_rows;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.head_size = head_size;
  a.rotary_size = rotary_size;
  a.q = q;
  a.q_stride = q_stride;
  a.k = k;
  a.k_stride = k_stride;
  a.q_out = q_out;
  a.qo_stride = qo_stride;
  a.positions = positions;
  a.turns = turns;
  a.magnitude = magnitude;
  a.v = v;
  a.v_stride = v_stride;
  a.slots = slots;
  a.kptr = key_block_ptrs;
  a.vptr = value_block_ptrs;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.kv_head_stride = kv_head_stride;
  return status_of(dw4::launch_rotary_cache(a, static_cast<hipStream_t>(stream)));
}

int dw4_token_slots(int num_rows, int max_blocks, int num_blocks, int block_size, const int32_t* tables, const int32_t* lens,
                    const int32_t* new_tokens, int num_tokens, int32_t* query_starts, int32_t* positions, int64_t* slots,
                    int32_t* rows, int32_t* excess, void* stream) {
  if (num_rows < 0 || max_blocks < 0 || num_blocks < 0 || num_tokens < 0) return DW4_ERR_INVALID_ARG;
  if ((block_size != 16 && block_size != 32) || num_rows > dw4::kSlotMaxRows) return DW4_ERR_UNSUPPORTED;
  if (query_starts == nullptr || excess == nullptr) return DW4_ERR_INVALID_ARG;
  if (num_rows > 0 && (lens == nullptr || new_tokens == nullptr || (max_blocks > 0 && tables == nullptr))) return DW4_ERR_INVALID_ARG;
  if (num_tokens > 0 && (positions == nullptr || slots == nullptr || rows == nullptr)) return DW4_ERR_INVALID_ARG;
  if (num_tokens > 1 << 28) return DW4_ERR_UNSUPPORTED;
  const dw4::SlotArgs a = {num_rows, max_blocks, num_blocks, block_size, num_tokens, tables, lens, new_tokens,
                           query_starts, positions, slots, rows, excess};
  return status_of(dw4::launch_token_slots(a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
