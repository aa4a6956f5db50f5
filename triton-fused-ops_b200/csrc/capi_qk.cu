// C-ABI layer of the query/key path: rotary tables, the rotation of query and
// key heads, and the per-head norm with the rotation and its gradients.
#include <string>

#include "capi_internal.h"
#include "common.cuh"
#include "tfo_b200.h"

namespace tfo {
namespace {

int fail(int code, const std::string& msg) { return report_error(code, msg.c_str()); }
int cuda_fail(cudaError_t e, const char* where) {
  return fail(TFO_ERR_CUDA, std::string(where) + ": " + cudaGetErrorName(e) + ": " + cudaGetErrorString(e));
}
bool is_float_dtype(int d) { return d == F16 || d == BF16 || d == F32; }

constexpr int64_t kMaxHeadDim = 1024;

void set_side(HeadSide* s, const void* x, const int64_t* strides, void* out, int64_t heads) {
  s->x = x;
  if (strides != nullptr) {
    s->stride_batch = strides[0];
    s->stride_seq = strides[1];
    s->stride_head = strides[2];
  }
  s->out = out;
  s->heads = static_cast<int>(heads);
}

// Fills everything but the weights and gradients of `a`, and checks it.
// *empty: there is no head to work on.
int set_heads(HeadArgs* a, const std::string& fn, const void* q, const int64_t* q_strides, const void* k,
              const int64_t* k_strides, const void* cos, const void* sin, int64_t table_stride, int64_t table_rows,
              const void* positions, int pos_dtype, int64_t pos_stride_batch, int64_t pos_stride_seq, void* q_out,
              void* k_out, int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads, int64_t head_dim,
              int64_t rotary_dim, int interleaved, int dtype, int table_dtype, bool* empty) {
  if (!is_float_dtype(dtype) || !is_float_dtype(table_dtype))
    return fail(TFO_ERR_DTYPE, fn + ": dtypes must be f16, bf16 or f32");
  if (pos_dtype < TFO_POS_NONE || pos_dtype > TFO_POS_I64)
    return fail(TFO_ERR_DTYPE, fn + ": positions must be int32 or int64");
  if (batch < 0 || seq < 0 || q_heads < 0 || k_heads < 0) return fail(TFO_ERR_INVALID, fn + ": negative dimension");
  if (head_dim <= 0 || head_dim > kMaxHeadDim) return fail(TFO_ERR_INVALID, fn + ": head_dim must be in 1..1024");
  if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return fail(TFO_ERR_INVALID, fn + ": rotary_dim must be even, positive and at most head_dim");
  if (batch > INT32_MAX || seq > INT32_MAX || q_heads > 65536 || k_heads > 65536)
    return fail(TFO_ERR_INVALID, fn + ": batch, seq or heads too large");
  *empty = batch == 0 || seq == 0 || q_heads + k_heads == 0;
  if (*empty) return TFO_OK;
  if (table_rows <= 0 || (pos_dtype == TFO_POS_NONE && table_rows < seq))
    return fail(TFO_ERR_INVALID, fn + ": the cos/sin table has fewer rows than the sequence has tokens");
  if (!cos || !sin || (q_heads > 0 && (!q || !q_strides || !q_out)) || (k_heads > 0 && (!k || !k_strides || !k_out)) ||
      (pos_dtype != TFO_POS_NONE && !positions))
    return fail(TFO_ERR_INVALID, fn + ": NULL pointer");
  set_side(&a->q, q, q_strides, q_out, q_heads);
  set_side(&a->k, k, k_strides, k_out, k_heads);
  a->t = HeadTables{cos,       sin,       table_stride,     table_rows,    table_dtype,
                    positions, pos_dtype, pos_stride_batch, pos_stride_seq};
  a->batch = batch;
  a->seq = seq;
  a->head_dim = static_cast<int>(head_dim);
  a->rotary_dim = static_cast<int>(rotary_dim);
  a->pairs = interleaved != 0;
  a->dtype = dtype;
  return TFO_OK;
}

}  // namespace
}  // namespace tfo

using namespace tfo;

extern "C" {

int tfo_rope_tables(const void* positions, int pos_dtype, int64_t n, const double* turns, int64_t half, double gain,
                    void* cos, void* sin, int out_dtype, void* stream) {
  const char* fn = "tfo_rope_tables";
  if (!is_float_dtype(out_dtype)) return fail(TFO_ERR_DTYPE, std::string(fn) + ": tables must be f16, bf16 or f32");
  if (pos_dtype < TFO_POS_NONE || pos_dtype > TFO_POS_I64)
    return fail(TFO_ERR_DTYPE, std::string(fn) + ": positions must be int32 or int64");
  if (n < 0 || half <= 0 || half > kMaxRopeHalf)
    return fail(TFO_ERR_INVALID, std::string(fn) + ": need n >= 0 and half in 1..256");
  if (n == 0) return TFO_OK;
  if (!turns || !cos || !sin || (pos_dtype != TFO_POS_NONE && !positions))
    return fail(TFO_ERR_INVALID, std::string(fn) + ": NULL pointer");
  for (int64_t i = 0; i < half; ++i) {
    if (!(turns[i] - turns[i] == 0.0)) return fail(TFO_ERR_INVALID, std::string(fn) + ": turns must be finite");
  }
  const RopeTablesArgs a{positions, pos_dtype, n, turns, static_cast<int>(half), gain, cos, sin, out_dtype};
  const cudaError_t e = rope_tables_launch(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TFO_OK : cuda_fail(e, fn);
}

int tfo_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* cos,
             const void* sin, int64_t table_stride, int64_t table_rows, const void* positions, int pos_dtype,
             int64_t pos_stride_batch, int64_t pos_stride_seq, void* q_out, void* k_out, int64_t batch, int64_t seq,
             int64_t q_heads, int64_t k_heads, int64_t head_dim, int64_t rotary_dim, int interleaved, int inverse,
             int dtype, int table_dtype, void* stream) {
  const char* fn = "tfo_rope";
  HeadArgs a{};
  bool empty = false;
  const int st = set_heads(&a, fn, q, q_strides, k, k_strides, cos, sin, table_stride, table_rows, positions, pos_dtype,
                           pos_stride_batch, pos_stride_seq, q_out, k_out, batch, seq, q_heads, k_heads, head_dim,
                           rotary_dim, interleaved, dtype, table_dtype, &empty);
  if (st != TFO_OK || empty) return st;
  a.inverse = inverse != 0;
  const cudaError_t e = qk_rope_launch(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TFO_OK : cuda_fail(e, fn);
}

int tfo_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                     const void* q_weight, const void* k_weight, const void* cos, const void* sin, int64_t table_stride,
                     int64_t table_rows, const void* positions, int pos_dtype, int64_t pos_stride_batch,
                     int64_t pos_stride_seq, void* q_out, void* k_out, int64_t batch, int64_t seq, int64_t q_heads,
                     int64_t k_heads, int64_t head_dim, int64_t rotary_dim, int interleaved, double eps, int dtype,
                     int q_w_dtype, int k_w_dtype, int table_dtype, void* stream) {
  const char* fn = "tfo_qk_norm_rope";
  if ((q_weight && !is_float_dtype(q_w_dtype)) || (k_weight && !is_float_dtype(k_w_dtype)))
    return fail(TFO_ERR_DTYPE, std::string(fn) + ": weights must be f16, bf16 or f32");
  HeadArgs a{};
  bool empty = false;
  const int st = set_heads(&a, fn, q, q_strides, k, k_strides, cos, sin, table_stride, table_rows, positions, pos_dtype,
                           pos_stride_batch, pos_stride_seq, q_out, k_out, batch, seq, q_heads, k_heads, head_dim,
                           rotary_dim, interleaved, dtype, table_dtype, &empty);
  if (st != TFO_OK || empty) return st;
  a.norm = true;
  a.eps = static_cast<float>(eps);
  a.q.weight = q_weight;
  a.q.w_dtype = q_w_dtype;
  a.k.weight = k_weight;
  a.k.w_dtype = k_w_dtype;
  const cudaError_t e = qk_rope_launch(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TFO_OK : cuda_fail(e, fn);
}

size_t tfo_qk_norm_rope_backward_workspace_bytes(int64_t head_dim) {
  if (head_dim <= 0 || head_dim > kMaxHeadDim) return 0;
  return qk_norm_rope_backward_workspace_bytes(static_cast<int>(head_dim));
}

int tfo_qk_norm_rope_backward(const void* dq_out, const int64_t* dq_out_strides, const void* dk_out,
                              const int64_t* dk_out_strides, const void* q, const int64_t* q_strides, const void* k,
                              const int64_t* k_strides, const void* q_weight, const void* k_weight, const void* cos,
                              const void* sin, int64_t table_stride, int64_t table_rows, const void* positions,
                              int pos_dtype, int64_t pos_stride_batch, int64_t pos_stride_seq, void* dq, void* dk,
                              void* dq_weight, void* dk_weight, int64_t batch, int64_t seq, int64_t q_heads,
                              int64_t k_heads, int64_t head_dim, int64_t rotary_dim, int interleaved, double eps,
                              int dtype, int q_w_dtype, int k_w_dtype, int table_dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* fn = "tfo_qk_norm_rope_backward";
  if ((q_weight && !is_float_dtype(q_w_dtype)) || (k_weight && !is_float_dtype(k_w_dtype)))
    return fail(TFO_ERR_DTYPE, std::string(fn) + ": weights must be f16, bf16 or f32");
  if ((dq_weight && !q_weight) || (dk_weight && !k_weight))
    return fail(TFO_ERR_INVALID, std::string(fn) + ": a weight's gradient needs the weight");
  HeadArgs a{};
  bool empty = false;
  const int s = set_heads(&a, fn, q, q_strides, k, k_strides, cos, sin, table_stride, table_rows, positions, pos_dtype,
                          pos_stride_batch, pos_stride_seq, dq, dk, batch, seq, q_heads, k_heads, head_dim, rotary_dim,
                          interleaved, dtype, table_dtype, &empty);
  if (s != TFO_OK) return s;
  auto st = static_cast<cudaStream_t>(stream);
  auto zero = [&](void* p, int w_dtype) {
    if (p == nullptr) return cudaSuccess;
    note_launch();
    return cudaMemsetAsync(p, 0, static_cast<size_t>(head_dim) * (w_dtype == F32 ? 4 : 2), st);
  };
  // a side without heads adds nothing to its weight's gradient
  cudaError_t e = cudaSuccess;
  if (empty || q_heads == 0) e = zero(dq_weight, q_w_dtype);
  if (e == cudaSuccess && (empty || k_heads == 0)) e = zero(dk_weight, k_w_dtype);
  if (e != cudaSuccess) return cuda_fail(e, fn);
  if (empty) return TFO_OK;
  if ((q_heads > 0 && (!dq_out || !dq_out_strides)) || (k_heads > 0 && (!dk_out || !dk_out_strides)))
    return fail(TFO_ERR_INVALID, std::string(fn) + ": NULL pointer");
  if ((dq_weight || dk_weight) && (!workspace || workspace_bytes < tfo_qk_norm_rope_backward_workspace_bytes(head_dim) ||
                                   reinterpret_cast<uintptr_t>(workspace) % sizeof(float) != 0))
    return fail(TFO_ERR_INVALID, std::string(fn) + ": workspace too small or not aligned");
  a.norm = true;
  a.eps = static_cast<float>(eps);
  auto grads = [](HeadSide* side, const void* w, int w_dtype, const void* dy, const int64_t* strides, void* dw) {
    side->weight = w;
    side->w_dtype = w_dtype;
    if (side->heads == 0) return;
    side->dy = dy;
    side->dy_stride_batch = strides[0];
    side->dy_stride_seq = strides[1];
    side->dy_stride_head = strides[2];
    side->dweight = dw;
  };
  grads(&a.q, q_weight, q_w_dtype, dq_out, dq_out_strides, dq_weight);
  grads(&a.k, k_weight, k_w_dtype, dk_out, dk_out_strides, dk_weight);
  e = qk_norm_rope_backward_launch(a, workspace, st);
  return e == cudaSuccess ? TFO_OK : cuda_fail(e, fn);
}

}  // extern "C"
