// C-ABI layer of the residual stream: dropout, and the sum of a block's branch
// with the norms before and after it.
#include <cmath>
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

int set_dropout(DropoutArgs* d, const std::string& fn, const tfo_dropout_params& p) {
  if (!(p.p >= 0.0 && p.p <= 1.0)) return fail(TFO_ERR_INVALID, fn + ": the dropout probability must be in 0..1");
  if (reinterpret_cast<uintptr_t>(p.seed) % sizeof(int64_t) != 0)
    return fail(TFO_ERR_INVALID, fn + ": the seed is not aligned");
  const double border = std::nearbyint(p.p * 4294967296.0);
  d->seed_ptr = p.seed;
  d->seed = p.seed_value;
  d->offset = p.offset;
  d->none = border == 0.0;
  d->all = border == 4294967296.0;
  d->threshold = d->all ? 0xffffffffu : static_cast<uint32_t>(border);
  d->scale = d->all ? 0.f : static_cast<float>(1.0 / (1.0 - p.p));
  return TFO_OK;
}

bool stream_types(int x_dtype, int res_dtype) {
  return is_float_dtype(x_dtype) && (res_dtype == x_dtype || res_dtype == F32);
}

constexpr int64_t kMaxHidden = 1 << 24;

// Sizes, types, parameters and dropout of `a`.
int set_rows(ResidualArgs* a, const std::string& fn, const void* x, int64_t x_stride, const void* res, int64_t res_stride,
             const tfo_row_param* params, int64_t rows, int64_t rows_per_seq, int64_t hidden,
             bool branch_norm, const tfo_dropout_params* dropout, int x_dtype, int res_dtype) {
  if (!stream_types(x_dtype, res_dtype))
    return fail(TFO_ERR_DTYPE, fn + ": x must be f16, bf16 or f32, and the residual stream of its type or f32");
  if (hidden <= 0 || hidden > kMaxHidden) return fail(TFO_ERR_INVALID, fn + ": hidden must be in 1..2^24");
  if (rows < 0 || rows > INT32_MAX) return fail(TFO_ERR_INVALID, fn + ": rows must be in 0..2^31 - 1");
  if (rows > 0 && (rows_per_seq <= 0 || rows % rows_per_seq != 0))
    return fail(TFO_ERR_INVALID, fn + ": rows_per_seq must divide rows");
  if (x_stride < 0 || res_stride < 0) return fail(TFO_ERR_INVALID, fn + ": negative row stride");
  if (params == nullptr || (rows > 0 && (x == nullptr || res == nullptr)))
    return fail(TFO_ERR_INVALID, fn + ": NULL pointer");
  RowParam* to[4] = {&a->branch_weight, &a->gate, &a->weight, &a->shift};
  for (int i = 0; i < 4; ++i) {
    const tfo_row_param& p = params[i];
    if (p.data != nullptr && !is_float_dtype(p.dtype)) return fail(TFO_ERR_DTYPE, fn + ": parameters must be f16, bf16 or f32");
    *to[i] = RowParam{p.data, p.dtype, p.data != nullptr ? p.seq_stride : 0, p.data != nullptr ? p.grad : nullptr};
  }
  if (!branch_norm && a->branch_weight.p != nullptr)
    return fail(TFO_ERR_INVALID, fn + ": a branch weight needs branch_norm");
  a->branch_norm = branch_norm;
  a->x = x;
  a->x_stride = x_stride;
  a->res = res;
  a->res_stride = res_stride;
  a->rows = rows;
  a->rows_per_seq = rows_per_seq;
  a->hidden = static_cast<int>(hidden);
  a->x_dtype = x_dtype;
  a->res_dtype = res_dtype;
  if (dropout != nullptr) {
    if (const int st = set_dropout(&a->drop, fn, *dropout); st != TFO_OK) return st;
    a->dropped = !a->drop.none;
  }
  return TFO_OK;
}

void set_grads(ResidualArgs* a, const void* dh, int64_t dh_stride, const void* dy, int64_t dy_stride, const void* dx,
               const void* dres) {
  a->dh = dh;
  a->dh_stride = dh_stride;
  a->dy = dy;
  a->dy_stride = dy_stride;
  a->dx = const_cast<void*>(dx);
  a->dres = const_cast<void*>(dres);
}

}  // namespace
}  // namespace tfo

using namespace tfo;

extern "C" {

int tfo_dropout(const void* x, const void* residual, void* out, int64_t n, const tfo_dropout_params* dropout, int x_dtype,
                int out_dtype, void* stream) {
  const char* fn = "tfo_dropout";
  if (!is_float_dtype(x_dtype) || !is_float_dtype(out_dtype) ||
      (x_dtype != out_dtype && (residual != nullptr ? out_dtype : x_dtype) != F32))
    return fail(TFO_ERR_DTYPE, std::string(fn) + ": x must be f16, bf16 or f32, out of its type, or F32 with a residual, or "
                                                 "16 bits for an F32 x without one");
  if (n < 0) return fail(TFO_ERR_INVALID, std::string(fn) + ": negative size");
  if (dropout == nullptr) return fail(TFO_ERR_INVALID, std::string(fn) + ": NULL pointer");
  DropoutArgs d{};
  if (const int st = set_dropout(&d, fn, *dropout); st != TFO_OK) return st;
  if (n == 0) return TFO_OK;
  if (!x || !out) return fail(TFO_ERR_INVALID, std::string(fn) + ": NULL pointer");
  const cudaError_t e = dropout_launch(x, x_dtype, residual, out, out_dtype, n, d, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TFO_OK : cuda_fail(e, fn);
}

int tfo_residual_rmsnorm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                         const tfo_row_param* params, void* h, void* y, float* rstd, int64_t rows, int64_t rows_per_seq,
                         int64_t hidden, int branch_norm, double scale, double eps, const tfo_dropout_params* dropout,
                         int x_dtype, int residual_dtype, void* stream) {
  const char* fn = "tfo_residual_rmsnorm";
  ResidualArgs a{};
  const int st = set_rows(&a, fn, x, x_stride, residual, residual_stride, params, rows, rows_per_seq, hidden,
                          branch_norm != 0, dropout, x_dtype, residual_dtype);
  if (st != TFO_OK || rows == 0) return st;
  if (!h) return fail(TFO_ERR_INVALID, std::string(fn) + ": NULL pointer");
  if (reinterpret_cast<uintptr_t>(rstd) % (2 * sizeof(float)) != 0)
    return fail(TFO_ERR_INVALID, std::string(fn) + ": rstd is not aligned");
  a.h = h;
  a.y = y;
  a.rstd = rstd;
  if (y == nullptr) a.weight = a.shift = RowParam{};
  a.scale = static_cast<float>(scale);
  a.eps = static_cast<float>(eps);
  const cudaError_t e = residual_norm_launch(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TFO_OK : cuda_fail(e, fn);
}

size_t tfo_residual_rmsnorm_backward_workspace_bytes(const void* dh, int64_t dh_stride, const void* dy, int64_t dy_stride,
                                                     const void* x, int64_t x_stride, const void* residual,
                                                     int64_t residual_stride, const tfo_row_param* params, const void* dx,
                                                     const void* dresidual, int64_t rows, int64_t rows_per_seq,
                                                     int64_t hidden, int x_dtype, int residual_dtype) {
  ResidualArgs a{};
  if (set_rows(&a, "tfo_residual_rmsnorm_backward", x, x_stride, residual, residual_stride, params, rows, rows_per_seq,
               hidden, true, nullptr, x_dtype, residual_dtype) != TFO_OK ||
      rows == 0)
    return 0;
  set_grads(&a, dh, dh_stride, dy, dy_stride, dx, dresidual);
  return residual_norm_backward_workspace_bytes(a);
}

int tfo_residual_rmsnorm_backward(const void* dh, int64_t dh_stride, const void* dy, int64_t dy_stride, const void* x,
                                  int64_t x_stride, const void* residual, int64_t residual_stride,
                                  const tfo_row_param* params, const float* rstd, void* dx, void* dresidual, int64_t rows,
                                  int64_t rows_per_seq, int64_t hidden, int branch_norm, double scale,
                                  const tfo_dropout_params* dropout, int x_dtype, int residual_dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* fn = "tfo_residual_rmsnorm_backward";
  ResidualArgs a{};
  const int st = set_rows(&a, fn, x, x_stride, residual, residual_stride, params, rows, rows_per_seq, hidden,
                          branch_norm != 0, dropout, x_dtype, residual_dtype);
  if (st != TFO_OK || rows == 0) return st;
  if (!rstd) return fail(TFO_ERR_INVALID, std::string(fn) + ": NULL pointer");
  if (reinterpret_cast<uintptr_t>(rstd) % (2 * sizeof(float)) != 0)
    return fail(TFO_ERR_INVALID, std::string(fn) + ": rstd is not aligned");
  a.rstd = const_cast<float*>(rstd);
  a.scale = static_cast<float>(scale);
  set_grads(&a, dh, dh_stride, dy, dy_stride, dx, dresidual);
  if (dh_stride < 0 || dy_stride < 0) return fail(TFO_ERR_INVALID, std::string(fn) + ": negative row stride");
  const size_t need = residual_norm_backward_workspace_bytes(a);
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return fail(TFO_ERR_INVALID, std::string(fn) + ": workspace too small or not aligned");
  const cudaError_t e = residual_norm_backward_launch(a, workspace, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TFO_OK : cuda_fail(e, fn);
}

}  // extern "C"
