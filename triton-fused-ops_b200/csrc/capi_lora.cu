// C-ABI layer of the low-rank adapters.
#include <string>

#include "capi_internal.h"
#include "common.cuh"
#include "tfo_b200.h"

namespace tfo {
namespace {
int fail(int code, const std::string& msg) { return report_error(code, msg.c_str()); }
bool is_float_dtype(int d) { return d == F16 || d == BF16 || d == F32; }
constexpr int64_t kMaxRank = 256, kMaxAdapters = 16384;
}  // namespace
}  // namespace tfo

using namespace tfo;

extern "C" {

size_t tfo_lora_workspace_bytes(int64_t tokens, int64_t adapters) {
  if (tokens <= 0 || adapters <= 0) return 0;
  return lora_workspace_bytes(tokens, adapters);
}

int tfo_lora(const void* x, int64_t x_stride, const void* a, const void* b, const void* ids, int ids_dtype,
             const float* scaling, const void* base, int64_t base_stride, void* out, int64_t out_stride, int64_t tokens,
             int64_t adapters, int64_t rank, int64_t k, int64_t n, int dtype, void* workspace, size_t workspace_bytes,
             void* stream) {
  const char* fn = "tfo_lora";
  if (!is_float_dtype(dtype)) return fail(TFO_ERR_DTYPE, std::string(fn) + ": dtype must be f16, bf16 or f32");
  if (ids_dtype != TFO_POS_I32 && ids_dtype != TFO_POS_I64)
    return fail(TFO_ERR_DTYPE, std::string(fn) + ": ids must be int32 or int64");
  if (tokens < 0 || n < 0 || tokens > INT32_MAX || n > INT32_MAX || k > INT32_MAX)
    return fail(TFO_ERR_INVALID, std::string(fn) + ": tokens, n and k must be non-negative and fit in int32");
  if (adapters <= 0 || adapters > kMaxAdapters)
    return fail(TFO_ERR_INVALID, std::string(fn) + ": adapters must be in 1..16384");
  if (rank <= 0 || rank > kMaxRank || k <= 0)
    return fail(TFO_ERR_INVALID, std::string(fn) + ": rank must be in 1..256 and k positive");
  if (tokens == 0 || n == 0) return TFO_OK;
  if (!x || !a || !b || !ids || !out) return fail(TFO_ERR_INVALID, std::string(fn) + ": NULL pointer");
  if (tokens > 1 && out_stride < n) return fail(TFO_ERR_INVALID, std::string(fn) + ": rows of out overlap");
  if (base == out && tokens > 1 && base_stride != out_stride)
    return fail(TFO_ERR_INVALID, std::string(fn) + ": base and out share memory but not their rows");
  const size_t need = lora_workspace_bytes(tokens, adapters);
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return fail(TFO_ERR_INVALID, std::string(fn) + ": workspace too small or not 16-byte aligned");
  const LoraArgs args{x,   x_stride,   a,      b,        ids,  ids_dtype, scaling, base, base_stride,
                      out, out_stride, tokens, adapters, rank, k,         n,       dtype};
  const cudaError_t e = lora_launch(args, workspace, static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) return TFO_OK;
  return fail(TFO_ERR_CUDA, std::string(fn) + ": " + cudaGetErrorName(e) + ": " + cudaGetErrorString(e));
}

}  // extern "C"
