// PyTorch extension over the C ABI for the calls whose kernels take a few
// microseconds (decode-size activations), where the host work of the Python
// wrappers (argument checks, two or three allocations, several ctypes calls)
// took longer than the kernels. One Python -> C++ call here checks the common
// case, allocates through torch's caching allocator, reuses a scratch buffer
// per (device, stream) and calls the library; anything outside the common
// case returns None and the Python wrapper takes its full path (which raises
// the package's exceptions). The arithmetic is the library's: these functions
// produce exactly what the Python path produces.
//
// Mirrors: triton_ops/kernels/fp8_quantize.py:128-173 (quantize_fp8, dynamic
// scale) and triton_ops/kernels/fp8_gemm.py:272-310 (FP8Linear.forward).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <array>
#include <mutex>
#include <stdexcept>
#include <string>
#include <vector>

#include "tfo_b200.h"

namespace py = pybind11;

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return TFO_DTYPE_F16;
    case at::kBFloat16: return TFO_DTYPE_BF16;
    case at::kFloat: return TFO_DTYPE_F32;
    case at::kByte: return TFO_DTYPE_U8;
    case at::kFloat8_e4m3fn: return TFO_DTYPE_E4M3;
    default: return -1;
  }
}

bool is_float(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat; }

// Non-zero status -> Python RuntimeError "tfo status <n>: <message>"; the
// wrapper maps it to the package's exception for that status.
void check(int status, const char* what) {
  if (status != TFO_OK) {
    const char* msg = tfo_last_error();
    throw std::runtime_error(std::string("tfo status ") + std::to_string(status) + ": " + what + ": " +
                             (msg ? msg : ""));
  }
}

// One grow-only scratch buffer per (device, stream), at most kMaxEntries kept
// (least recently used dropped), as the Python wrappers do; a fresh tensor
// while the stream is being captured into a CUDA graph.
constexpr size_t kMaxEntries = 8;
struct WsEntry {
  int device;
  cudaStream_t stream;
  at::Tensor buf;
};
std::mutex g_ws_mu;
std::vector<WsEntry> g_ws;  // most recently used last

// `st` is torch's current stream on `dev` (the device guard is set).
at::Tensor workspace(size_t bytes, const at::Device& dev, cudaStream_t st) {
  bytes = std::max<size_t>(bytes, 16);
  const auto opts = at::TensorOptions().dtype(at::kByte).device(dev);
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None)
    return at::empty({static_cast<int64_t>(bytes)}, opts);
  std::lock_guard<std::mutex> lock(g_ws_mu);
  for (size_t i = 0; i < g_ws.size(); ++i) {
    if (g_ws[i].device == dev.index() && g_ws[i].stream == st) {
      WsEntry e = g_ws[i];
      g_ws.erase(g_ws.begin() + static_cast<long>(i));
      if (static_cast<size_t>(e.buf.numel()) < bytes)
        e.buf = at::empty({static_cast<int64_t>(std::max(bytes, 2 * static_cast<size_t>(e.buf.numel())))}, opts);
      g_ws.push_back(e);
      return e.buf;
    }
  }
  g_ws.push_back(WsEntry{dev.index(), st, at::empty({static_cast<int64_t>(bytes)}, opts)});
  if (g_ws.size() > kMaxEntries) g_ws.erase(g_ws.begin());
  return g_ws.back().buf;
}

void clear_workspaces() {
  std::lock_guard<std::mutex> lock(g_ws_mu);
  g_ws.clear();
}

bool common_ok(const at::Tensor& x) { return x.is_cuda() && x.is_contiguous() && is_float(x.scalar_type()); }

// quantize_fp8(x) with a dynamic scale: (codes shaped like x, 0-dim fp32 scale),
// or None outside the common case (CUDA, contiguous, f16/bf16/f32 input,
// uint8 or float8_e4m3fn codes).
py::object quantize_dynamic(const at::Tensor& x, int64_t out_code) {
  if (!common_ok(x) || (out_code != TFO_DTYPE_U8 && out_code != TFO_DTYPE_E4M3)) return py::none();
  const c10::cuda::CUDAGuard guard(x.device());
  const auto st = at::cuda::getCurrentCUDAStream(x.device().index()).stream();
  const auto code_type = out_code == TFO_DTYPE_U8 ? at::kByte : at::kFloat8_e4m3fn;
  at::Tensor out = at::empty(x.sizes(), x.options().dtype(code_type));
  at::Tensor scale = at::empty({}, x.options().dtype(at::kFloat));
  const int64_t n = x.numel();
  at::Tensor ws = workspace(tfo_fp8_scale_workspace_bytes(n), x.device(), st);
  check(tfo_fp8_quantize(x.data_ptr(), n, dtype_code(x.scalar_type()), nullptr, scale.data_ptr<float>(),
                         out.data_ptr(), static_cast<int>(out_code), ws.data_ptr(), static_cast<size_t>(ws.numel()),
                         st),
        "tfo_fp8_quantize");
  return py::make_tuple(out, scale);
}

// FP8Linear.forward with the weight prepared once (w_s8 = codes ^ 0x80, w_sums
// its row sums): x [..., K] -> dynamic quantize -> GEMM with the bias in the
// epilogue -> [..., N] in x's dtype (torch's promotion with the bias dtype).
// None outside the common case.
py::object linear_prepared(const at::Tensor& x, const at::Tensor& w_s8, const at::Tensor& w_sums,
                           const at::Tensor& w_scale, const c10::optional<at::Tensor>& bias) {
  if (!common_ok(x) || x.dim() < 1) return py::none();
  const int64_t K = x.size(-1);
  const int64_t N = w_s8.size(0);
  if (K % 16 != 0 || w_s8.dim() != 2 || w_s8.size(1) != K || w_s8.scalar_type() != at::kChar ||
      !w_s8.is_contiguous() || w_s8.device() != x.device() || w_sums.device() != x.device() ||
      w_sums.scalar_type() != at::kInt || w_scale.device() != x.device() || w_scale.scalar_type() != at::kFloat ||
      !w_scale.is_contiguous() || w_scale.numel() != 1)
    return py::none();
  const at::Tensor* b = nullptr;
  if (bias.has_value()) {
    b = &bias.value();
    if (b->device() != x.device() || !b->is_contiguous() || !is_float(b->scalar_type()) || b->numel() != N)
      return py::none();
  }
  const c10::cuda::CUDAGuard guard(x.device());
  const auto st = at::cuda::getCurrentCUDAStream(x.device().index()).stream();
  const int64_t M = x.numel() / K;
  const auto gemm_type = x.scalar_type();
  const auto res_type = b ? at::promote_types(gemm_type, b->scalar_type()) : gemm_type;
  std::vector<int64_t> out_shape(x.sizes().begin(), x.sizes().end());
  out_shape.back() = N;
  at::Tensor out = at::empty(out_shape, x.options().dtype(res_type));
  if (out.numel() == 0) return py::cast(out);
  at::Tensor codes = at::empty({M, K}, x.options().dtype(at::kByte));
  at::Tensor x_scale = at::empty({}, x.options().dtype(at::kFloat));
  const size_t ws_bytes = std::max(tfo_fp8_scale_workspace_bytes(M * K),
                                   tfo_fp8_gemm_workspace_bytes(M, N, K, TFO_DTYPE_U8, TFO_B_NK));
  at::Tensor ws = workspace(ws_bytes, x.device(), st);  // the two calls run in stream order
  check(tfo_fp8_quantize(x.data_ptr(), M * K, dtype_code(gemm_type), nullptr, x_scale.data_ptr<float>(),
                         codes.data_ptr(), TFO_DTYPE_U8, ws.data_ptr(), static_cast<size_t>(ws.numel()), st),
        "tfo_fp8_quantize");
  check(tfo_fp8_linear_prepared(codes.data_ptr(), w_s8.data_ptr(), w_sums.data_ptr<int32_t>(),
                                x_scale.data_ptr<float>(), w_scale.data_ptr<float>(), b ? b->data_ptr() : nullptr,
                                b ? dtype_code(b->scalar_type()) : -1, out.data_ptr(), M, N, K, dtype_code(gemm_type),
                                dtype_code(res_type), ws.data_ptr(), static_cast<size_t>(ws.numel()), st),
        "tfo_fp8_linear_prepared");
  return py::cast(out);
}

// ---------------------------------------------------------------------------
// The query/key path: rotary tables, rotation of heads, per-head norm with the
// rotation, with their gradients as autograd nodes (the Python wrappers carry
// the same for inputs outside the common case).
// ---------------------------------------------------------------------------
using OptTensor = c10::optional<at::Tensor>;

// A contiguous tensor straight from the CUDA allocator (at::empty takes the
// dispatcher's way to the same place, about half a microsecond longer).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

// Scratch of one call of several launches (undefined for none). Not kept
// between calls: gradients run on a thread of their own and two threads may
// call on one stream, so that launches of two calls may alternate there.
at::Tensor scratch(size_t bytes, const at::Device& dev) {
  return bytes == 0 ? at::Tensor() : fresh({static_cast<int64_t>(bytes)}, at::kByte, dev);
}

using Strides3 = std::array<int64_t, 3>;

int pos_code(at::ScalarType t) {
  return t == at::kInt ? TFO_POS_I32 : t == at::kLong ? TFO_POS_I64 : -1;
}

// (batch, seq, head) strides of [batch, seq, heads, dim] or [tokens, heads, dim].
Strides3 strides_of(const at::Tensor& t) {
  if (t.dim() == 4) return {t.stride(0), t.stride(1), t.stride(2)};
  return {0, t.stride(0), t.stride(1)};
}

bool heads_ok(const at::Tensor& t) {
  return t.is_cuda() && is_float(t.scalar_type()) && (t.dim() == 3 || t.dim() == 4) && t.numel() > 0 &&
         t.stride(-1) == 1;
}

bool weight_ok(const OptTensor& w, const at::Tensor& q) {
  return !w.has_value() || (w->device() == q.device() && is_float(w->scalar_type()) && w->dim() == 1 &&
                            w->size(0) == q.size(-1) && w->is_contiguous() && !w->_fw_grad(0).defined());
}

// Forward mode: the Python wrappers refuse what carries a tangent.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }

// Everything the shared arguments of the head functions must satisfy here.
bool heads_common(const at::Tensor& q, const OptTensor& k, const at::Tensor& cos, const at::Tensor& sin,
                  const OptTensor& positions) {
  if (!heads_ok(q)) return false;
  if (k.has_value()) {
    if (!heads_ok(*k) || k->device() != q.device() || k->scalar_type() != q.scalar_type() || k->dim() != q.dim() ||
        k->size(-1) != q.size(-1))
      return false;
    for (int64_t i = 0; i < q.dim() - 2; ++i)
      if (k->size(i) != q.size(i)) return false;
  }
  if (cos.device() != q.device() || sin.device() != q.device() || cos.dim() != 2 || sin.dim() != 2 ||
      !is_float(cos.scalar_type()) || sin.scalar_type() != cos.scalar_type() || cos.sizes() != sin.sizes() ||
      cos.strides() != sin.strides() || cos.stride(1) != 1 || cos.requires_grad() || sin.requires_grad())
    return false;
  if (has_tangent(q) || has_tangent(k) || has_tangent(cos) || has_tangent(sin)) return false;
  const int64_t dim = q.size(-1), rot = cos.size(1);
  if (dim < 2 || dim > 1024 || rot < 2 || rot % 2 != 0 || rot > dim || cos.size(0) == 0) return false;
  if (!positions.has_value()) return cos.size(0) >= q.size(-3);
  if (positions->device() != q.device() || pos_code(positions->scalar_type()) < 0 || positions->dim() != q.dim() - 2)
    return false;
  for (int64_t i = 0; i < q.dim() - 2; ++i)
    if (positions->size(i) != q.size(i)) return false;
  return true;
}

struct HeadsCall {  // the C ABI's shared arguments
  const at::Tensor* positions;
  int pos_dtype = TFO_POS_NONE;
  int64_t pos_sb = 0, pos_ss = 0, batch, seq, q_heads, k_heads, dim, rot;
  HeadsCall(const at::Tensor& q, const at::Tensor& k, const at::Tensor& cos, const at::Tensor& pos) : positions(&pos) {
    if (pos.defined()) {
      pos_dtype = pos_code(pos.scalar_type());
      pos_sb = q.dim() == 4 ? pos.stride(0) : 0;
      pos_ss = pos.stride(-1);
    }
    batch = q.dim() == 4 ? q.size(0) : 1;
    seq = q.size(-3);
    q_heads = q.size(-2);
    k_heads = k.defined() ? k.size(-2) : 0;
    dim = q.size(-1);
    rot = cos.size(1);
  }
  const void* pos_ptr() const { return positions->defined() ? positions->data_ptr() : nullptr; }
};

const void* ptr_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* out_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
at::Tensor empty_heads(const at::Tensor& t) {
  return t.defined() ? fresh(t.sizes(), t.scalar_type(), t.device()) : at::Tensor();
}
at::Tensor dense_heads(const at::Tensor& t) {
  return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
int weight_code(const at::Tensor& w) { return w.defined() ? dtype_code(w.scalar_type()) : TFO_DTYPE_F32; }

std::array<at::Tensor, 2> rope_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& cos,
                                    const at::Tensor& sin, const at::Tensor& positions, bool interleaved, bool inverse) {
  const c10::cuda::CUDAGuard guard(q.device());
  const HeadsCall h(q, k, cos, positions);
  std::array<at::Tensor, 2> out{empty_heads(q), empty_heads(k)};
  const Strides3 qs = strides_of(q), ks = k.defined() ? strides_of(k) : Strides3{};
  check(tfo_rope(q.data_ptr(), qs.data(), ptr_or_null(k), ks.data(), cos.data_ptr(), sin.data_ptr(), cos.stride(0),
                 cos.size(0), h.pos_ptr(), h.pos_dtype, h.pos_sb, h.pos_ss, out[0].data_ptr(), out_or_null(out[1]),
                 h.batch, h.seq, h.q_heads, h.k_heads, h.dim, h.rot, interleaved, inverse,
                 dtype_code(q.scalar_type()), dtype_code(cos.scalar_type()),
                 at::cuda::getCurrentCUDAStream(q.device().index()).stream()),
        "tfo_rope");
  return out;
}

std::array<at::Tensor, 2> qk_norm_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw,
                                       const at::Tensor& kw, const at::Tensor& cos, const at::Tensor& sin,
                                       const at::Tensor& positions, double eps, bool interleaved) {
  const c10::cuda::CUDAGuard guard(q.device());
  const HeadsCall h(q, k, cos, positions);
  std::array<at::Tensor, 2> out{empty_heads(q), empty_heads(k)};
  const Strides3 qs = strides_of(q), ks = k.defined() ? strides_of(k) : Strides3{};
  check(tfo_qk_norm_rope(q.data_ptr(), qs.data(), ptr_or_null(k), ks.data(), ptr_or_null(qw), ptr_or_null(kw),
                         cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.size(0), h.pos_ptr(), h.pos_dtype, h.pos_sb,
                         h.pos_ss, out[0].data_ptr(), out_or_null(out[1]), h.batch, h.seq, h.q_heads, h.k_heads, h.dim,
                         h.rot, interleaved, eps, dtype_code(q.scalar_type()), weight_code(qw), weight_code(kw),
                         dtype_code(cos.scalar_type()), at::cuda::getCurrentCUDAStream(q.device().index()).stream()),
        "tfo_qk_norm_rope");
  return out;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

variable_list outputs_of(const std::array<at::Tensor, 2>& out) {
  return out[1].defined() ? variable_list{out[0], out[1]} : variable_list{out[0]};
}

// Forward mode over a backward pass: a gradient's tangent would be lost.
void refuse_tangents(const variable_list& grads) {
  for (const at::Tensor& g : grads)
    TORCH_CHECK_VALUE(!g.defined() || !has_tangent(g), "a gradient carries a forward-mode tangent: only reverse-mode gradients are there");
}

// Puts a node that only raises between the gradients and what they depend on.
void differentiable_once(const variable_list& gradients, const variable_list& sources) {
  const auto node = std::make_shared<torch::autograd::Error>(
      "fused_qk_norm_rope is differentiable once: its gradients cannot be differentiated",
      torch::autograd::collect_next_edges(sources));
  for (const at::Tensor& g : gradients)
    if (g.defined()) torch::autograd::set_history(g, node);
}

// The gradient of a rotation is the rotation by the opposite angle, itself differentiable.
struct RopeNode : public torch::autograd::Function<RopeNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const OptTensor& k, const at::Tensor& cos,
                               const at::Tensor& sin, const OptTensor& positions, bool interleaved, bool inverse) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor pos = positions.value_or(at::Tensor()), kt = k.value_or(at::Tensor());
    ctx->save_for_backward({cos, sin, pos});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    return outputs_of(rope_call(q, kt, cos, sin, pos, interleaved, inverse));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_tangents(grads);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor dq = dense_heads(grads[0]);
    OptTensor dk, pos;
    if (grads.size() > 1) dk = dense_heads(grads[1]);
    if (saved[2].defined()) pos = saved[2];
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = !ctx->saved_data["inverse"].toBool();
    const variable_list d =
        at::GradMode::is_enabled()
            ? RopeNode::apply(dq, dk, saved[0], saved[1], pos, interleaved, inverse)
            : outputs_of(rope_call(dq, dk.value_or(at::Tensor()), saved[0], saved[1], saved[2], interleaved, inverse));
    return {d[0], d.size() > 1 ? d[1] : at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor()};
  }
};

struct QKNormRopeNode : public torch::autograd::Function<QKNormRopeNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const OptTensor& k, const OptTensor& qw,
                               const OptTensor& kw, const at::Tensor& cos, const at::Tensor& sin,
                               const OptTensor& positions, double eps, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor kt = k.value_or(at::Tensor()), qwt = qw.value_or(at::Tensor()), kwt = kw.value_or(at::Tensor()),
                     pos = positions.value_or(at::Tensor());
    ctx->save_for_backward({q, kt, qwt, kwt, cos, sin, pos});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["dqw"] = qwt.defined() && qwt.requires_grad();
    ctx->saved_data["dkw"] = kwt.defined() && kwt.requires_grad();
    return outputs_of(qk_norm_call(q, kt, qwt, kwt, cos, sin, pos, eps, interleaved));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list d = gradients(ctx, saved, grads);
    if (at::GradMode::is_enabled()) {  // create_graph: differentiating one of the gradients is the error
      variable_list sources(saved.begin(), saved.begin() + 4);
      sources.insert(sources.end(), grads.begin(), grads.end());
      differentiable_once(d, sources);
    }
    return d;
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& saved, const variable_list& grads) {
    const at::AutoGradMode no_graph(false);
    refuse_tangents(grads);
    const at::Tensor &q = saved[0], &k = saved[1], &qw = saved[2], &kw = saved[3], &cos = saved[4], &sin = saved[5];
    const c10::cuda::CUDAGuard guard(q.device());
    const auto st = at::cuda::getCurrentCUDAStream(q.device().index()).stream();
    const HeadsCall h(q, k, cos, saved[6]);
    const at::Tensor gq = dense_heads(grads[0]), gk = k.defined() ? dense_heads(grads[1]) : at::Tensor();
    const at::Tensor dq = empty_heads(q), dk = empty_heads(k);
    at::Tensor dqw, dkw, ws;
    if (ctx->saved_data["dqw"].toBool()) dqw = fresh(qw.sizes(), qw.scalar_type(), qw.device());
    if (ctx->saved_data["dkw"].toBool()) dkw = fresh(kw.sizes(), kw.scalar_type(), kw.device());
    if (dqw.defined() || dkw.defined()) ws = scratch(tfo_qk_norm_rope_backward_workspace_bytes(h.dim), q.device());
    const Strides3 qs = strides_of(q), gqs = strides_of(gq), ks = k.defined() ? strides_of(k) : Strides3{},
                   gks = k.defined() ? strides_of(gk) : Strides3{};
    check(tfo_qk_norm_rope_backward(
              gq.data_ptr(), gqs.data(), ptr_or_null(gk), gks.data(), q.data_ptr(), qs.data(), ptr_or_null(k), ks.data(),
              ptr_or_null(qw), ptr_or_null(kw), cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.size(0), h.pos_ptr(),
              h.pos_dtype, h.pos_sb, h.pos_ss, dq.data_ptr(), out_or_null(dk), out_or_null(dqw), out_or_null(dkw),
              h.batch, h.seq, h.q_heads, h.k_heads, h.dim, h.rot, ctx->saved_data["interleaved"].toBool(),
              ctx->saved_data["eps"].toDouble(), dtype_code(q.scalar_type()), weight_code(qw), weight_code(kw),
              dtype_code(cos.scalar_type()), out_or_null(ws), ws.defined() ? static_cast<size_t>(ws.numel()) : 0, st),
          "tfo_qk_norm_rope_backward");
    return {dq, dk, dqw, dkw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

py::object pair_of(const variable_list& out) {
  if (out.size() > 1) return py::make_tuple(out[0], out[1]);
  return py::make_tuple(out[0], py::none());
}

// fused_rope: (q, k or None) rotated, or None outside the common case.
py::object rope(const at::Tensor& q, const OptTensor& k, const at::Tensor& cos, const at::Tensor& sin,
                const OptTensor& positions, bool interleaved) {
  if (!heads_common(q, k, cos, sin, positions)) return py::none();
  if (at::GradMode::is_enabled() && (q.requires_grad() || wants_grad(k)))
    return pair_of(RopeNode::apply(q, k, cos, sin, positions, interleaved, false));
  return pair_of(outputs_of(rope_call(q, k.value_or(at::Tensor()), cos, sin, positions.value_or(at::Tensor()),
                                      interleaved, false)));
}

// fused_qk_norm_rope: (q, k or None) normed and rotated, or None outside the common case.
py::object qk_norm_rope(const at::Tensor& q, const OptTensor& k, const OptTensor& qw, const OptTensor& kw,
                        const at::Tensor& cos, const at::Tensor& sin, const OptTensor& positions, double eps,
                        bool interleaved) {
  if (!heads_common(q, k, cos, sin, positions) || !weight_ok(qw, q) || (k.has_value() ? !weight_ok(kw, q) : kw.has_value()))
    return py::none();
  if (at::GradMode::is_enabled() && (q.requires_grad() || wants_grad(k) || wants_grad(qw) || wants_grad(kw)))
    return pair_of(QKNormRopeNode::apply(q, k, qw, kw, cos, sin, positions, eps, interleaved));
  return pair_of(outputs_of(qk_norm_call(q, k.value_or(at::Tensor()), qw.value_or(at::Tensor()),
                                         kw.value_or(at::Tensor()), cos, sin, positions.value_or(at::Tensor()), eps,
                                         interleaved)));
}

// rope_tables of given positions: (cos, sin), or None outside the common case. turns: doubles in host memory.
py::object rope_tables(const at::Tensor& positions, const at::Tensor& turns, double gain, int64_t out_code) {
  if (!positions.is_cuda() || !positions.is_contiguous() || pos_code(positions.scalar_type()) < 0) return py::none();
  if (!turns.is_cpu() || turns.scalar_type() != at::kDouble || !turns.is_contiguous()) return py::none();
  const c10::cuda::CUDAGuard guard(positions.device());
  const int64_t half = turns.numel();
  std::vector<int64_t> shape(positions.sizes().begin(), positions.sizes().end());
  shape.push_back(2 * half);
  const auto type = out_code == TFO_DTYPE_F16 ? at::kHalf : out_code == TFO_DTYPE_BF16 ? at::kBFloat16 : at::kFloat;
  at::Tensor cos = fresh(shape, type, positions.device());
  at::Tensor sin = fresh(shape, type, positions.device());
  check(tfo_rope_tables(positions.data_ptr(), pos_code(positions.scalar_type()), positions.numel(),
                        turns.data_ptr<double>(), half, gain, cos.data_ptr(), sin.data_ptr(),
                        static_cast<int>(out_code),
                        at::cuda::getCurrentCUDAStream(positions.device().index()).stream()),
        "tfo_rope_tables");
  return py::make_tuple(cos, sin);
}

// fused_lora on 2-D operands: the result, or None outside the common case.
py::object lora(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const at::Tensor& ids,
                const OptTensor& scaling, const OptTensor& base, const OptTensor& out) {
  if (!x.is_cuda() || !is_float(x.scalar_type()) || x.dim() != 2 || x.stride(1) != 1 || a.dim() != 3 || b.dim() != 3)
    return py::none();
  const int64_t tokens = x.size(0), k = x.size(1), adapters = a.size(0), rank = a.size(1), n = b.size(1);
  auto same = [&](const at::Tensor& t) { return t.device() == x.device() && t.scalar_type() == x.scalar_type(); };
  if (!same(a) || !same(b) || !a.is_contiguous() || !b.is_contiguous() || a.size(2) != k || b.size(0) != adapters ||
      b.size(2) != rank || adapters < 1 || adapters > 16384 || rank < 1 || rank > 256 || k < 1 || n < 1 || tokens < 1)
    return py::none();
  if (ids.device() != x.device() || pos_code(ids.scalar_type()) < 0 || ids.dim() != 1 || ids.size(0) != tokens ||
      !ids.is_contiguous())
    return py::none();
  if (scaling.has_value() && (scaling->device() != x.device() || scaling->scalar_type() != at::kFloat ||
                              scaling->dim() != 1 || scaling->size(0) != adapters || !scaling->is_contiguous()))
    return py::none();
  for (const OptTensor* t : {&base, &out}) {
    if (t->has_value() && (!same(**t) || (*t)->dim() != 2 || (*t)->size(0) != tokens || (*t)->size(1) != n ||
                           (*t)->stride(1) != 1))
      return py::none();
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || a.requires_grad() || b.requires_grad() ||
                                     wants_grad(scaling) || wants_grad(base) || wants_grad(out)))
    return py::none();
  if (has_tangent(x) || has_tangent(a) || has_tangent(b) || has_tangent(scaling) || has_tangent(base) || has_tangent(out))
    return py::none();
  // rows of one output may not share memory
  if (out.has_value() && tokens > 1 && out->stride(0) < n) return py::none();
  const c10::cuda::CUDAGuard guard(x.device());
  const auto st = at::cuda::getCurrentCUDAStream(x.device().index()).stream();
  at::Tensor y = out.has_value() ? *out : fresh({tokens, n}, x.scalar_type(), x.device());
  // written through its pointer: autograd has to know, if it keeps out for a backward pass
  if (out.has_value() && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
  const int dtype = dtype_code(x.scalar_type());
  const at::Tensor ws = scratch(tfo_lora_workspace_bytes(tokens, adapters), x.device());
  check(tfo_lora(x.data_ptr(), x.stride(0), a.data_ptr(), b.data_ptr(), ids.data_ptr(), pos_code(ids.scalar_type()),
                 scaling.has_value() ? scaling->data_ptr<float>() : nullptr,
                 base.has_value() ? base->data_ptr() : nullptr, base.has_value() ? base->stride(0) : 0, y.data_ptr(),
                 y.stride(0), tokens, adapters, rank, k, n, dtype, out_or_null(ws),
                 ws.defined() ? static_cast<size_t>(ws.numel()) : 0, st),
        "tfo_lora");
  return py::cast(y);
}

}  // namespace

PYBIND11_MODULE(_tfo_ext, m) {
  m.doc() = "PyTorch entry points over the tfo_b200 C ABI for launch-latency-bound calls";
  m.def("quantize_dynamic", &quantize_dynamic, "dynamic-scale quantize (codes, scale) or None");
  m.def("linear_prepared", &linear_prepared, "FP8Linear forward with a prepared weight, or None");
  m.def("rope", &rope, "fused_rope, or None");
  m.def("qk_norm_rope", &qk_norm_rope, "fused_qk_norm_rope, or None");
  m.def("rope_tables", &rope_tables, "rope_tables of given positions, or None");
  m.def("lora", &lora, "fused_lora on 2-D operands, or None");
  m.def("clear_workspaces", &clear_workspaces, "releases the cached scratch buffers");
}
