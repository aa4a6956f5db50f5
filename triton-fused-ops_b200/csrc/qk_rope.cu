// Rotation of query and key heads by rotary table rows, alone or after an
// RMSNorm of each head, in one pass over both tensors.
//
//   u = x / sqrt(mean(x^2) + eps) * w      (norm only; mean over the head)
//   (y1, y2) = (u1 c - u2 s, u1 s + u2 c)  for each rotated pair of columns
//   columns at or past rotary_dim: y = u
//
// Everything is held in fp32 from the load of x to one rounding of y.
//
// Bound by HBM: x is read once and y written once, the table rows come from
// L2. A group of lanes (two vectors each, heads.cuh) owns NH consecutive heads
// of one token: the lane's table columns and weights are loaded once and used
// for the NH heads, whose loads are all issued before the first is used.
#include "heads.cuh"

namespace tfo {

template <typename T, int E, bool PAIRS, bool NORM, int NH>
__global__ void __launch_bounds__(256) qk_rope_kernel(const HeadArgs a, int lane_shift, uint32_t groups, uint32_t q_chunks,
                                                      uint32_t chunks, uint32_t* err) {
  using V = HeadVec<T, E>;
  griddep_launch_dependents();
  griddep_wait();
  const uint32_t thread = blockIdx.x * 256u + threadIdx.x;
  const uint32_t gid = min(thread >> lane_shift, groups - 1);  // spare lanes repeat the last group and store nothing
  const bool live = (thread >> lane_shift) < groups;
  const int lanes = 1 << lane_shift;
  const int p = threadIdx.x & (lanes - 1);
  const uint32_t token = gid / chunks;
  const uint32_t chunk = gid - token * chunks;
  const uint32_t b = token / static_cast<uint32_t>(a.seq);
  const uint32_t sq = token - b * static_cast<uint32_t>(a.seq);
  const HeadSide& side = chunk < q_chunks ? a.q : a.k;
  const int h0 = static_cast<int>(chunk < q_chunks ? chunk : chunk - q_chunks) * NH;
  const int heads = side.heads;
  const int D = a.head_dim;
  const LaneCols col = lane_cols<PAIRS>(p, D / E, a.rotary_dim / E);

  const T* x = static_cast<const T*>(side.x) + b * side.stride_batch + sq * side.stride_seq;
  typename V::Raw ra[NH], rb[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const T* row = x + (h0 + i) * side.stride_head;
    const bool in = h0 + i < heads;
    ra[i] = in && col.va >= 0 ? V::load(row + col.va * E) : V::zero();
    rb[i] = in && col.vb >= 0 ? V::load(row + col.vb * E) : V::zero();
  }
  const int64_t pos = token_position(a.t, b, sq, err, p == 0);
  float c[E], s[E];
  lane_table<E>(a.t, pos, p, col.rotated, a.inverse, c, s);
  float wa[E], wb[E];
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < E; ++j) wa[j] = wb[j] = 1.f;
    if (side.weight != nullptr) {
      if (col.va >= 0) load_floats<E>(side.weight, col.va * E, side.w_dtype, wa);
      if (col.vb >= 0) load_floats<E>(side.weight, col.vb * E, side.w_dtype, wb);
    }
  }
  T* out = static_cast<T*>(side.out) + (static_cast<int64_t>(token) * heads + h0) * D;
  const float inv_d = 1.f / static_cast<float>(D);
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    float fa[E], fb[E];
    V::unpack(ra[i], fa);
    V::unpack(rb[i], fb);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) ss += fa[j] * fa[j] + fb[j] * fb[j];
      const float rstd = rsqrtf(group_sum(ss, lanes) * inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        fa[j] *= rstd * wa[j];
        fb[j] *= rstd * wb[j];
      }
    }
    rotate_lane<E, PAIRS>(fa, fb, c, s, col.rotated);
    if (live && h0 + i < heads) {
      if (col.va >= 0) V::store(out + i * D + col.va * E, fa);
      if (col.vb >= 0) V::store(out + i * D + col.vb * E, fb);
    }
  }
}

// Any head width, stride and alignment: one warp per head, scalar accesses.
template <typename T>
__global__ void __launch_bounds__(256) qk_rope_any_kernel(const HeadArgs a, int64_t rows, uint32_t* err) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int all = a.q.heads + a.k.heads;
  const int D = a.head_dim, half = a.rotary_dim / 2;
  for (int64_t r = blockIdx.x * 8ll + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8ll) {
    const int64_t token = r / all;
    const int at = static_cast<int>(r - token * all);
    const HeadSide& side = at < a.q.heads ? a.q : a.k;
    const int h = at < a.q.heads ? at : at - a.q.heads;
    const int64_t b = token / a.seq, sq = token - b * a.seq;
    const T* x = static_cast<const T*>(side.x) + b * side.stride_batch + sq * side.stride_seq + h * side.stride_head;
    T* out = static_cast<T*>(side.out) + (token * side.heads + h) * D;
    float rstd = 1.f;
    if (a.norm) {
      float ss = 0.f;
      for (int i = lane; i < D; i += 32) {
        const float v = Ty<T>::to_f(x[i]);
        ss += v * v;
      }
      rstd = rsqrtf(warp_sum(ss) / static_cast<float>(D) + a.eps);
    }
    auto value = [&](int i) {
      const float v = Ty<T>::to_f(x[i]);
      if (!a.norm) return v;
      return v * (rstd * (side.weight != nullptr ? load_as_float(side.weight, i, side.w_dtype) : 1.f));
    };
    const int64_t pos = token_position(a.t, b, sq, err, lane == 0);
    for (int i = lane; i < half; i += 32) {
      float c, s;
      if (pos < 0) {
        c = s = __int_as_float(0x7fffffff);
      } else {
        c = load_as_float(a.t.cos, pos * a.t.row_stride + i, a.t.dtype);
        s = load_as_float(a.t.sin, pos * a.t.row_stride + i, a.t.dtype);
      }
      if (a.inverse) s = -s;
      const int i1 = a.pairs ? 2 * i : i, i2 = a.pairs ? 2 * i + 1 : i + half;
      const float u = value(i1), v = value(i2);
      out[i1] = Ty<T>::from_f(u * c - v * s);
      out[i2] = Ty<T>::from_f(u * s + v * c);
    }
    for (int i = 2 * half + lane; i < D; i += 32) out[i] = Ty<T>::from_f(value(i));
  }
}

namespace {
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }

// Every vector of `bytes` bytes of a strided [batch, seq, heads, D] tensor is aligned.
bool rows_aligned(const void* x, const HeadArgs& a, int heads, int64_t sb, int64_t ss, int64_t sh, int esz, int bytes) {
  return aligned(x, bytes) && (a.batch <= 1 || sb * esz % bytes == 0) && (a.seq <= 1 || ss * esz % bytes == 0) &&
         (heads <= 1 || sh * esz % bytes == 0);
}
}  // namespace

int head_vector_elems(const HeadArgs& a, bool backward) {
  const int esz = a.dtype == F32 ? 4 : 2;
  const int64_t tokens = a.batch * a.seq;
  if (tokens * (a.q.heads + a.k.heads) >= (1ll << 26)) return 0;
  for (int bytes = 16; bytes >= 8; bytes /= 2) {
    const int e = bytes / esz;
    if (a.head_dim % e != 0 || a.head_dim / e > 64) continue;
    if (a.pairs ? a.rotary_dim % e != 0 : (a.rotary_dim / 2) % e != 0) continue;
    const int tsz = a.t.dtype == F32 ? 4 : 2;
    const int tb = std::min(16, e * tsz);
    if (!aligned(a.t.cos, tb) || !aligned(a.t.sin, tb) || (a.t.rows > 1 && a.t.row_stride * tsz % tb != 0)) continue;
    bool ok = true;
    for (const HeadSide* s : {&a.q, &a.k}) {
      if (s->heads == 0) continue;
      ok = ok && rows_aligned(s->x, a, s->heads, s->stride_batch, s->stride_seq, s->stride_head, esz, bytes);
      ok = ok && aligned(s->out, bytes);
      const int wsz = s->w_dtype == F32 ? 4 : 2;
      ok = ok && (s->weight == nullptr || aligned(s->weight, std::min(16, e * wsz)));
      if (backward)
        ok = ok && rows_aligned(s->dy, a, s->heads, s->dy_stride_batch, s->dy_stride_seq, s->dy_stride_head, esz, bytes);
    }
    if (ok) return e;
  }
  return 0;
}

namespace {
template <typename T, int E, bool PAIRS, bool NORM, int NH>
cudaError_t launch_vec(const HeadArgs& a, int lane_shift, cudaStream_t st) {
  const uint32_t qc = (a.q.heads + NH - 1) / NH, kc = (a.k.heads + NH - 1) / NH;
  const uint32_t groups = static_cast<uint32_t>(a.batch * a.seq) * (qc + kc);
  const int64_t blocks = ((static_cast<int64_t>(groups) << lane_shift) + 255) / 256;
  note_launch();
  return launch_dependent(qk_rope_kernel<T, E, PAIRS, NORM, NH>, static_cast<int>(blocks), 256, st, a, lane_shift, groups,
                          qc, qc + kc, error_word_ptr());
}

template <typename T, int E>
cudaError_t launch_elems(const HeadArgs& a, cudaStream_t st) {
  const int lanes = (a.head_dim / E + 1) / 2;
  int shift = 0;
  while ((1 << shift) < lanes) ++shift;
  // Four heads per group share the table columns and keep four times the loads
  // in flight; with few tokens one head per group spreads over more SMs.
  const int64_t warps4 = (a.batch * a.seq * ((a.q.heads + 3) / 4 + (a.k.heads + 3) / 4) << shift) / 32;
  const bool many = warps4 >= static_cast<int64_t>(num_sms()) * 16;
#define TFO_QK(P, N) (many ? launch_vec<T, E, P, N, 4>(a, shift, st) : launch_vec<T, E, P, N, 1>(a, shift, st))
  if (a.pairs) return a.norm ? TFO_QK(true, true) : TFO_QK(true, false);
  return a.norm ? TFO_QK(false, true) : TFO_QK(false, false);
#undef TFO_QK
}

template <typename T>
cudaError_t launch_type(const HeadArgs& a, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const int e = head_vector_elems(a, false);
  if (e == E) return launch_elems<T, E>(a, st);
  if (e == E / 2) return launch_elems<T, E / 2>(a, st);
  const int64_t rows = a.batch * a.seq * (a.q.heads + a.k.heads);
  const int64_t blocks = std::min<int64_t>((rows + 7) / 8, static_cast<int64_t>(num_sms()) * 64);
  note_launch();
  return launch_dependent(qk_rope_any_kernel<T>, static_cast<int>(blocks), 256, st, a, rows, error_word_ptr());
}
}  // namespace

cudaError_t qk_rope_launch(const HeadArgs& a, cudaStream_t st) {
  if (a.dtype == F16) return launch_type<__half>(a, st);
  if (a.dtype == BF16) return launch_type<__nv_bfloat16>(a, st);
  return launch_type<float>(a, st);
}

}  // namespace tfo
