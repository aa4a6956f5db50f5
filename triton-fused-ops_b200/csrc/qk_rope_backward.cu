// Gradients of the per-head RMSNorm with rotation (qk_rope.cu).
//
//   r  = 1 / sqrt(mean(x^2) + eps)
//   b  = the inverse rotation of dy           (b = dy past rotary_dim)
//   dx = r * (b w) - x * r^3 * mean(b w x)
//   dw = sum over tokens and heads of b * x * r
//
// Both means come from one read of x and dy; nothing of the forward pass is
// stored. Bound by HBM (x and dy read, dx written). CTAs are persistent, split
// between queries and keys by their work; a lane keeps fp32 sums of dw for its
// columns over all its rows, a CTA joins its lanes' sums through shared memory
// into one partial row, and a second kernel adds the partial rows in order, so
// the result does not depend on scheduling (no atomics).
#include "heads.cuh"

namespace tfo {

constexpr int kBwdThreads = 256;
constexpr int kBwdWarps = kBwdThreads / 32;
constexpr int kBwdCtasPerSm = 4;

struct SideSplit {  // CTAs [0, q_ctas) take the queries, the rest the keys
  int q_ctas, k_ctas;
};

template <typename T, int E, bool PAIRS, int NH>
__global__ void __launch_bounds__(kBwdThreads) qk_norm_rope_backward_kernel(const HeadArgs a, int lane_shift,
                                                                            SideSplit split, float* __restrict__ partials,
                                                                            uint32_t* err) {
  using V = HeadVec<T, E>;
  extern __shared__ float red[];  // [kBwdWarps][head_dim]
  griddep_launch_dependents();
  griddep_wait();
  const bool is_q = blockIdx.x < static_cast<unsigned>(split.q_ctas);
  const HeadSide& side = is_q ? a.q : a.k;
  const uint32_t cta = is_q ? blockIdx.x : blockIdx.x - split.q_ctas;
  const uint32_t ctas = is_q ? split.q_ctas : split.k_ctas;
  const int D = a.head_dim, heads = side.heads;
  const int lanes = 1 << lane_shift;
  const int p = threadIdx.x & (lanes - 1);
  const uint32_t per_cta = kBwdThreads >> lane_shift;
  const uint32_t chunks = (heads + NH - 1) / NH;
  const uint32_t groups = static_cast<uint32_t>(a.batch * a.seq) * chunks;
  const LaneCols col = lane_cols<PAIRS>(p, D / E, a.rotary_dim / E);
  const float inv_d = 1.f / static_cast<float>(D);

  float wa[E], wb[E], acc_a[E], acc_b[E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    wa[j] = wb[j] = 1.f;
    acc_a[j] = acc_b[j] = 0.f;
  }
  if (side.weight != nullptr) {
    if (col.va >= 0) load_floats<E>(side.weight, col.va * E, side.w_dtype, wa);
    if (col.vb >= 0) load_floats<E>(side.weight, col.vb * E, side.w_dtype, wb);
  }
  for (uint32_t base = cta * per_cta; base < groups; base += ctas * per_cta) {
    const uint32_t want = base + (threadIdx.x >> lane_shift);
    const bool live = want < groups;
    const uint32_t gid = live ? want : groups - 1;
    const uint32_t token = gid / chunks;
    const int h0 = static_cast<int>(gid - token * chunks) * NH;
    const uint32_t b = token / static_cast<uint32_t>(a.seq);
    const uint32_t sq = token - b * static_cast<uint32_t>(a.seq);
    const T* x = static_cast<const T*>(side.x) + b * side.stride_batch + sq * side.stride_seq;
    const T* dy = static_cast<const T*>(side.dy) + b * side.dy_stride_batch + sq * side.dy_stride_seq;
    typename V::Raw xa[NH], xb[NH], ga[NH], gb[NH];
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      const bool in = live && h0 + i < heads;
      const T* xr = x + (h0 + i) * side.stride_head;
      const T* gr = dy + (h0 + i) * side.dy_stride_head;
      xa[i] = in && col.va >= 0 ? V::load(xr + col.va * E) : V::zero();
      xb[i] = in && col.vb >= 0 ? V::load(xr + col.vb * E) : V::zero();
      ga[i] = in && col.va >= 0 ? V::load(gr + col.va * E) : V::zero();
      gb[i] = in && col.vb >= 0 ? V::load(gr + col.vb * E) : V::zero();
    }
    const int64_t pos = token_position(a.t, b, sq, err, p == 0);
    float c[E], s[E];
    lane_table<E>(a.t, pos, p, col.rotated, true, c, s);
    T* out = static_cast<T*>(side.out) + (static_cast<int64_t>(token) * heads + h0) * D;
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      float ua[E], ub[E], fa[E], fb[E];
      V::unpack(xa[i], ua);
      V::unpack(xb[i], ub);
      V::unpack(ga[i], fa);
      V::unpack(gb[i], fb);
      rotate_lane<E, PAIRS>(fa, fb, c, s, col.rotated);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        ss += ua[j] * ua[j] + ub[j] * ub[j];
        dot += fa[j] * wa[j] * ua[j] + fb[j] * wb[j] * ub[j];
      }
      ss = group_sum(ss, lanes);
      dot = group_sum(dot, lanes);
      const float r = rsqrtf(ss * inv_d + a.eps);
      const float k = dot * inv_d * r * r * r;  // in this order: r^3 alone can overflow
      if (live && h0 + i < heads) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          acc_a[j] += fa[j] * (ua[j] * r);
          acc_b[j] += fb[j] * (ub[j] * r);
          ua[j] = r * (fa[j] * wa[j]) - ua[j] * k;
          ub[j] = r * (fb[j] * wb[j]) - ub[j] * k;
        }
        if (col.va >= 0) V::store(out + i * D + col.va * E, ua);
        if (col.vb >= 0) V::store(out + i * D + col.vb * E, ub);
      }
    }
  }
  if (side.dweight == nullptr) return;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    for (int o = lanes; o < 32; o <<= 1) {
      acc_a[j] += __shfl_xor_sync(0xffffffffu, acc_a[j], o);
      acc_b[j] += __shfl_xor_sync(0xffffffffu, acc_b[j], o);
    }
  }
  float* mine = red + (threadIdx.x >> 5) * D;
  if ((threadIdx.x & 31) < lanes) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (col.va >= 0) mine[col.va * E + j] = acc_a[j];
      if (col.vb >= 0) mine[col.vb * E + j] = acc_b[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kBwdThreads) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kBwdWarps; ++w) t += red[w * D + i];
    partials[static_cast<int64_t>(blockIdx.x) * D + i] = t;
  }
}

// Any head width, stride and alignment: one warp per head, scalar accesses,
// the sums of dw in shared memory (each column belongs to one lane).
template <typename T>
__global__ void __launch_bounds__(kBwdThreads) qk_norm_rope_backward_any_kernel(const HeadArgs a, SideSplit split,
                                                                                float* __restrict__ partials,
                                                                                uint32_t* err) {
  extern __shared__ float red[];  // [kBwdWarps][head_dim]
  griddep_launch_dependents();
  griddep_wait();
  const bool is_q = blockIdx.x < static_cast<unsigned>(split.q_ctas);
  const HeadSide& side = is_q ? a.q : a.k;
  const int64_t cta = is_q ? blockIdx.x : blockIdx.x - split.q_ctas;
  const int64_t ctas = is_q ? split.q_ctas : split.k_ctas;
  const int D = a.head_dim, half = a.rotary_dim / 2, heads = side.heads;
  const int lane = threadIdx.x & 31;
  float* acc = red + (threadIdx.x >> 5) * D;
  for (int i = lane; i < D; i += 32) acc[i] = 0.f;
  __syncwarp();
  const int64_t rows = a.batch * a.seq * heads;
  for (int64_t row = cta * kBwdWarps + (threadIdx.x >> 5); row < rows; row += ctas * kBwdWarps) {
    const int64_t token = row / heads;
    const int h = static_cast<int>(row - token * heads);
    const int64_t b = token / a.seq, sq = token - b * a.seq;
    const T* x = static_cast<const T*>(side.x) + b * side.stride_batch + sq * side.stride_seq + h * side.stride_head;
    const T* dy =
        static_cast<const T*>(side.dy) + b * side.dy_stride_batch + sq * side.dy_stride_seq + h * side.dy_stride_head;
    T* out = static_cast<T*>(side.out) + row * D;
    const int64_t pos = token_position(a.t, b, sq, err, lane == 0);
    auto weight = [&](int i) { return side.weight != nullptr ? load_as_float(side.weight, i, side.w_dtype) : 1.f; };
    // calls f(column, b) for each of this lane's columns
    auto each = [&](auto f) {
      for (int i = lane; i < half; i += 32) {
        float c, s;
        if (pos < 0) {
          c = s = __int_as_float(0x7fffffff);
        } else {
          c = load_as_float(a.t.cos, pos * a.t.row_stride + i, a.t.dtype);
          s = load_as_float(a.t.sin, pos * a.t.row_stride + i, a.t.dtype);
        }
        const int i1 = a.pairs ? 2 * i : i, i2 = a.pairs ? 2 * i + 1 : i + half;
        const float u = Ty<T>::to_f(dy[i1]), v = Ty<T>::to_f(dy[i2]);
        f(i1, u * c + v * s);
        f(i2, v * c - u * s);
      }
      for (int i = 2 * half + lane; i < D; i += 32) f(i, Ty<T>::to_f(dy[i]));
    };
    float ss = 0.f, dot = 0.f;
    each([&](int i, float g) {
      const float v = Ty<T>::to_f(x[i]);
      ss += v * v;
      dot += g * weight(i) * v;
    });
    const float r = rsqrtf(warp_sum(ss) / static_cast<float>(D) + a.eps);
    const float k = warp_sum(dot) / static_cast<float>(D) * r * r * r;
    each([&](int i, float g) {
      const float v = Ty<T>::to_f(x[i]);
      acc[i] += g * (v * r);
      out[i] = Ty<T>::from_f(r * (g * weight(i)) - v * k);
    });
  }
  if (side.dweight == nullptr) return;
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kBwdThreads) {
    float t = 0.f;
    for (int w = 0; w < kBwdWarps; ++w) t += red[w * D + i];
    partials[static_cast<int64_t>(blockIdx.x) * D + i] = t;
  }
}

// dw[i] = the sum of a side's partial rows: 32 columns per CTA, one side per grid row.
__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const HeadArgs a, SideSplit split,
                                                              const float* __restrict__ partials) {
  __shared__ float red[32][33];
  griddep_launch_dependents();
  griddep_wait();
  const HeadSide& side = blockIdx.y == 0 ? a.q : a.k;
  if (side.dweight == nullptr) return;
  const int first = blockIdx.y == 0 ? 0 : split.q_ctas;
  const int rows = blockIdx.y == 0 ? split.q_ctas : split.k_ctas;
  const int D = a.head_dim;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + x;
  float t = 0.f;
  if (i < D) {
    for (int r = y; r < rows; r += 32) t += partials[static_cast<int64_t>(first + r) * D + i];
  }
  red[y][x] = t;
  __syncthreads();
  t = warp_sum(red[x][y]);  // warp y sums column y
  const int o = blockIdx.x * 32 + y;
  if (x == 0 && o < D) {
    if (side.w_dtype == F32) {
      static_cast<float*>(side.dweight)[o] = t;
    } else if (side.w_dtype == F16) {
      static_cast<__half*>(side.dweight)[o] = __float2half_rn(t);
    } else {
      static_cast<__nv_bfloat16*>(side.dweight)[o] = __float2bfloat16_rn(t);
    }
  }
}

namespace {
// CTAs of each side in proportion to its heads, at most one wave and no more than `units(heads)` CTAs of work.
template <typename F> SideSplit split_ctas(const HeadArgs& a, F units) {
  const int64_t all = static_cast<int64_t>(num_sms()) * kBwdCtasPerSm;
  const int heads = a.q.heads + a.k.heads;
  auto share = [&](int h) -> int {
    if (h == 0) return 0;
    return static_cast<int>(std::min<int64_t>(units(h), std::max<int64_t>(1, all * h / heads)));
  };
  return SideSplit{share(a.q.heads), share(a.k.heads)};
}

template <typename... KArgs, typename... Args>
cudaError_t launch_smem(void (*kernel)(KArgs...), int grid, int block, size_t smem, cudaStream_t st, Args&&... args) {
  return launch_gemm_grid(kernel, block, grid, 1, smem, st, std::forward<Args>(args)...);
}

template <typename T, int E, bool PAIRS>
cudaError_t launch_vec(const HeadArgs& a, SideSplit* split, float* partials, cudaStream_t st) {
  constexpr int NH = 2;
  const int lanes = (a.head_dim / E + 1) / 2;
  int shift = 0;
  while ((1 << shift) < lanes) ++shift;
  const int64_t per_cta = kBwdThreads >> shift;
  *split = split_ctas(a, [&](int h) { return (a.batch * a.seq * ((h + NH - 1) / NH) + per_cta - 1) / per_cta; });
  note_launch();
  return launch_smem(qk_norm_rope_backward_kernel<T, E, PAIRS, NH>, split->q_ctas + split->k_ctas, kBwdThreads,
                     sizeof(float) * kBwdWarps * a.head_dim, st, a, shift, *split, partials, error_word_ptr());
}

template <typename T>
cudaError_t launch_type(const HeadArgs& a, SideSplit* split, float* partials, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const int e = head_vector_elems(a, true);
  if (e == E)
    return a.pairs ? launch_vec<T, E, true>(a, split, partials, st) : launch_vec<T, E, false>(a, split, partials, st);
  if (e == E / 2)
    return a.pairs ? launch_vec<T, E / 2, true>(a, split, partials, st)
                   : launch_vec<T, E / 2, false>(a, split, partials, st);
  *split = split_ctas(a, [&](int h) { return (a.batch * a.seq * h + kBwdWarps - 1) / kBwdWarps; });
  note_launch();
  return launch_smem(qk_norm_rope_backward_any_kernel<T>, split->q_ctas + split->k_ctas, kBwdThreads,
                     sizeof(float) * kBwdWarps * a.head_dim, st, a, *split, partials, error_word_ptr());
}
}  // namespace

size_t qk_norm_rope_backward_workspace_bytes(int head_dim) {
  return sizeof(float) * static_cast<size_t>(num_sms() * kBwdCtasPerSm + 1) * head_dim;
}

cudaError_t qk_norm_rope_backward_launch(const HeadArgs& a, void* ws, cudaStream_t st) {
  SideSplit split{};
  float* partials = static_cast<float*>(ws);
  cudaError_t e = a.dtype == F16    ? launch_type<__half>(a, &split, partials, st)
                  : a.dtype == BF16 ? launch_type<__nv_bfloat16>(a, &split, partials, st)
                                    : launch_type<float>(a, &split, partials, st);
  if (e != cudaSuccess || (a.q.dweight == nullptr && a.k.dweight == nullptr)) return e;
  const dim3 grid((a.head_dim + 31) / 32, 2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, qk_weight_grad_kernel, a, split, static_cast<const float*>(partials));
}

}  // namespace tfo
