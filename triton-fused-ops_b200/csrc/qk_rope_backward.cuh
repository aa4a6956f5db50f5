// Gradients of the per-head RMSNorm with rotation (qk_rope.cu).
//
//   r  = 1 / sqrt(mean(x^2) + eps)
//   b  = the inverse rotation of dy           (b = dy past rotary_dim)
//   dx = r * (b w) - x * r^3 * mean(b w x)
//   dw = sum over tokens and heads of b * x * r
//
// Both means come from one read of x and dy; nothing of the forward pass is
// stored. CTAs are persistent, split between queries and keys by their work,
// and stream both tensors through shared memory (HeadStream); a lane keeps
// fp32 sums of dw for its columns over all its heads, a CTA joins its lanes'
// sums through shared memory into one partial row, and a second kernel adds
// the partial rows in order, so the result does not depend on scheduling (no
// atomics).
//
// Floor: HBM (x and dy read, dx written). Measured at 32768 tokens of 32 + 8
// heads of 128 columns, bf16: 183 us with the weights' gradients, 84 % of the
// measured copy rate; 8192 tokens 53 us (73 %). What bounds it is latency within
// a warp, of which an SM holds 16 (128 registers a thread): the schedulers issue in
// 50 % of the cycles, and waits for loads are the longest stall. A unit's copies are
// issued after the arithmetic of the one before, so that with two stages none is in
// flight meanwhile: a copy's whole latency shows in every unit.
//
// AXES: as for qk_rope.cuh (qk_rope_backward.cu, qk_rope_backward_axes.cu).
#pragma once

#include "heads.cuh"

namespace tfo {

constexpr int kBwdThreads = 256;
constexpr int kBwdWarps = kBwdThreads / 32;
constexpr int kBwdCtasPerSm = 4;

template <typename T, int E, bool PAIRS, int NH, int STAGES, bool FULL, bool AXES>
__global__ void __launch_bounds__(kBwdThreads, 2) qk_norm_rope_backward_kernel(
    const HeadArgs a, int lanes, SideSplit split, FastDiv by_seq, FastDiv by_q_chunks, FastDiv by_k_chunks,
    float* __restrict__ partials, uint32_t* err) {
  using V = HeadVec<T, E>;
  extern __shared__ __align__(16) uint8_t smem[];
  griddep_launch_dependents();
  griddep_wait();
  const bool is_q = blockIdx.x < static_cast<unsigned>(split.q_ctas);
  const HeadSide& side = is_q ? a.q : a.k;
  const uint32_t cta = is_q ? blockIdx.x : blockIdx.x - split.q_ctas;
  const uint32_t per_warp = 32 / lanes;
  const uint32_t groups = static_cast<uint32_t>(is_q ? split.q_ctas : split.k_ctas) * kBwdWarps * per_warp;
  const LaneGroup group(lanes);
  const int D = a.head_dim, heads = side.heads;
  const LaneCols col = lane_cols<PAIRS>(group.p, lanes, D / E, a.rotary_dim / E);
  const int column = max(0, col.va) * E;
  const TokenTable<E, PAIRS, AXES> table(a.t, col);

  HeadStream<T, E, NH, STAGES, 2, FULL> st;
  st.in[0] = {static_cast<const T*>(side.x) + column, side.stride_batch, side.stride_seq, side.stride_head};
  st.in[1] = {static_cast<const T*>(side.dy) + column, side.dy_stride_batch, side.dy_stride_seq, side.dy_stride_head};
  st.vb_offset = col.vb * E - column;
  st.has_a = col.va >= 0 && !group.spare;
  st.has_b = col.vb >= 0 && !group.spare;
  st.by_seq = by_seq;
  st.by_chunks = is_q ? by_q_chunks : by_k_chunks;
  st.seq = static_cast<uint32_t>(a.seq);
  st.chunks = (heads + NH - 1) / NH;
  st.units = static_cast<uint32_t>(a.batch * a.seq) * st.chunks;
  st.heads = heads;
  // the warp's groups walk in step: the first one's unit decides the end
  uint32_t lead = (cta * kBwdWarps + (threadIdx.x >> 5)) * per_warp;
  st.start(smem, lead + group.group, groups);

  F2 wa[E / 2], wb[E / 2], acc_a[E / 2], acc_b[E / 2];
  {
    float fa[E], fb[E];
#pragma unroll
    for (int j = 0; j < E; ++j) fa[j] = fb[j] = 1.f;
    if (side.weight != nullptr) {
      if (col.va >= 0) load_floats<E>(side.weight, col.va * E, side.w_dtype, fa);
      if (col.vb >= 0) load_floats<E>(side.weight, col.vb * E, side.w_dtype, fb);
    }
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      wa[j] = f2(fa[2 * j], fa[2 * j + 1]);
      wb[j] = f2(fb[2 * j], fb[2 * j + 1]);
      acc_a[j] = acc_b[j] = f2(0.f, 0.f);
    }
  }
  const float inv_d = 1.f / static_cast<float>(D);
  const int most = min(NH, heads);
  int stage = 0;
  for (; lead < st.units; lead += groups) {
    const uint32_t unit = min(lead + group.group, st.units - 1);
    const uint32_t token = st.by_chunks.div(unit);
    const int h0 = static_cast<int>(unit - token * st.chunks) * NH;
    const int mine = lead + group.group < st.units ? heads - h0 : 0;  // heads of this unit
    const uint32_t b = by_seq.div(token);
    PlainRotation<E, PAIRS> rot;  // the inverse rotation
    {
      float c[E], s[E];
      table.load(a.t, b, token - b * st.seq, col, true, group.p == 0, err, c, s);
      rot.set(c, s);
    }
    T* out = static_cast<T*>(side.out) + (static_cast<int64_t>(token) * heads + h0) * D + column;
    st.wait();
    // Heads of full warps one at a time. In the others lane groups mostly sum by a
    // shuffle for each lane (LaneGroup::sum): there the sums of all heads go side by side and
    // the heads are read again after them (12 + 3 heads of 80 columns, f16, 32768
    // tokens 69.0 -> 62.6 us; heads of 128 no faster).
    constexpr int AT_ONCE = FULL ? 1 : NH;
#pragma unroll
    for (int i0 = 0; i0 < NH; i0 += AT_ONCE) {
      if (i0 >= most) break;
      F2 ua[E / 2], ub[E / 2], fa[E / 2], fb[E / 2], ta[E / 2], tb[E / 2];
      auto read = [&](int i) {  // a head, with its sums
        V::unpack(*st.slot(stage, 0, i, 0), ua);
        V::unpack(*st.slot(stage, 0, i, 1), ub);
        V::unpack(*st.slot(stage, 1, i, 0), fa);
        V::unpack(*st.slot(stage, 1, i, 1), fb);
        rot.apply(fa, fb, col);
        F2 ss = f2(0.f, 0.f), dot = ss;
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          ss = fma2(ub[j], ub[j], fma2(ua[j], ua[j], ss));
          ta[j] = mul2(fa[j], ua[j]);
          tb[j] = mul2(fb[j], ub[j]);
          dot = fma2(tb[j], wb[j], fma2(ta[j], wa[j], dot));
        }
        return make_float2(ss.x + ss.y, dot.x + dot.y);
      };
      float sums[2 * AT_ONCE];  // of squares, and of b w x, of each head
#pragma unroll
      for (int n = 0; n < AT_ONCE; ++n) {
        const float2 both = read(i0 + n);
        sums[2 * n] = both.x;
        sums[2 * n + 1] = both.y;
      }
      group.sum(sums);
      if constexpr (AT_ONCE > 1) asm volatile("" ::: "memory");  // registers are not kept over the sums
#pragma unroll
      for (int n = 0; n < AT_ONCE; ++n) {
        const int i = i0 + n;
        if constexpr (AT_ONCE > 1) read(i);
        const float r = rsqrtf(sums[2 * n] * inv_d + a.eps);
        const float k = sums[2 * n + 1] * inv_d * r * r * r;  // in this order: r^3 alone can overflow
        if (i < mine) {
          const F2 r2 = f2(r, r), k2 = f2(-k, -k);
#pragma unroll
          for (int j = 0; j < E / 2; ++j) {
            acc_a[j] = fma2(ta[j], r2, acc_a[j]);
            acc_b[j] = fma2(tb[j], r2, acc_b[j]);
            fa[j] = fma2(mul2(fa[j], wa[j]), r2, mul2(ua[j], k2));
            fb[j] = fma2(mul2(fb[j], wb[j]), r2, mul2(ub[j], k2));
          }
          if (FULL || st.has_a) V::store(out + i * D, fa);
          if (FULL || st.has_b) V::store(out + i * D + st.vb_offset, fb);
        }
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    st.load();  // into the stage that the unit before this one has left
  }
  if (side.dweight == nullptr) return;
  // the warp's groups, then the CTA's warps (the ring is done with: no load is in flight past the last unit)
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < E / 2; ++j) {
    const F2 own_a = acc_a[j], own_b = acc_b[j];
    for (uint32_t g = 1; g < per_warp; ++g) {
      const int from = min(31, lane + static_cast<int>(g) * lanes);
      acc_a[j].x += __shfl_sync(0xffffffffu, own_a.x, from);
      acc_a[j].y += __shfl_sync(0xffffffffu, own_a.y, from);
      acc_b[j].x += __shfl_sync(0xffffffffu, own_b.x, from);
      acc_b[j].y += __shfl_sync(0xffffffffu, own_b.y, from);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);  // [warps][head_dim]
  float* mine = red + (threadIdx.x >> 5) * D;
  if (lane < lanes) {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      if (col.va >= 0) {
        mine[col.va * E + 2 * j] = acc_a[j].x;
        mine[col.va * E + 2 * j + 1] = acc_a[j].y;
      }
      if (col.vb >= 0) {
        mine[col.vb * E + 2 * j] = acc_b[j].x;
        mine[col.vb * E + 2 * j + 1] = acc_b[j].y;
      }
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
template <typename T, bool AXES>
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
    int64_t pos = AXES ? 0 : token_position(a.t, b, sq, err, lane == 0);
    auto weight = [&](int i) { return side.weight != nullptr ? load_as_float(side.weight, i, side.w_dtype) : 1.f; };
    // calls f(column, b) for each of this lane's columns
    auto each = [&](auto f) {
      for (int i = lane; i < half; i += 32) {
        float c, s;
        if constexpr (AXES) pos = axis_position(a.t, b, sq, LaneAxes::of(a.t, i), err);
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
static __global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const HeadArgs a, SideSplit split,
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
// One wave of resident CTAs (at most kBwdCtasPerSm on an SM), shared between
// the sides by their units of work, at most one CTA for `per_cta` units.
SideSplit split_ctas(const void* kernel, size_t smem, int64_t q_units, int64_t k_units, int64_t per_cta) {
  const int64_t all =
      static_cast<int64_t>(num_sms()) * std::min(kBwdCtasPerSm, cached_occupancy(kernel, kBwdThreads, smem));
  auto share = [&](int64_t u) {
    if (u == 0) return 0;
    const double part = static_cast<double>(u) / static_cast<double>(q_units + k_units);
    return static_cast<int>(std::min((u + per_cta - 1) / per_cta, std::max<int64_t>(1, static_cast<int64_t>(all * part))));
  };
  return SideSplit{share(q_units), share(k_units)};
}

template <typename T, int E, bool PAIRS, bool AXES>
cudaError_t launch_vec(const HeadArgs& a, SideSplit* split, float* partials, cudaStream_t st) {
  // 16-byte slots: 3 heads x 2 tensors x 2 stages = 96 KB a CTA, two CTAs an SM.
  // Measured, us at 8192 / 32768 tokens of 32 + 8 heads of 128 columns, bf16:
  // 3 heads, 2 stages 53 / 183; 2 heads, 3 stages 59 / 215; 1 head, 5 stages
  // 71 / 255; 4 heads, 2 stages (one CTA of 416 threads) 65 / 232.
  constexpr int NH = 3, STAGES = 2;
  const int lanes = (a.head_dim / E + 1) / 2;
  const bool full = a.head_dim == 2 * E * lanes && 32 % lanes == 0;
  auto* kernel = full ? qk_norm_rope_backward_kernel<T, E, PAIRS, NH, STAGES, true, AXES>
                      : qk_norm_rope_backward_kernel<T, E, PAIRS, NH, STAGES, false, AXES>;
  constexpr size_t smem = HeadStream<T, E, NH, STAGES, 2, true>::kSmemBytes;
  static_assert(smem >= sizeof(float) * kBwdWarps * 64 * E, "the weight sums fit into the ring");
  const void* fn = reinterpret_cast<const void*>(kernel);
  if (const cudaError_t e = ensure_smem_attr(fn, smem); e != cudaSuccess) return e;
  const uint32_t qc = (a.q.heads + NH - 1) / NH, kc = (a.k.heads + NH - 1) / NH;
  const int64_t tokens = a.batch * a.seq;
  *split = split_ctas(fn, smem, tokens * qc, tokens * kc, kBwdWarps * (32 / lanes));
  note_launch();
  return launch_gemm_grid(kernel, kBwdThreads, split->q_ctas + split->k_ctas, 1, smem, st, a, lanes, *split,
                          FastDiv::make(static_cast<uint32_t>(a.seq)), FastDiv::make(std::max(1u, qc)),
                          FastDiv::make(std::max(1u, kc)), partials, error_word_ptr());
}

template <typename T, bool AXES>
cudaError_t launch_type(const HeadArgs& a, SideSplit* split, float* partials, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const int e = head_vector_elems(a, true);
  if (e == E)
    return a.pairs ? launch_vec<T, E, true, AXES>(a, split, partials, st) : launch_vec<T, E, false, AXES>(a, split, partials, st);
  if (e == E / 2)
    return a.pairs ? launch_vec<T, E / 2, true, AXES>(a, split, partials, st)
                   : launch_vec<T, E / 2, false, AXES>(a, split, partials, st);
  auto* kernel = qk_norm_rope_backward_any_kernel<T, AXES>;
  const size_t smem = sizeof(float) * kBwdWarps * a.head_dim;
  const int64_t tokens = a.batch * a.seq;
  *split = split_ctas(reinterpret_cast<const void*>(kernel), smem, tokens * a.q.heads, tokens * a.k.heads, kBwdWarps);
  note_launch();
  return launch_gemm_grid(kernel, kBwdThreads, split->q_ctas + split->k_ctas, 1, smem, st, a, *split, partials,
                          error_word_ptr());
}

template <bool AXES>
cudaError_t launch_backward(const HeadArgs& a, void* ws, cudaStream_t st) {
  SideSplit split{};
  float* partials = static_cast<float*>(ws);
  cudaError_t e = a.dtype == F16    ? launch_type<__half, AXES>(a, &split, partials, st)
                  : a.dtype == BF16 ? launch_type<__nv_bfloat16, AXES>(a, &split, partials, st)
                                    : launch_type<float, AXES>(a, &split, partials, st);
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
}  // namespace

}  // namespace tfo
