// A block's branch added to the residual stream, and the norm before the next
// block, in one pass:
//
//   u = x / sqrt(mean(x^2) + eps) * w1        (or x itself)
//   h = residual + scale * gate * dropout(u)
//   y = h / sqrt(mean(h^2) + eps) * w2 + shift
//
// w1, gate, w2 and shift are rows of `hidden` columns, one for all rows or one
// for each sequence. Everything is held in fp32 from the loads to one rounding
// of h and one of y; y is made of the h that was not rounded.
//
// Floor: HBM (x and residual read once, h and y written once; parameters come
// from L2). A group of threads keeps its columns of a row in registers over
// both sums, which depend on one another, and streams the next rows meanwhile
// (residual.cuh). w1, gate, scale and 1 / (1 - p) are one coefficient.
#include "residual.cuh"

namespace tfo {

// scale * gate * w1 (* 1 / (1 - p)) of a sequence: what a normed branch is multiplied by.
template <int E, int V>
__device__ __forceinline__ void branch_coefficient(const ResidualArgs& a, const RowCols<E, V>& cols, int64_t seq,
                                                   F2 (&c)[RowCols<E, V>::P]) {
  constexpr int P = RowCols<E, V>::P;
  F2 g[P];
  cols.param(a.branch_weight, seq, 1.f, c);
  cols.param(a.gate, seq, 1.f, g);
  const float s = a.dropped ? a.scale * a.drop.scale : a.scale;
#pragma unroll
  for (int j = 0; j < P; ++j) c[j] = mul2(mul2(c[j], g[j]), f2(s, s));
}

// Parameters stay in registers up to this many columns a thread; above it they are read again for every row.
constexpr int kParamCols = 16;

template <typename TX, typename TR, int E, int V, int STAGES>
__global__ void __launch_bounds__(kRowThreads, 1)
    residual_norm_kernel(const __grid_constant__ ResidualArgs a, RowPlan plan) {
  using Cols = RowCols<E, V>;
  constexpr int P = Cols::P;
  constexpr bool KEEP_PARAMS = Cols::N <= kParamCols;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[2][kMaxRowWarps][kMaxRowWarps];
  griddep_launch_dependents();
  const int warps = plan.threads / 32;
  const int group = (threadIdx.x >> 5) / warps, warp = (threadIdx.x >> 5) - group * warps;
  const int t = threadIdx.x - group * plan.threads;
  for (int i = threadIdx.x; i < 2 * kMaxRowWarps * kMaxRowWarps; i += blockDim.x) (&red[0][0][0])[i] = 0.f;
  __syncthreads();
  griddep_wait();
  const int64_t groups = static_cast<int64_t>(gridDim.x) * plan.groups;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * plan.groups + group;
  const int64_t r0 = me * a.rows / groups, r1 = (me + 1) * a.rows / groups;
  if (r0 >= r1) return;
  const Cols cols(t, plan.threads, a.hidden);
  RowStream<TX, TR, E, V, 1, 1, STAGES> rows;
  rows.base[0] = a.x;
  rows.stride[0] = a.x_stride;
  rows.base[1] = a.res;
  rows.stride[1] = a.res_stride;
  rows.start(cols, smem, r0, r1);
  const DropKey key(a.drop);
  const float inv_h = 1.f / static_cast<float>(a.hidden);
  const int bar = 1 + group;
  int turn = 0;  // of the parts of a sum
  int64_t seq = r0 / a.rows_per_seq, seq_end = (seq + 1) * a.rows_per_seq;
  const bool by_seq = (a.branch_weight.seq_stride | a.gate.seq_stride | a.weight.seq_stride) != 0;
  F2 c[P], w[P];
  if constexpr (KEEP_PARAMS) {
    branch_coefficient(a, cols, seq, c);
    cols.param(a.weight, seq, 1.f, w);
  }
  for (int64_t r = r0; r < r1; ++r) {
    if (r == seq_end) {
      ++seq;
      seq_end += a.rows_per_seq;
      if (KEEP_PARAMS && by_seq) {
        branch_coefficient(a, cols, seq, c);
        cols.param(a.weight, seq, 1.f, w);
      }
    }
    const uint32_t bits = a.dropped ? cols.kept(a.drop, key, r) : ~0u;
    rows.advance(cols);
    F2 h[P];
    float r_branch = 1.f;
    {
      F2 x[P], res[P];
      rows.template get<0>(x);
      rows.template get<1>(res);
      if (a.branch_norm) {
        F2 s2 = f2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < P; ++j) s2 = fma2(x[j], x[j], s2);
        float s[1] = {s2.x + s2.y};
        row_sum(s, red[turn ^= 1][group], warps, warp, bar);
        r_branch = rsqrtf(s[0] * inv_h + a.eps);
      }
      if constexpr (!KEEP_PARAMS) branch_coefficient(a, cols, seq, c);
#pragma unroll
      for (int j = 0; j < P; ++j) x[j] = mul2(mul2(x[j], f2(r_branch, r_branch)), c[j]);
      if (a.dropped) Cols::drop(bits, x);
#pragma unroll
      for (int j = 0; j < P; ++j) h[j] = add2(res[j], x[j]);
    }
    cols.store(static_cast<TR*>(a.h) + r * a.hidden, h);
    float r_sum = 1.f;
    if (a.y != nullptr) {
      F2 s2 = f2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < P; ++j) s2 = fma2(h[j], h[j], s2);
      float s[1] = {s2.x + s2.y};
      row_sum(s, red[turn ^= 1][group], warps, warp, bar);
      r_sum = rsqrtf(s[0] * inv_h + a.eps);
      if constexpr (!KEEP_PARAMS) cols.param(a.weight, seq, 1.f, w);
#pragma unroll
      for (int j = 0; j < P; ++j) h[j] = mul2(mul2(h[j], f2(r_sum, r_sum)), w[j]);
      if (a.shift.p != nullptr) {
        F2 b[P];
        cols.param(a.shift, seq, 0.f, b);
#pragma unroll
        for (int j = 0; j < P; ++j) h[j] = add2(h[j], b[j]);
      }
      cols.store(static_cast<TX*>(a.y) + r * a.hidden, h);
    }
    if (a.rstd != nullptr && t == 0) *reinterpret_cast<float2*>(a.rstd + 2 * r) = make_float2(r_branch, r_sum);
  }
}

// Rows of any width: a CTA for each, which reads it again for the second sum and for the results (from L1 and L2).
template <typename TX, typename TR>
__global__ void __launch_bounds__(kRowThreads) residual_norm_any_kernel(const __grid_constant__ ResidualArgs a) {
  __shared__ __align__(16) float red[2][kMaxRowWarps];
  griddep_launch_dependents();
  griddep_wait();
  const DropKey key(a.drop);
  const float s_branch = a.dropped ? a.scale * a.drop.scale : a.scale;
  const float inv_h = 1.f / static_cast<float>(a.hidden);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int64_t seq = r / a.rows_per_seq;
    const TX* x = static_cast<const TX*>(a.x) + r * a.x_stride;
    const TR* res = static_cast<const TR*>(a.res) + r * a.res_stride;
    auto param = [&](const RowParam& p, int i, float otherwise) {
      return p.p != nullptr ? load_as_float(p.p, seq * p.seq_stride + i, p.dtype) : otherwise;
    };
    float r_branch = 1.f, r_sum = 1.f;
    if (a.branch_norm) {
      float s[1] = {0.f};
      for (int i = threadIdx.x; i < a.hidden; i += kRowThreads) {
        const float v = Ty<TX>::to_f(x[i]);
        s[0] = fmaf(v, v, s[0]);
      }
      row_sum(s, red[0], kMaxRowWarps, threadIdx.x >> 5, 1);
      r_branch = rsqrtf(s[0] * inv_h + a.eps);
    }
    auto sum = [&](int i) {
      const float u = Ty<TX>::to_f(x[i]) * r_branch * (param(a.branch_weight, i, 1.f) * param(a.gate, i, 1.f) * s_branch);
      const bool keep = !a.dropped || (!a.drop.all && key.kept<1>(static_cast<uint64_t>(r * a.hidden + i)));
      return Ty<TR>::to_f(res[i]) + (keep ? u : 0.f);
    };
    if (a.y != nullptr) {
      float s[1] = {0.f};
      for (int i = threadIdx.x; i < a.hidden; i += kRowThreads) {
        const float v = sum(i);
        s[0] = fmaf(v, v, s[0]);
      }
      row_sum(s, red[1], kMaxRowWarps, threadIdx.x >> 5, 1);
      r_sum = rsqrtf(s[0] * inv_h + a.eps);
    }
    for (int i = threadIdx.x; i < a.hidden; i += kRowThreads) {
      const float v = sum(i);
      static_cast<TR*>(a.h)[r * a.hidden + i] = Ty<TR>::from_f(v);
      if (a.y != nullptr)
        static_cast<TX*>(a.y)[r * a.hidden + i] = Ty<TX>::from_f(v * r_sum * param(a.weight, i, 1.f) + param(a.shift, i, 0.f));
    }
    if (a.rstd != nullptr && threadIdx.x == 0) *reinterpret_cast<float2*>(a.rstd + 2 * r) = make_float2(r_branch, r_sum);
    __syncthreads();  // the next row's sums use the same parts
  }
}

namespace {
template <typename TX, typename TR, int E, int V>
cudaError_t launch_rows(const ResidualArgs& a, int threads, cudaStream_t st) {
  constexpr int STAGES = row_stages<TX, TR>(E * V, 1, 1);
  auto* kernel = residual_norm_kernel<TX, TR, E, V, STAGES>;
  using Stream = RowStream<TX, TR, E, V, 1, 1, STAGES>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  // as many groups a CTA as still leave every SM a row
  const int groups =
      static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kRowThreads / threads, a.rows / num_sms())));
  const int block = groups * threads;
  const size_t smem = Stream::smem_bytes(block);
  // the limit of the largest block: also below it the static part comes on top
  if (const cudaError_t e = ensure_smem_attr(fn, Stream::smem_bytes(kRowThreads)); e != cudaSuccess) return e;
  const int64_t all = static_cast<int64_t>(num_sms()) * std::max(1, cached_occupancy(fn, block, smem));
  const int64_t grid = std::min<int64_t>(all, (a.rows + groups - 1) / groups);
  note_launch();
  return launch_gemm_grid(kernel, block, static_cast<int>(grid), 1, smem, st, a, RowPlan{threads, groups});
}

template <typename TX, typename TR>
cudaError_t launch_types(const ResidualArgs& a, cudaStream_t st) {
  constexpr int E = kRowChunk<TX, TR>;
  if (row_chunk(a, false) == E) {
    // A warp a row as far as 16 columns a thread carry it, then 16 columns a thread.
    constexpr int FULL = 16 / E;
    if (a.hidden <= 32 * E) return launch_rows<TX, TR, E, 1>(a, 32, st);
    if (FULL > 2 && a.hidden <= 64 * E) return launch_rows<TX, TR, E, 2>(a, 32, st);
    if (const int t = row_threads(a.hidden, E, FULL)) return launch_rows<TX, TR, E, FULL>(a, t, st);
    if (const int t = row_threads(a.hidden, E, 2 * FULL)) return launch_rows<TX, TR, E, 2 * FULL>(a, t, st);
  } else {
    if (const int t = row_threads(a.hidden, 1, 4)) return launch_rows<TX, TR, 1, 4>(a, t, st);
    if (const int t = row_threads(a.hidden, 1, 8)) return launch_rows<TX, TR, 1, 8>(a, t, st);
  }
  note_launch();
  return launch_dependent(residual_norm_any_kernel<TX, TR>, static_cast<int>(std::min<int64_t>(a.rows, num_sms() * 4ll)),
                          kRowThreads, st, a);
}
}  // namespace

cudaError_t residual_norm_launch(const ResidualArgs& a, cudaStream_t st) {
  if (a.x_dtype == F16)
    return a.res_dtype == F32 ? launch_types<__half, float>(a, st) : launch_types<__half, __half>(a, st);
  if (a.x_dtype == BF16)
    return a.res_dtype == F32 ? launch_types<__nv_bfloat16, float>(a, st)
                              : launch_types<__nv_bfloat16, __nv_bfloat16>(a, st);
  return launch_types<float, float>(a, st);
}

}  // namespace tfo
