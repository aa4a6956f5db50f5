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
//
// Measured, of the copy rate: bf16 65536 x 4096 331 us (99 %), 8192 x 8192 87
// (93 %), 8192 x 4096 46 (88 %, its start and end weigh); with an fp32 stream 68
// (89 %); with dropout 70 (58 %: a row's mask is made between two rows' sums; no unit
// is full, issue slots 53 % at 16 warps an SM).
#include "residual.cuh"

namespace tfo {

// Parameters stay in registers up to this many columns a thread; above it they are read again for every row.
constexpr int kParamCols = 16;

template <typename TX, typename TR, int E, int V, bool SHIFTED, int STAGES>
__global__ void __launch_bounds__(kRowThreads, 1)
    residual_norm_kernel(const __grid_constant__ ResidualArgs a, const __grid_constant__ RowPlan plan) {
  using Cols = RowCols<E, V, SHIFTED>;
  constexpr int NB = Cols::BLOCKS, BP = Cols::BP;
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
  const uint32_t me = blockIdx.x * plan.groups + group;
  const uint32_t by = plan.stride != 0 ? plan.stride : 1u;
  uint32_t row = plan.stride != 0 ? me : plan.share.first(me);
  const uint32_t end = plan.stride != 0 ? static_cast<uint32_t>(a.rows) : plan.share.first(me + 1);
  if (row >= end) return;
  const Cols cols(t, plan.threads, a.hidden);
  RowStream<TX, TR, E, V, SHIFTED, 1, 1, STAGES> rows;
  rows.start(cols, plan, smem, row, end, by);
  const DropKey key(a.drop);
  const float inv_h = 1.f / static_cast<float>(a.hidden);
  const int bar = 1 + group;
  int turn = 0;  // of the parts of a sum
  const uint32_t per = static_cast<uint32_t>(a.rows_per_seq);
  uint32_t seq = row / per, seq_end = (seq + 1) * per;
  const bool by_seq = (a.branch_weight.seq_stride | a.gate.seq_stride | a.weight.seq_stride) != 0;
  F2 c[KEEP_PARAMS ? NB : 1][BP], w[KEEP_PARAMS ? NB : 1][BP];
  auto params = [&] {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      cols.branch_coefficient(a, seq, b, c[b]);
      cols.param(a.weight, seq, 1.f, b, w[b]);
    }
  };
  if constexpr (KEEP_PARAMS) params();
  for (;;) {
    const uint64_t element = static_cast<uint64_t>(row) * static_cast<uint32_t>(a.hidden);  // the row's first
    const uint32_t bits = a.dropped ? cols.kept(a.drop, key, element) : ~0u;
    rows.advance(cols, plan);
    F2 h[NB][BP];
    float r_branch = 1.f;
    if (a.branch_norm) {
      F2 s2 = f2(0.f, 0.f);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        rows.template get<0>(cols, plan, row, b, h[b]);
#pragma unroll
        for (int j = 0; j < BP; ++j) s2 = fma2(h[b][j], h[b][j], s2);
      }
      float s[1] = {s2.x + s2.y};
      row_sum(s, red[turn ^= 1][group], warps, warp, bar);
      r_branch = rsqrtf(s[0] * inv_h + a.eps);
    }
    F2 s2 = f2(0.f, 0.f);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      F2 res[BP];
      if (!a.branch_norm) rows.template get<0>(cols, plan, row, b, h[b]);
      rows.template get<1>(cols, plan, row, b, res);
      F2(&cb)[BP] = c[KEEP_PARAMS ? b : 0];
      if constexpr (!KEEP_PARAMS) cols.branch_coefficient(a, seq, b, cb);
#pragma unroll
      for (int j = 0; j < BP; ++j) h[b][j] = mul2(mul2(h[b][j], f2(r_branch, r_branch)), cb[j]);
      if (a.dropped) Cols::drop(bits, b, h[b]);
#pragma unroll
      for (int j = 0; j < BP; ++j) {
        h[b][j] = add2(res[j], h[b][j]);
        s2 = fma2(h[b][j], h[b][j], s2);
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) cols.store(static_cast<TR*>(a.h) + element, b, h[b]);
    float r_sum = 1.f;
    if (a.y != nullptr) {
      float s[1] = {s2.x + s2.y};
      row_sum(s, red[turn ^= 1][group], warps, warp, bar);
      r_sum = rsqrtf(s[0] * inv_h + a.eps);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        F2(&wb)[BP] = w[KEEP_PARAMS ? b : 0];
        if constexpr (!KEEP_PARAMS) cols.param(a.weight, seq, 1.f, b, wb);
#pragma unroll
        for (int j = 0; j < BP; ++j) h[b][j] = mul2(mul2(h[b][j], f2(r_sum, r_sum)), wb[j]);
        if (a.shift.p != nullptr) {
          F2 sh[BP];
          cols.param(a.shift, seq, 0.f, b, sh);
#pragma unroll
          for (int j = 0; j < BP; ++j) h[b][j] = add2(h[b][j], sh[j]);
        }
        cols.store(static_cast<TX*>(a.y) + element, b, h[b]);
      }
    }
    if (a.rstd != nullptr && t == 0) reinterpret_cast<float2*>(a.rstd)[row] = make_float2(r_branch, r_sum);
    row += by;
    if (row >= end) return;
    if (row == seq_end) {  // (runs: with a stride no parameter differs between sequences)
      ++seq;
      seq_end += per;
      if (KEEP_PARAMS && by_seq) params();
    }
  }
}

// Rows of any width: a CTA for each, which reads it again for the second sum and for the results (from L1 and L2).
// 4096 x 8196 bf16 with an fp32 stream 135 us (45 % of the copy rate): loads of one column, none ahead.
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
template <typename TX, typename TR, int V, bool SHIFTED, int STAGES>
cudaError_t launch_groups(const ResidualArgs& a, RowPlan plan, int threads, int groups, cudaStream_t st) {
  constexpr int E = kRowChunk<TX, TR>;
  auto* kernel = residual_norm_kernel<TX, TR, E, V, SHIFTED, STAGES>;
  using Stream = RowStream<TX, TR, E, V, SHIFTED, 1, 1, STAGES>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  const int block = groups * threads;
  const size_t smem = Stream::kSmemBytes;
  // at least a little over 48 KB: the sums' static part comes on top
  if (const cudaError_t e = ensure_smem_attr(fn, std::max<size_t>(smem, 49 * 1024)); e != cudaSuccess) return e;
  const int64_t all = static_cast<int64_t>(num_sms()) * std::max(1, cached_occupancy(fn, block, smem));
  const int64_t grid = std::min<int64_t>(all, (a.rows + groups - 1) / groups);
  plan.threads = threads;
  plan.groups = groups;
  plan.share = Split::make(a.rows, grid * groups);
  const bool by_seq = (a.branch_weight.seq_stride | a.gate.seq_stride | a.weight.seq_stride | a.shift.seq_stride) != 0;
  plan.stride = by_seq ? 0 : static_cast<uint32_t>(grid * groups);
  note_launch();
  return launch_gemm_grid(kernel, block, static_cast<int>(grid), 1, smem, st, a, plan);
}

template <typename TX, typename TR, int V, bool SHIFTED>
cudaError_t launch_rows(const ResidualArgs& a, const RowPlan& plan, int threads, cudaStream_t st) {
  constexpr int COLS = kRowChunk<TX, TR> * V, MOST = row_stages<TX, TR>(COLS, 1, 1, SHIFTED);
  // as many groups a CTA as still leave every SM a row
  const int groups =
      static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kRowThreads / threads, a.rows / num_sms())));
  // One row ahead is enough where a CTA's groups wait for different rows, and reads and writes lie closer together in
  // memory than with two or three: bf16 65536 x 4096 356 -> 331 us, 65536 x 2048 186 -> 165, with an fp32 stream
  // 16384 x 4096 137 -> 130. A group alone needs more (8192 x 8192 93 us, with two ahead 87), and the first rows come
  // faster with more, which tells where a group has few of them (bf16 8192 x 4096 47 us, with three ahead 46; one row
  // ahead is only 32 KB an SM there, and 48 or 64 with a type of 32 bits).
  if constexpr (!SHIFTED && COLS == 16 && MOST > 2) {
    const int64_t many = sizeof(TX) + sizeof(TR) > 4 ? 24 : 96;
    if (groups > 2 || (groups == 2 && a.rows / (num_sms() * groups) >= many))
      return launch_groups<TX, TR, V, SHIFTED, 2>(a, plan, threads, groups, st);
  }
  return launch_groups<TX, TR, V, SHIFTED, MOST>(a, plan, threads, groups, st);
}

// A warp a row as far as 16 columns a thread carry it, then 16 columns a thread, then (aligned rows) 32.
template <typename TX, typename TR, bool SHIFTED>
cudaError_t launch_width(const ResidualArgs& a, const RowPlan& plan, cudaStream_t st, bool* done) {
  constexpr int E = kRowChunk<TX, TR>, FULL = 16 / E;
  *done = true;
  if (a.hidden <= 32 * E) return launch_rows<TX, TR, 1, SHIFTED>(a, plan, 32, st);
  if (FULL > 2 && a.hidden <= 64 * E) return launch_rows<TX, TR, 2, SHIFTED>(a, plan, 32, st);
  if (const int t = row_threads(a.hidden, E, FULL)) return launch_rows<TX, TR, FULL, SHIFTED>(a, plan, t, st);
  if constexpr (!SHIFTED) {
    if (const int t = row_threads(a.hidden, E, 2 * FULL)) return launch_rows<TX, TR, 2 * FULL, SHIFTED>(a, plan, t, st);
  }
  *done = false;
  return cudaSuccess;
}

template <typename TX, typename TR>
cudaError_t launch_types(const ResidualArgs& a, cudaStream_t st) {
  RowPlan plan{};
  if (set_tensors(&plan, {{a.x, a.x_stride * static_cast<int64_t>(sizeof(TX))}, {a.res, a.res_stride * static_cast<int64_t>(sizeof(TR))}})) {
    bool done = false;
    const cudaError_t e = rows_aligned(a, false) ? launch_width<TX, TR, false>(a, plan, st, &done)
                                                 : launch_width<TX, TR, true>(a, plan, st, &done);
    if (done) return e;
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
