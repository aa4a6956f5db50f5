// Gradients of the residual stream with its norms (residual_norm.cu). With
// c = scale * gate * w1 / (1 - p), k the kept elements, r1 and r2 the saved
// 1 / sqrt(mean + eps), x' = x r1, u = k c x', h = residual + u, h' = h r2 and
// g = dy w2:
//
//   dH        = dh + r2 (g - h' mean(g h'))
//   dresidual = dH
//   dx        = r1 (k c dH - x' mean(u dH)),  or k c dH where the branch is not normed
//   dw2       = sum over rows of dy h',   dshift = sum of dy
//   A         = sum over rows of k dH x' / (1 - p):
//   dgate     = scale w1 A,   dw1 = scale gate A   (summed over sequences where one is not)
//
// The second mean needs dH, which needs the first; written out,
//   sum(u dH) = sum(u dh) + r2 (sum(u g) - mean(g h') sum(u h')),
// so that one pass over a row and one exchange between its threads give both.
// h is made again from x and residual: nothing but r1 and r2 is stored.
//
// Threads keep fp32 sums of A, dy h' and dy for their columns over the rows of
// an item (a run of rows of one sequence, a fixed split) and write them out as
// partial rows; a second kernel adds these in order, in fp64, with the other
// parameter's factor. No atomics: the results do not depend on scheduling.
//
// Floor: HBM (x, residual, dy and dh read, dx and dresidual written).
// Measured, of the copy rate, with the second kernel (4 us): bf16 32768 x 4096 266
// us (92 %), 8192 x 4096 83 (74 %: the start with its parameters, the end with its
// sums), 8192 x 8192 150 (82 %), fp32 4096 x 4096 69 (88 %), with dropout 8192 x
// 4096 bf16 103 (60 %).
#include "residual.cuh"

namespace tfo {

// Sums over rows that the parameters' gradients are made of.
enum RowSum : int { SUM_BRANCH = 0, SUM_WEIGHT = 1, SUM_SHIFT = 2, SUMS = 3 };

// The split of the rows into items: `chunks` runs for each of `seqs` sequences (one of all rows where no parameter is
// a sequence's own).
struct RowItems {
  int64_t seqs, seq_rows, chunks;
  Split runs;  // a sequence's rows over its items
  __host__ __device__ int64_t count() const { return seqs * chunks; }
  __device__ uint32_t first_row(uint32_t item) const {
    const uint32_t b = item / static_cast<uint32_t>(chunks), c = item - b * static_cast<uint32_t>(chunks);
    return b * static_cast<uint32_t>(seq_rows) + runs.first(c);
  }
};

// What a thread keeps from row to row, in blocks of its columns: the sums over
// rows, c and w2. With 16 columns these are 80 values, which live in tensor
// memory: a block of 8 is read or written by one instruction, and the registers
// are free for the row. Warp w of the CTA uses the lanes of its sub-partition
// (w % 4) and columns of its own. With 8 columns or less they are registers.
// These instructions take a warp whose lanes are together; what stands before them
// parts the lanes where a row ends inside the warp (its copies, the columns past its
// end, its stores). Each of them therefore joins the lanes first.
enum Kept : int { KEPT_C = SUMS, KEPT_W = SUMS + 1, KEPT = SUMS + 2 };
template <class Cols, bool TENSOR> struct RowKept {
  F2 v[KEPT][Cols::BLOCKS][Cols::BP];
  __device__ explicit RowKept(uint32_t) {}
  __device__ void settle() {}
  __device__ void read(int i, int b, F2 (&out)[Cols::BP]) const {
#pragma unroll
    for (int j = 0; j < Cols::BP; ++j) out[j] = v[i][b][j];
  }
  __device__ void wait() {}
  __device__ void arrived(F2 (&)[Cols::BP]) const {}
  __device__ void write(int i, int b, const F2 (&in)[Cols::BP]) {
#pragma unroll
    for (int j = 0; j < Cols::BP; ++j) v[i][b][j] = in[j];
  }
};
template <class Cols> struct RowKept<Cols, true> {
  static_assert(Cols::N == 16 && Cols::B == 8, "two blocks of 8 columns");
  static constexpr uint32_t kColumns = 512;  // of the CTA: KEPT * 16 for each of a sub-partition's four warps, a power of two
  uint32_t mine;
  __device__ explicit RowKept(uint32_t base) {
    const uint32_t w = threadIdx.x >> 5;
    mine = base + ((w & 3u) << 21) + (w >> 2) * (KEPT * 16);  // lane 32 * (w % 4) in the upper half
  }
  // Between a write and a read of the same values.
  __device__ void settle() {
    __syncwarp();
    tmem_st_wait();
  }
  // Asks for a block; it is there after wait() and arrived() of it.
  __device__ void read(int i, int b, F2 (&out)[4]) const {
    __syncwarp();
    tmem_ld8(mine + 16 * i + 8 * b, *reinterpret_cast<uint32_t(*)[8]>(&out));
  }
  __device__ void wait() {
    __syncwarp();
    tmem_ld_wait();
  }
  __device__ void arrived(F2 (&out)[4]) const { tmem_ld_fence(*reinterpret_cast<uint32_t(*)[8]>(&out)); }
  __device__ void write(int i, int b, const F2 (&in)[4]) {
    __syncwarp();
    tmem_st8(mine + 16 * i + 8 * b, *reinterpret_cast<const uint32_t(*)[8]>(&in));
  }
};

struct BackwardPlan {
  RowPlan rows;
  RowItems items;
  bool joined;            // an item for each CTA, whose groups share its rows and join their sums; else items by group
  float* partials[SUMS];  // [items][hidden], or NULL: not wanted
};

template <typename TX, typename TR, int E, int V, bool SHIFTED, int STAGES>
__global__ void __launch_bounds__(kRowThreads, 1)
    residual_norm_backward_kernel(const __grid_constant__ ResidualArgs a, const __grid_constant__ BackwardPlan plan) {
  using Cols = RowCols<E, V, SHIFTED>;
  constexpr int NB = Cols::BLOCKS, BP = Cols::BP;
  constexpr bool TENSOR = Cols::N == 16;
  using KeptRows = RowKept<Cols, TENSOR>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float red[2][kMaxRowWarps][4 * kMaxRowWarps];
  __shared__ uint32_t tensor_base;
  if constexpr (TENSOR) {
    if (threadIdx.x < 32) {
      tmem_alloc(&tensor_base, KeptRows::kColumns);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  // only now: a dependent kernel that takes tensor memory and then waits for this one must not come first
  griddep_launch_dependents();
  const int threads = plan.rows.threads, warps = threads / 32;
  const int group = (threadIdx.x >> 5) / warps, warp = (threadIdx.x >> 5) - group * warps;
  const int t = threadIdx.x - group * threads;
  for (int i = threadIdx.x; i < 8 * kMaxRowWarps * kMaxRowWarps; i += blockDim.x) (&red[0][0][0])[i] = 0.f;
  __syncthreads();
  griddep_wait();
  const uint32_t me = blockIdx.x * plan.rows.groups + group;
  const RowItems items = plan.items;
  uint32_t item = plan.joined ? blockIdx.x : plan.rows.share.first(me);
  const uint32_t last = plan.joined ? item + 1 : plan.rows.share.first(me + 1);
  uint32_t row = 0, end = 0, by = 1;
  if (plan.rows.stride != 0) {
    row = me;
    end = static_cast<uint32_t>(a.rows);
    by = plan.rows.stride;
  } else if (item < last) {
    row = items.first_row(item);
    end = items.first_row(last);
    if (plan.joined) {
      const uint32_t n = plan.rows.groups, rows = end - row;
      end = row + rows * (group + 1) / n;
      row += rows * group / n;
    }
  }
  const Cols cols(t, threads, a.hidden);
  KeptRows kept(TENSOR ? tensor_base : 0u);
  auto clear = [&] {
    F2 zero[BP];
#pragma unroll
    for (int j = 0; j < BP; ++j) zero[j] = f2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < SUMS; ++i) {
#pragma unroll
      for (int b = 0; b < NB; ++b) kept.write(i, b, zero);
    }
  };
  // This thread's columns of the sums to a partial row.
  auto give = [&](int i, float* to) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      F2 v[BP];
      kept.read(i, b, v);
      kept.wait();
      kept.arrived(v);
      if constexpr (SHIFTED) {
#pragma unroll
        for (int j = 0; j < Cols::B; ++j) {
          const int k = b * Cols::BC + j / E;
          if (j % E < cols.count(k)) to[cols.col(k) + j % E] = lane_of(v, j);
        }
      } else {
        cols.store_floats(to, b, v);
      }
      __syncwarp();
    }
  };
  clear();
  if (row < end) {
    RowStream<TX, TR, E, V, SHIFTED, 2, 2, STAGES> rows;
    rows.start(cols, plan.rows, smem, row, end, by);
    const DropKey key(a.drop);
    const float inv_h = 1.f / static_cast<float>(a.hidden);
    const int bar = 1 + group;
    int turn = 0;  // of the parts of a sum
    const float2* rstd = reinterpret_cast<const float2*>(a.rstd);
    float2 next_r = rstd[row];  // loaded a row ahead
    const uint32_t per = static_cast<uint32_t>(a.rows_per_seq);
    uint32_t seq = row / per, seq_end = (seq + 1) * per;
    const bool by_seq = (a.branch_weight.seq_stride | a.gate.seq_stride | a.weight.seq_stride) != 0;
    auto params = [&] {
      F2 c[NB][BP], w[NB][BP];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        cols.branch_coefficient(a, seq, b, c[b]);
        cols.param(a.weight, seq, 1.f, b, w[b]);
      }
      __syncwarp();
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        kept.write(KEPT_C, b, c[b]);
        kept.write(KEPT_W, b, w[b]);
      }
    };
    const bool sum_branch = plan.partials[SUM_BRANCH] != nullptr, sum_weight = plan.partials[SUM_WEIGHT] != nullptr,
               sum_shift = plan.partials[SUM_SHIFT] != nullptr, normed = a.dy != nullptr;
    // a branch that is not normed is dropped itself, so that infinities there stay out of the sum of A
    const bool drop_x = a.dropped && !a.branch_norm, drop_u = a.dropped && a.branch_norm;
    params();
    uint32_t item_end = plan.joined ? 0u : static_cast<uint32_t>(items.first_row(item + 1));
    for (;;) {
      const uint64_t element = static_cast<uint64_t>(row) * static_cast<uint32_t>(a.hidden);  // the row's first
      const uint32_t bits = a.dropped ? cols.kept(a.drop, key, element) : ~0u;
      const float2 rs = next_r;
      if (row + by < end) next_r = rstd[row + by];
      rows.advance(cols, plan.rows);
      kept.settle();
      F2 x[NB][BP], q[NB][BP], hat[NB][BP];  // x', dH and what it is made of, h'
      F2 s0 = f2(0.f, 0.f), s1 = s0, s2 = s0, s3 = s0;  // of g h', u dh, u g, u h'
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        F2 u[BP], c[BP];
        kept.read(KEPT_C, b, c);
        rows.template get<0>(cols, plan.rows, row, b, x[b]);
        rows.template get<3>(cols, plan.rows, row, b, q[b]);
        if (drop_x) Cols::drop(bits, b, x[b]);
        kept.wait();
        kept.arrived(c);
#pragma unroll
        for (int j = 0; j < BP; ++j) {
          x[b][j] = mul2(x[b][j], f2(rs.x, rs.x));
          u[j] = mul2(x[b][j], c[j]);
        }
        if (drop_u) Cols::drop(bits, b, u);
#pragma unroll
        for (int j = 0; j < BP; ++j) s1 = fma2(u[j], q[b][j], s1);
        if (normed) {
          F2 dy[BP], w[BP], sum[BP];
          kept.read(KEPT_W, b, w);
          kept.read(SUM_WEIGHT, b, sum);
          rows.template get<1>(cols, plan.rows, row, b, dy);
          rows.template get<2>(cols, plan.rows, row, b, hat[b]);
          kept.wait();
          kept.arrived(w);
          kept.arrived(sum);
#pragma unroll
          for (int j = 0; j < BP; ++j) {
            hat[b][j] = mul2(add2(hat[b][j], u[j]), f2(rs.y, rs.y));
            sum[j] = fma2(dy[j], hat[b][j], sum[j]);
            const F2 g = mul2(dy[j], w[j]);
            s0 = fma2(g, hat[b][j], s0);
            s2 = fma2(u[j], g, s2);
            s3 = fma2(u[j], hat[b][j], s3);
            q[b][j] = fma2(g, f2(rs.y, rs.y), q[b][j]);
          }
          if (sum_weight) kept.write(SUM_WEIGHT, b, sum);
          if (sum_shift) {
            kept.read(SUM_SHIFT, b, sum);
            kept.wait();
            kept.arrived(sum);
#pragma unroll
            for (int j = 0; j < BP; ++j) sum[j] = add2(dy[j], sum[j]);
            kept.write(SUM_SHIFT, b, sum);
          }
        }
      }
      float s[4] = {s0.x + s0.y, s1.x + s1.y, s2.x + s2.y, s3.x + s3.y};
      if (a.branch_norm) {
        row_sum(s, red[turn ^= 1][group], warps, warp, bar);
      } else if (normed) {
        float one[1] = {s[0]};
        row_sum(one, red[turn ^= 1][group], warps, warp, bar);
        s[0] = one[0];
      }
      const float mean = s[0] * inv_h, m = -mean * rs.y;
      const float m1 = a.branch_norm ? -(s[1] + rs.y * (s[2] - mean * s[3])) * inv_h : 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        F2 c[BP], sum[BP];
        kept.read(KEPT_C, b, c);
        kept.read(SUM_BRANCH, b, sum);
        if (normed) {
#pragma unroll
          for (int j = 0; j < BP; ++j) q[b][j] = fma2(hat[b][j], f2(m, m), q[b][j]);
        }
        kept.wait();
        kept.arrived(c);
        kept.arrived(sum);
        if (a.dres != nullptr) cols.store(static_cast<TR*>(a.dres) + element, b, q[b]);
        if (a.dropped) Cols::drop(bits, b, q[b]);
        if (sum_branch) {
#pragma unroll
          for (int j = 0; j < BP; ++j) sum[j] = fma2(q[b][j], x[b][j], sum[j]);
          __syncwarp();
          kept.write(SUM_BRANCH, b, sum);
        }
        if (a.dx != nullptr) {
#pragma unroll
          for (int j = 0; j < BP; ++j) q[b][j] = mul2(q[b][j], c[j]);
          if (a.branch_norm) {
#pragma unroll
            for (int j = 0; j < BP; ++j) q[b][j] = mul2(fma2(x[b][j], f2(m1, m1), q[b][j]), f2(rs.x, rs.x));
          }
          cols.store(static_cast<TX*>(a.dx) + element, b, q[b]);
        }
        __syncwarp();
      }
      row += by;
      if (row == item_end) {
        kept.settle();
#pragma unroll
        for (int i = 0; i < SUMS; ++i)
          if (plan.partials[i] != nullptr) give(i, plan.partials[i] + static_cast<int64_t>(item) * a.hidden);
        clear();
        ++item;
        if (item < last) item_end = items.first_row(item + 1);
      }
      if (row >= end) break;
      if (row == seq_end) {
        ++seq;
        seq_end += per;
        if (by_seq) params();
      }
    }
  }
  kept.settle();
  if (plan.joined) {
    // over the ring: no copy is in flight past the last row, and the other groups are done with theirs
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float* parts = reinterpret_cast<float*>(smem);  // [SUMS][groups][hidden]
#pragma unroll
    for (int i = 0; i < SUMS; ++i) {
      if (plan.partials[i] == nullptr) continue;
      give(i, plan.rows.groups > 1 ? parts + (i * plan.rows.groups + group) * a.hidden
                                   : plan.partials[i] + static_cast<int64_t>(blockIdx.x) * a.hidden);
    }
    if (plan.rows.groups > 1) __syncthreads();
    for (int i = 0; i < SUMS && plan.rows.groups > 1; ++i) {
      if (plan.partials[i] == nullptr) continue;
      for (int c = threadIdx.x; c < a.hidden; c += blockDim.x) {
        float v = 0.f;
        for (int g = 0; g < plan.rows.groups; ++g) v += parts[(i * plan.rows.groups + g) * a.hidden + c];
        plan.partials[i][static_cast<int64_t>(blockIdx.x) * a.hidden + c] = v;
      }
    }
  }
  if constexpr (TENSOR) {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x < 32) tmem_dealloc(tensor_base, KeptRows::kColumns);
  }
}

// Rows of any width: a CTA for each, which reads it again for the results (from L1 and L2); a CTA's items' sums are
// added up in the partial rows themselves, each column by one thread. Slow: it waits for its loads of one column and for the
// partial rows (4096 x 12288 bf16 2237 us, 4 % of the copy rate; 4096 x 5329 fp32 692 us, 12 %).
template <typename TX, typename TR>
__global__ void __launch_bounds__(kRowThreads)
    residual_norm_backward_any_kernel(const __grid_constant__ ResidualArgs a, const __grid_constant__ BackwardPlan plan) {
  __shared__ __align__(16) float red[2][4 * kMaxRowWarps];
  griddep_launch_dependents();
  griddep_wait();
  const DropKey key(a.drop);
  const float s_branch = a.dropped ? a.scale * a.drop.scale : a.scale;
  const float inv_h = 1.f / static_cast<float>(a.hidden);
  const RowItems items = plan.items;
  int turn = 0;
  for (int64_t item = blockIdx.x; item < items.count(); item += gridDim.x) {
    const int64_t r0 = items.first_row(item), r1 = items.first_row(item + 1);
    for (int64_t r = r0; r < r1; ++r) {
      const int64_t seq = r / a.rows_per_seq;
      const TX* x = static_cast<const TX*>(a.x) + r * a.x_stride;
      const TX* dy = static_cast<const TX*>(a.dy) + r * a.dy_stride;
      const TR* res = static_cast<const TR*>(a.res) + r * a.res_stride;
      const TR* dh = static_cast<const TR*>(a.dh) + r * a.dh_stride;
      const float2 rs = reinterpret_cast<const float2*>(a.rstd)[r];
      auto param = [&](const RowParam& p, int i, float otherwise) {
        return p.p != nullptr ? load_as_float(p.p, seq * p.seq_stride + i, p.dtype) : otherwise;
      };
      struct At {
        float x, c, hat, g, dy, dh;
        bool keep;
      };
      auto at = [&](int i) {
        At v;
        v.x = Ty<TX>::to_f(x[i]) * rs.x;
        v.c = param(a.branch_weight, i, 1.f) * param(a.gate, i, 1.f) * s_branch;
        v.keep = !a.dropped || (!a.drop.all && key.kept<1>(static_cast<uint64_t>(r * a.hidden + i)));
        v.dh = a.dh != nullptr ? Ty<TR>::to_f(dh[i]) : 0.f;
        v.dy = v.g = v.hat = 0.f;
        if (a.dy != nullptr) {
          v.dy = Ty<TX>::to_f(dy[i]);
          v.g = v.dy * param(a.weight, i, 1.f);
          v.hat = (Ty<TR>::to_f(res[i]) + (v.keep ? v.x * v.c : 0.f)) * rs.y;
        }
        return v;
      };
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      for (int i = threadIdx.x; i < a.hidden; i += kRowThreads) {
        const At v = at(i);
        const float u = v.keep ? v.x * v.c : 0.f;
        s[0] = fmaf(v.g, v.hat, s[0]);
        s[1] = fmaf(u, v.dh, s[1]);
        s[2] = fmaf(u, v.g, s[2]);
        s[3] = fmaf(u, v.hat, s[3]);
      }
      row_sum(s, red[turn ^= 1], kMaxRowWarps, threadIdx.x >> 5, 1);
      const float mean = s[0] * inv_h;
      const float m1 = a.branch_norm ? (s[1] + rs.y * (s[2] - mean * s[3])) * inv_h : 0.f;
      for (int i = threadIdx.x; i < a.hidden; i += kRowThreads) {
        const At v = at(i);
        const float d = v.dh + rs.y * (v.g - v.hat * mean);
        const float e = v.keep ? d : 0.f;
        if (a.dres != nullptr) static_cast<TR*>(a.dres)[r * a.hidden + i] = Ty<TR>::from_f(d);
        if (a.dx != nullptr) {
          const float b = e * v.c;
          static_cast<TX*>(a.dx)[r * a.hidden + i] = Ty<TX>::from_f(a.branch_norm ? rs.x * (b - v.x * m1) : b);
        }
        const float add[SUMS] = {v.keep ? e * v.x : 0.f, v.dy * v.hat, v.dy};
#pragma unroll
        for (int p = 0; p < SUMS; ++p) {
          if (plan.partials[p] == nullptr) continue;
          float* o = plan.partials[p] + item * a.hidden + i;
          *o = r == r0 ? add[p] : *o + add[p];
        }
      }
    }
  }
}

// One parameter's gradient: out[o, i] = factor * sum over the output's partial rows of other[sequence, i] * partials[m, i].
struct ParamSum {
  const float* partials;
  RowParam out;    // `grad` with dtype; one row for all or (seq_stride not 0) one for each sequence
  RowParam other;  // the parameter that multiplies it, by sequence (p NULL: none)
  float factor;
};
struct ParamSums {
  ParamSum of[4];
  int n;
  uint32_t parts, chunks, seqs;  // partial rows; of a sequence; sequences
  int hidden;
};

// C neighbouring columns of one output for each lane of a CTA, whose warps take every so manyth partial row, several
// loads in flight; sums in fp64. Bound by latency: the partial rows come from L2.
template <int C>
__global__ void __launch_bounds__(512) residual_param_grad_kernel(const __grid_constant__ ParamSums s) {
  constexpr int AHEAD = 10;  // 16 warps of them cover a partial row for each SM
  __shared__ double red[16][32 * C + 1];
  griddep_launch_dependents();
  const ParamSum& p = s.of[blockIdx.y];
  const uint32_t col_blocks = (s.hidden + 32 * C - 1) / (32 * C);
  const bool own = p.out.seq_stride != 0;
  const uint32_t jobs = (own ? s.seqs : 1u) * col_blocks;
  const uint32_t warps = blockDim.x / 32, warp = threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  // a factor that differs between the rows of an output goes into the sum, another one behind it
  const bool inside = p.other.p != nullptr && p.other.seq_stride != 0 && !own;
  griddep_wait();
  for (uint32_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const uint32_t o = job / col_blocks;
    const int i = static_cast<int>(job - o * col_blocks) * 32 * C + lane * C;
    const uint32_t m1 = own ? (o + 1) * s.chunks : s.parts;
    double t[C] = {};
    if (i < s.hidden) {
      for (uint32_t m0 = (own ? o * s.chunks : 0u) + warp; m0 < m1; m0 += warps * AHEAD) {
        float v[AHEAD][C];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const uint32_t m = m0 + k * warps;
#pragma unroll
          for (int j = 0; j < C; ++j) v[k][j] = 0.f;
          if (m < m1) load_floats<C>(p.partials, static_cast<int64_t>(m) * s.hidden + i, F32, v[k]);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const uint32_t m = m0 + k * warps;
#pragma unroll
          for (int j = 0; j < C; ++j) {
            double x = v[k][j];
            if (inside && m < m1)
              x *= load_as_float(p.other.p, static_cast<int64_t>(m / s.chunks) * p.other.seq_stride + i + j, p.other.dtype);
            t[j] += x;
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < C; ++j) red[warp][lane * C + j] = t[j];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * C; c += blockDim.x) {
      const int col = i - lane * C + c;
      if (col >= s.hidden) break;
      double sum = 0.0;
#pragma unroll
      for (int w = 0; w < 16; ++w)
        if (w < static_cast<int>(warps)) sum += red[w][c];
      if (p.other.p != nullptr && !inside)
        sum *= load_as_float(p.other.p, static_cast<int64_t>(own ? o : 0u) * p.other.seq_stride + col, p.other.dtype);
      const float v = static_cast<float>(sum * p.factor);
      const int64_t at = static_cast<int64_t>(o) * s.hidden + col;
      if (p.out.dtype == F32) static_cast<float*>(p.out.grad)[at] = v;
      else if (p.out.dtype == F16) static_cast<__half*>(p.out.grad)[at] = __float2half_rn(v);
      else static_cast<__nv_bfloat16*>(p.out.grad)[at] = __float2bfloat16_rn(v);
    }
    __syncthreads();
  }
}

namespace {
constexpr int64_t kItemRows = 2048;  // most rows that a thread adds up in fp32

bool wants(const ResidualArgs& a, int sum) {
  if (sum == SUM_BRANCH) return a.gate.grad != nullptr || a.branch_weight.grad != nullptr;
  return sum == SUM_WEIGHT ? a.weight.grad != nullptr : a.shift.grad != nullptr;
}

struct Shape {
  int cols, threads;  // columns a thread; 0: any
  bool shifted;
};
Shape shape_of(const ResidualArgs& a) {
  const int e = 16 / std::max(row_elem_bytes(a.x_dtype), row_elem_bytes(a.res_dtype));
  const bool shifted = !rows_aligned(a, true);
  // A warp a row as far as 8 columns a thread carry it, then 16 columns a thread; with 4 bytes a column, or two vectors
  // for each chunk, 8 as far as they go, for which more rows fit into shared memory.
  for (const auto& [stride, dtype] : {std::pair<int64_t, int>{a.x_stride, a.x_dtype}, {a.dy_stride, a.x_dtype},
                                      {a.res_stride, a.res_dtype}, {a.dh_stride, a.res_dtype}})
    if (stride * row_elem_bytes(dtype) > UINT32_MAX) return {0, kRowThreads, shifted};
  if (a.hidden <= 256) return {8, 32, shifted};
  if (a.x_dtype == F32 || shifted)
    if (const int t = row_threads(a.hidden, e, 8 / e)) return {8, t, shifted};
  if (const int t = row_threads(a.hidden, e, 16 / e); t != 0 && !(shifted && a.res_dtype == F32)) return {16, t, shifted};
  return {0, kRowThreads, shifted};
}

// The split. One item for each CTA of a full grid where that leaves few of them without one and the rows of an item are
// few enough for fp32 sums; else (many sequences, very many rows) items for every group.
RowItems items_of(const ResidualArgs& a, const Shape& sh, bool* joined) {
  bool by_seq = false;
  for (const RowParam* p : {&a.branch_weight, &a.gate, &a.weight, &a.shift}) by_seq = by_seq || (p->seq_stride != 0);
  RowItems it;
  it.seqs = by_seq ? a.rows / a.rows_per_seq : 1;
  it.seq_rows = by_seq ? a.rows_per_seq : a.rows;
  const int64_t ctas = num_sms(), per_cta = kRowThreads / sh.threads;
  it.chunks = std::min(std::max<int64_t>(1, ctas / it.seqs), it.seq_rows);
  const int64_t rows = (it.seq_rows + it.chunks - 1) / it.chunks;
  *joined = sh.cols > 0 && it.count() <= ctas && rows <= kItemRows * std::min(per_cta, rows) &&
            (it.seqs == 1 || it.count() * 10 >= ctas * 9);
  if (!*joined) {
    it.chunks = std::max({ctas * per_cta / it.seqs, (it.seq_rows + kItemRows - 1) / kItemRows, int64_t{1}});
    it.chunks = std::min(it.chunks, it.seq_rows);
  }
  it.runs = Split::make(it.seq_rows, it.chunks);
  return it;
}

template <typename TX, typename TR, int V, bool SHIFTED>
cudaError_t launch_rows(const ResidualArgs& a, BackwardPlan& plan, cudaStream_t st) {
  constexpr int E = kRowChunk<TX, TR>, STAGES = row_stages<TX, TR>(E * V, 2, 2, SHIFTED);
  auto* kernel = residual_norm_backward_kernel<TX, TR, E, V, SHIFTED, STAGES>;
  using Stream = RowStream<TX, TR, E, V, SHIFTED, 2, 2, STAGES>;
  // A launch before it may let this one start before its own CTAs have their tensor memory: none of those (120 KB and
  // more of shared memory) shares an SM with a CTA of this one, whose allocation would keep theirs waiting.
  static_assert(E * V != 16 || Stream::kSmemBytes >= 120 * 1024, "alone on its SM beside kernels with tensor memory");
  const int threads = plan.rows.threads;
  const int64_t count = plan.items.count();
  // groups of a CTA: as many as have rows of their own
  const int64_t most = plan.joined ? (plan.items.seq_rows + plan.items.chunks - 1) / plan.items.chunks : count / num_sms();
  plan.rows.groups = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kRowThreads / threads, most)));
  const int block = plan.rows.groups * threads;
  // the ring, and in its place the groups' sums
  const size_t smem = std::max(Stream::kSmemBytes, sizeof(float) * SUMS * kRowThreads * E * V);
  const void* fn = reinterpret_cast<const void*>(kernel);
  // at least a little over 48 KB: the sums' static part comes on top
  if (const cudaError_t e = ensure_smem_attr(fn, std::max<size_t>(smem, 49 * 1024)); e != cudaSuccess) return e;
  const int64_t all = static_cast<int64_t>(num_sms()) * std::max(1, cached_occupancy(fn, block, smem));
  const int64_t grid = plan.joined ? count : std::min<int64_t>(all, (count + plan.rows.groups - 1) / plan.rows.groups);
  plan.rows.share = Split::make(count, grid * plan.rows.groups);
  plan.rows.stride = plan.joined && plan.items.seqs == 1 ? static_cast<uint32_t>(grid * plan.rows.groups) : 0;
  note_launch();
  return launch_gemm_grid(kernel, block, static_cast<int>(grid), 1, smem, st, a, plan);
}

template <typename TX, typename TR>
cudaError_t launch_types(const ResidualArgs& a, BackwardPlan& plan, const Shape& sh, cudaStream_t st) {
  constexpr int HALF = 8 / kRowChunk<TX, TR>;  // chunks of 8 columns
  constexpr int64_t x = sizeof(TX), r = sizeof(TR);
  set_tensors(&plan.rows, {{a.x, a.x_stride * x}, {a.dy, a.dy_stride * x}, {a.dy ? a.res : nullptr, a.res_stride * r},  // h serves the norm
                           {a.dh, a.dh_stride * r}});
  if (sh.cols == 8) return sh.shifted ? launch_rows<TX, TR, HALF, true>(a, plan, st) : launch_rows<TX, TR, HALF, false>(a, plan, st);
  if (sh.cols == 16) {
    if (!sh.shifted) return launch_rows<TX, TR, 2 * HALF, false>(a, plan, st);
    // two vectors a chunk of 4 bytes a column: more than shared memory holds
    if constexpr (sizeof(TR) == 2) return launch_rows<TX, TR, 2 * HALF, true>(a, plan, st);
  }
  note_launch();
  return launch_dependent(residual_norm_backward_any_kernel<TX, TR>,
                          static_cast<int>(std::min<int64_t>(plan.items.count(), num_sms() * 4ll)), kRowThreads, st, a, plan);
}
}  // namespace

size_t residual_norm_backward_workspace_bytes(const ResidualArgs& a) {
  int64_t wanted = 0;
  for (int i = 0; i < SUMS; ++i) wanted += wants(a, i);
  if (wanted == 0) return 0;
  const int64_t row = (static_cast<int64_t>(a.hidden) * 4 + 15) / 16 * 16;
  bool joined;
  return static_cast<size_t>(wanted * items_of(a, shape_of(a), &joined).count() * row);
}

cudaError_t residual_norm_backward_launch(const ResidualArgs& a, void* ws, cudaStream_t st) {
  const Shape sh = shape_of(a);
  BackwardPlan plan{};
  plan.rows.threads = sh.threads;
  plan.items = items_of(a, sh, &plan.joined);
  float* at = static_cast<float*>(ws);
  const int64_t count = plan.items.count();
  bool any = false;
  for (int i = 0; i < SUMS; ++i) {
    if (!wants(a, i)) continue;
    plan.partials[i] = at;
    at += count * ((a.hidden + 3) / 4 * 4);
    any = true;
  }
  cudaError_t e;
  if (a.x_dtype == F16)
    e = a.res_dtype == F32 ? launch_types<__half, float>(a, plan, sh, st) : launch_types<__half, __half>(a, plan, sh, st);
  else if (a.x_dtype == BF16)
    e = a.res_dtype == F32 ? launch_types<__nv_bfloat16, float>(a, plan, sh, st)
                           : launch_types<__nv_bfloat16, __nv_bfloat16>(a, plan, sh, st);
  else
    e = launch_types<float, float>(a, plan, sh, st);
  if (e != cudaSuccess || !any) return e;
  ParamSums s{};
  s.parts = static_cast<uint32_t>(count);
  s.chunks = static_cast<uint32_t>(plan.items.chunks);
  s.seqs = static_cast<uint32_t>(a.rows / a.rows_per_seq);
  s.hidden = a.hidden;
  const float f = a.dropped ? a.scale * a.drop.scale : a.scale;
  const RowParam none{};
  auto add = [&](int sum, const RowParam& p, const RowParam& other, float factor) {
    if (p.grad != nullptr) s.of[s.n++] = ParamSum{plan.partials[sum], p, other, factor};
  };
  add(SUM_BRANCH, a.gate, a.branch_weight, f);
  add(SUM_BRANCH, a.branch_weight, a.gate, f);
  add(SUM_WEIGHT, a.weight, none, 1.f);
  add(SUM_SHIFT, a.shift, none, 1.f);
  int64_t outs = 1, most = 1;  // outputs, and partial rows of one
  for (int i = 0; i < s.n; ++i) {
    const bool own = s.of[i].out.seq_stride != 0;
    outs = std::max<int64_t>(outs, own ? s.seqs : 1);
    most = std::max(most, own ? plan.items.chunks : count);
  }
  const int c = a.hidden % 2 == 0 ? 2 : 1;
  const int warps = static_cast<int>(std::min<int64_t>(16, (most + 1) / 2));  // two loads a lane at least
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(outs * ((a.hidden + 32 * c - 1) / (32 * c)), num_sms() * 16ll)), s.n);
  cfg.blockDim = dim3(std::max(1, warps) * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, c == 2 ? residual_param_grad_kernel<2> : residual_param_grad_kernel<1>, s);
}

}  // namespace tfo
