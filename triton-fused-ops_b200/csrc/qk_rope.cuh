// Rotation of query and key heads by rotary table rows, alone or after an
// RMSNorm of each head, in one pass over both tensors.
//
//   u = x / sqrt(mean(x^2) + eps) * w      (norm only; mean over the head)
//   (y1, y2) = (u1 c - u2 s, u1 s + u2 c)  for each rotated pair of columns
//   columns at or past rotary_dim: y = u
//
// Everything is held in fp32 from the load of x to one rounding of y.
//
// Floor: HBM (x read once, y written once; table rows and weights come from
// L2). A group of lanes (two vectors each, heads.cuh) owns NH consecutive heads
// of one token: the lane's table columns and weights are combined once into
// the coefficients of the rotation and used for the NH heads.
//
// Measured: 8 x 8192 tokens of 32 + 8 heads of 128 columns, bf16, with the
// norm: 215 us, 95 % of the measured copy rate (1.34 GB); 65536 tokens of
// 16 + 16 heads of 64, fp32: 174 us (94 %); of 12 + 3 heads of 80, f16: 69 us
// (70 %; five lanes a head, summed by five shuffles); of 8 + 1 heads of 256,
// bf16: 126 us (73 %; a unit of the keys holds one head where it has room for four,
// and both sides read a token's table row). One token: 1.9 us, a launch.
//
// AXES: a token has a position on each of several axes and a pair of columns
// turns by that of its own (qk_rope_axes.cu); else one position (qk_rope.cu).
#pragma once

#include "heads.cuh"

namespace tfo {

template <int E, bool PAIRS, bool NORM>
using Rotation = std::conditional_t<NORM, WeightedRotation<E, PAIRS>, PlainRotation<E, PAIRS>>;

// This lane's part of a head's sum of squares.
template <int E>
__device__ __forceinline__ float lane_squares(const F2 (&fa)[E / 2], const F2 (&fb)[E / 2]) {
  F2 ss = mul2(fa[0], fa[0]);
#pragma unroll
  for (int j = 1; j < E / 2; ++j) ss = fma2(fa[j], fa[j], ss);
#pragma unroll
  for (int j = 0; j < E / 2; ++j) ss = fma2(fb[j], fb[j], ss);
  return ss.x + ss.y;
}

// One head on a lane's two vectors, in place; `squares`: of the whole head.
template <int E, bool PAIRS, bool NORM>
__device__ __forceinline__ void norm_rotate(F2 (&fa)[E / 2], F2 (&fb)[E / 2], const Rotation<E, PAIRS, NORM>& rot, const LaneCols& col,
                                            float squares, float inv_d, float eps) {
  float rstd = 1.f;
  if constexpr (NORM) rstd = rsqrtf(squares * inv_d + eps);
  rot.apply(fa, fb, col);
  if constexpr (NORM) {
    const F2 r2 = f2(rstd, rstd);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      fa[j] = mul2(fa[j], r2);
      fb[j] = mul2(fb[j], r2);
    }
  }
}

// The rotation (with the weights) of a token for this lane's columns.
template <int E, bool PAIRS, bool NORM, bool AXES>
__device__ __forceinline__ void token_rotation(Rotation<E, PAIRS, NORM>& rot, const HeadArgs& a, const HeadSide& side,
                                               const LaneCols& col, const TokenTable<E, PAIRS, AXES>& table, int64_t b,
                                               int64_t sq, bool report, uint32_t* err) {
  float c[E], s[E];
  table.load(a.t, b, sq, col, a.inverse, report, err, c, s);
  if constexpr (NORM) {
    float wa[E], wb[E];
#pragma unroll
    for (int j = 0; j < E; ++j) wa[j] = wb[j] = 1.f;
    if (side.weight != nullptr) {
      if (col.va >= 0) load_floats<E>(side.weight, col.va * E, side.w_dtype, wa);
      if (col.vb >= 0) load_floats<E>(side.weight, col.vb * E, side.w_dtype, wb);
    }
    rot.set(c, s, wa, wb, col);
  } else {
    rot.set(c, s);
  }
}

// Few tokens: a CTA per handful of groups, one unit each.
template <typename T, int E, bool PAIRS, bool NORM, int NH, bool AXES>
__global__ void __launch_bounds__(256) qk_rope_kernel(const HeadArgs a, int lanes, uint32_t units, uint32_t q_chunks,
                                                      uint32_t chunks, FastDiv by_chunks, FastDiv by_seq, uint32_t* err) {
  using V = HeadVec<T, E>;
  griddep_launch_dependents();
  griddep_wait();
  const LaneGroup group(lanes);
  const uint32_t want = (blockIdx.x * 8u + (threadIdx.x >> 5)) * (32 / lanes) + group.group;
  const uint32_t unit = min(want, units - 1);  // spare groups repeat the last unit and store nothing
  const uint32_t token = by_chunks.div(unit);
  const uint32_t chunk = unit - token * chunks;
  const uint32_t b = by_seq.div(token);
  const uint32_t sq = token - b * static_cast<uint32_t>(a.seq);
  const HeadSide& side = chunk < q_chunks ? a.q : a.k;
  const int h0 = static_cast<int>(chunk < q_chunks ? chunk : chunk - q_chunks) * NH;
  const int heads = want < units && !group.spare ? side.heads - h0 : 0;  // of this unit
  const int D = a.head_dim;
  const LaneCols col = lane_cols<PAIRS>(group.p, lanes, D / E, a.rotary_dim / E);

  const T* x = static_cast<const T*>(side.x) + b * side.stride_batch + sq * side.stride_seq + h0 * side.stride_head;
  typename V::Raw ra[NH], rb[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i, x += side.stride_head) {
    ra[i] = i < heads && col.va >= 0 ? V::load(x + col.va * E) : V::zero();
    rb[i] = i < heads && col.vb >= 0 ? V::load(x + col.vb * E) : V::zero();
  }
  Rotation<E, PAIRS, NORM> rot;
  token_rotation<E, PAIRS, NORM, AXES>(rot, a, side, col, TokenTable<E, PAIRS, AXES>(a.t, col), b, sq, group.p == 0, err);
  T* out = static_cast<T*>(side.out) + (static_cast<int64_t>(token) * side.heads + h0) * D;
  const float inv_d = 1.f / static_cast<float>(D);
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    F2 fa[E / 2], fb[E / 2];
    V::unpack(ra[i], fa);
    V::unpack(rb[i], fb);
    const float squares = NORM ? group.sum(lane_squares<E>(fa, fb)) : 0.f;
    norm_rotate<E, PAIRS, NORM>(fa, fb, rot, col, squares, inv_d, a.eps);
    if (i < heads) {
      if (col.va >= 0) V::store(out + i * D + col.va * E, fa);
      if (col.vb >= 0) V::store(out + i * D + col.vb * E, fb);
    }
  }
}

// Many tokens: resident CTAs, each lane group streaming units of one side
// through shared memory (HeadStream). FULL: every lane has both its vectors.
template <typename T, int E, bool PAIRS, bool NORM, int NH, int STAGES, bool FULL, bool AXES>
__global__ void __launch_bounds__(256, 2) qk_rope_stream_kernel(const HeadArgs a, int lanes, SideSplit split,
                                                                FastDiv by_seq, FastDiv by_q_chunks, FastDiv by_k_chunks,
                                                                uint32_t* err) {
  using V = HeadVec<T, E>;
  extern __shared__ __align__(16) uint8_t smem[];
  griddep_launch_dependents();
  griddep_wait();
  const bool is_q = blockIdx.x < static_cast<unsigned>(split.q_ctas);
  const HeadSide& side = is_q ? a.q : a.k;
  const uint32_t cta = is_q ? blockIdx.x : blockIdx.x - split.q_ctas;
  const uint32_t per_warp = 32 / lanes;
  const uint32_t groups = static_cast<uint32_t>(is_q ? split.q_ctas : split.k_ctas) * 8u * per_warp;
  const LaneGroup group(lanes);
  const int D = a.head_dim, heads = side.heads;
  const LaneCols col = lane_cols<PAIRS>(group.p, lanes, D / E, a.rotary_dim / E);
  const int column = max(0, col.va) * E;
  const TokenTable<E, PAIRS, AXES> table(a.t, col);

  HeadStream<T, E, NH, STAGES, 1, FULL> st;
  st.in[0] = {static_cast<const T*>(side.x) + column, side.stride_batch, side.stride_seq, side.stride_head};
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
  uint32_t lead = (cta * 8u + (threadIdx.x >> 5)) * per_warp;
  st.start(smem, lead + group.group, groups);
  const float inv_d = 1.f / static_cast<float>(D);
  const int most = min(NH, heads);
  int stage = 0;
  for (; lead < st.units; lead += groups) {
    const uint32_t unit = min(lead + group.group, st.units - 1);
    const uint32_t token = st.by_chunks.div(unit);
    const int h0 = static_cast<int>(unit - token * st.chunks) * NH;
    const int mine = lead + group.group < st.units ? heads - h0 : 0;  // heads of this unit
    const uint32_t b = by_seq.div(token);
    Rotation<E, PAIRS, NORM> rot;
    token_rotation<E, PAIRS, NORM, AXES>(rot, a, side, col, table, b, token - b * st.seq, group.p == 0, err);
    T* out = static_cast<T*>(side.out) + (static_cast<int64_t>(token) * heads + h0) * D + column;
    st.wait();
    // Lane groups that do not fill the warp mostly sum by a shuffle for each lane: there
    // the heads' sums go side by side and the heads are read again after them
    // (12 + 3 heads of 80, f16, 65536 tokens 72.4 -> 68.8 us).
    constexpr int AT_ONCE = FULL || !NORM ? 1 : NH;
#pragma unroll
    for (int i0 = 0; i0 < NH; i0 += AT_ONCE) {
      if (i0 >= most) break;
      F2 fa[E / 2], fb[E / 2];
      auto read = [&](int i) {
        V::unpack(*st.slot(stage, 0, i, 0), fa);
        V::unpack(*st.slot(stage, 0, i, 1), fb);
      };
      float squares[AT_ONCE] = {};
#pragma unroll
      for (int n = 0; n < AT_ONCE; ++n) {
        read(i0 + n);
        if constexpr (NORM) squares[n] = lane_squares<E>(fa, fb);
      }
      if constexpr (NORM && AT_ONCE == 1) squares[0] = group.sum(squares[0]);
      if constexpr (NORM && AT_ONCE > 1) group.sum(squares);
      if constexpr (AT_ONCE > 1) asm volatile("" ::: "memory");  // registers are not kept over the sums
#pragma unroll
      for (int n = 0; n < AT_ONCE; ++n) {
        const int i = i0 + n;
        if constexpr (AT_ONCE > 1) read(i);
        norm_rotate<E, PAIRS, NORM>(fa, fb, rot, col, squares[n], inv_d, a.eps);
        if (i < mine) {
          if (FULL || st.has_a) V::store(out + i * D, fa);
          if (FULL || st.has_b) V::store(out + i * D + st.vb_offset, fb);
        }
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    st.load();  // into the stage that the unit before this one has left
  }
}

// Any head width, stride and alignment: one warp per head, scalar accesses.
template <typename T, bool AXES>
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
    int64_t pos = AXES ? 0 : token_position(a.t, b, sq, err, lane == 0);
    for (int i = lane; i < half; i += 32) {
      float c, s;
      if constexpr (AXES) pos = axis_position(a.t, b, sq, LaneAxes::of(a.t, i), err);
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
// Warps that units of four heads make.
inline int64_t head_warps4(const HeadArgs& a, int elems) {
  const int lanes = (a.head_dim / elems + 1) / 2;
  return a.batch * a.seq * ((a.q.heads + 3) / 4 + (a.k.heads + 3) / 4) / (32 / lanes);
}

template <typename T, int E, bool PAIRS, bool NORM, int NH, bool AXES>
cudaError_t launch_units(const HeadArgs& a, int lanes, cudaStream_t st) {
  const uint32_t qc = (a.q.heads + NH - 1) / NH, kc = (a.k.heads + NH - 1) / NH;
  const uint32_t units = static_cast<uint32_t>(a.batch * a.seq) * (qc + kc);
  const uint32_t per_cta = 8u * (32 / lanes);
  note_launch();
  return launch_dependent(qk_rope_kernel<T, E, PAIRS, NORM, NH, AXES>, static_cast<int>((units + per_cta - 1) / per_cta), 256,
                          st, a, lanes, units, qc, qc + kc, FastDiv::make(qc + kc),
                          FastDiv::make(static_cast<uint32_t>(a.seq)), error_word_ptr());
}

template <typename T, int E, bool PAIRS, bool NORM, int NH, int STAGES, bool AXES>
cudaError_t launch_stream(const HeadArgs& a, int lanes, cudaStream_t st) {
  const bool full = a.head_dim == 2 * E * lanes && 32 % lanes == 0;
  auto* kernel = full ? qk_rope_stream_kernel<T, E, PAIRS, NORM, NH, STAGES, true, AXES>
                      : qk_rope_stream_kernel<T, E, PAIRS, NORM, NH, STAGES, false, AXES>;
  constexpr size_t smem = HeadStream<T, E, NH, STAGES, 1, true>::kSmemBytes;
  const void* fn = reinterpret_cast<const void*>(kernel);
  if (const cudaError_t e = ensure_smem_attr(fn, smem); e != cudaSuccess) return e;
  // one wave of CTAs, shared between the sides by their units
  const uint32_t qc = (a.q.heads + NH - 1) / NH, kc = (a.k.heads + NH - 1) / NH;
  const int64_t all = static_cast<int64_t>(num_sms()) * cached_occupancy(fn, 256, smem);
  const int64_t per_cta = 8 * (32 / lanes);
  auto share = [&](uint32_t c) {
    const int64_t most = (a.batch * a.seq * c + per_cta - 1) / per_cta;
    return c == 0 ? 0 : static_cast<int>(std::min(most, std::max<int64_t>(1, all * c / (qc + kc))));
  };
  const SideSplit split{share(qc), share(kc)};
  note_launch();
  return launch_gemm_grid(kernel, 256, split.q_ctas + split.k_ctas, 1, smem, st, a, lanes, split,
                          FastDiv::make(static_cast<uint32_t>(a.seq)), FastDiv::make(std::max(1u, qc)),
                          FastDiv::make(std::max(1u, kc)), error_word_ptr());
}

template <typename T, int E, bool PAIRS, bool NORM, bool AXES>
cudaError_t launch_form(const HeadArgs& a, cudaStream_t st) {
  const int lanes = (a.head_dim / E + 1) / 2;
  // By the warps that units of four heads make on an SM. Measured (q + k heads,
  // columns, type; us for one head per unit / four / four streamed):
  //   below 8:  256 tokens of 32 + 8, 128, bf16 (4.3 warps): 3.0 / 3.5 / 3.6
  //   8 to 24: 1024 tokens of 32 + 8, 128, bf16 (17): 7.3 / 6.3 / 6.3;
  //            2048 tokens of 12 + 3, 80, f16 (9): 5.1 / 4.8 / 5.6
  //   above:   4096 tokens of 32 + 8, 128, bf16 (69): 28.9 / 21.2 / 18.5;
  //            65536: 425 / 289 / 214
  // A few tokens want every SM at work, four heads share the table columns and
  // the division of the token index, the stream keeps more loads in flight.
  const int64_t warps4 = head_warps4(a, E);
  if (head_streams(a, E)) return launch_stream<T, E, PAIRS, NORM, 4, 3, AXES>(a, lanes, st);
  if (warps4 >= static_cast<int64_t>(num_sms()) * 8) return launch_units<T, E, PAIRS, NORM, 4, AXES>(a, lanes, st);
  return launch_units<T, E, PAIRS, NORM, 1, AXES>(a, lanes, st);
}

template <typename T, int E, bool AXES>
cudaError_t launch_elems(const HeadArgs& a, cudaStream_t st) {
  if (a.pairs) return a.norm ? launch_form<T, E, true, true, AXES>(a, st) : launch_form<T, E, true, false, AXES>(a, st);
  return a.norm ? launch_form<T, E, false, true, AXES>(a, st) : launch_form<T, E, false, false, AXES>(a, st);
}

template <typename T, bool AXES>
cudaError_t launch_type(const HeadArgs& a, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const int e = head_vector_elems(a, false);
  if (e == E) return launch_elems<T, E, AXES>(a, st);
  if (e == E / 2) return launch_elems<T, E / 2, AXES>(a, st);
  const int64_t rows = a.batch * a.seq * (a.q.heads + a.k.heads);
  const int64_t blocks = std::min<int64_t>((rows + 7) / 8, static_cast<int64_t>(num_sms()) * 64);
  note_launch();
  return launch_dependent(qk_rope_any_kernel<T, AXES>, static_cast<int>(blocks), 256, st, a, rows, error_word_ptr());
}

template <bool AXES>
cudaError_t launch_rope(const HeadArgs& a, cudaStream_t st) {
  if (a.dtype == F16) return launch_type<__half, AXES>(a, st);
  if (a.dtype == BF16) return launch_type<__nv_bfloat16, AXES>(a, st);
  return launch_type<float, AXES>(a, st);
}
}  // namespace

}  // namespace tfo
