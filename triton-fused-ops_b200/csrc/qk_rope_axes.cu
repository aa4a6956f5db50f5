// The rotation of query and key heads at positions of several axes (qk_rope.cuh).
//
// A lane whose columns all turn by one axis reads its vector of that axis' row,
// as it does for one position. Where a vector's columns belong to several axes
// (axes that take turns, sections that are no multiple of a vector) it would
// read them one by one, for every unit of heads again. With enough tokens their
// rows are therefore joined first, a small part of the heads' bytes, and the
// rotation is that of one position (8192 tokens of 32 + 8 heads of 128, bf16,
// axes taking turns: 39 instead of 62 us with the norm, its gradients 64 of 132).
#include "qk_rope.cuh"

namespace tfo {

// Each token's row: pair i's entry of the row at its axis' position.
template <typename T>
__global__ void __launch_bounds__(256) join_axes_kernel(const __grid_constant__ HeadTables t, int64_t tokens, FastDiv by_seq, uint32_t seq,
                                                        int pairs, FastDiv by_pairs, T* __restrict__ cos, T* __restrict__ sin,
                                                        uint32_t* err) {
  griddep_launch_dependents();
  griddep_wait();
  const uint32_t per_cta = 256u / pairs > 0 ? 256u / pairs : 1u;  // tokens at a time
  const uint32_t in = by_pairs.div(threadIdx.x);
  const T nan = Ty<T>::from_f(__int_as_float(0x7fffffff));
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * per_cta; first < tokens; first += static_cast<int64_t>(gridDim.x) * per_cta) {
    const int64_t token = first + (pairs < 256 ? in : 0u);
    if (pairs < 256 && (in >= per_cta || token >= tokens)) continue;
    const uint32_t b = by_seq.div(static_cast<uint32_t>(token)), s = static_cast<uint32_t>(token) - b * seq;
    for (int i = pairs < 256 ? threadIdx.x - in * pairs : threadIdx.x; i < pairs; i += 256) {
      const int64_t pos = axis_position(t, b, s, LaneAxes::of(t, i), err);
      const int64_t at = pos * t.row_stride + i;
      cos[token * pairs + i] = pos < 0 ? nan : static_cast<const T*>(t.cos)[at];
      sin[token * pairs + i] = pos < 0 ? nan : static_cast<const T*>(t.sin)[at];
    }
  }
}

size_t axes_workspace_bytes(int64_t tokens, int pairs, int table_dtype) {
  const size_t row = static_cast<size_t>(tokens) * pairs * (table_dtype == F32 ? 4 : 2);
  return 2 * ((row + 15) / 16 * 16);
}

namespace {
// Whether a vector of a lane's columns holds pairs of several axes.
bool mixed(const HeadArgs& a, int elems) {
  const int pairs = a.rotary_dim / 2, of_vector = a.pairs ? elems / 2 : elems;
  auto axis = [&](int i) { return a.t.axis_bits[i / 16] >> (2 * (i % 16)) & 3u; };
  for (int i = 0; i < pairs; ++i)
    if (axis(i) != axis(i / of_vector * of_vector)) return true;
  return false;
}

// With vectors of `elems` elements: whether joining the rows is the faster way.
bool joins(const HeadArgs& a, int elems) {
  return a.batch * a.seq <= INT32_MAX /* tokens are 32-bit numbers there */ && head_streams(a, elems) && mixed(a, elems);
}

template <typename T>
cudaError_t join(const HeadArgs& a, void* cos, void* sin, cudaStream_t st) {
  const int pairs = a.rotary_dim / 2;
  const int64_t tokens = a.batch * a.seq, per_cta = std::max(1, 256 / pairs);
  note_launch();
  return launch_dependent(join_axes_kernel<T>, static_cast<int>(std::min<int64_t>((tokens + per_cta - 1) / per_cta, num_sms() * 16ll)),
                          256, st, a.t, tokens, FastDiv::make(static_cast<uint32_t>(a.seq)), static_cast<uint32_t>(a.seq), pairs,
                          FastDiv::make(static_cast<uint32_t>(pairs)), static_cast<T*>(cos), static_cast<T*>(sin), error_word_ptr());
}
}  // namespace

bool axes_may_join(const HeadArgs& a) {
  const int esz = a.dtype == F32 ? 4 : 2;
  for (const int elems : {16 / esz, 8 / esz})
    if (head_vectors_fit(a, elems) && joins(a, elems)) return true;
  return false;
}

cudaError_t join_axes(HeadArgs* a, bool backward, cudaStream_t st) {
  const int elems = head_vector_elems(*a, backward);
  if (a->t.joined == nullptr || elems == 0 || !joins(*a, elems)) return cudaSuccess;
  const int pairs = a->rotary_dim / 2;
  void* cos = a->t.joined;
  void* sin = static_cast<char*>(cos) + axes_workspace_bytes(a->batch * a->seq, pairs, a->t.dtype) / 2;
  const cudaError_t e = a->t.dtype == F32   ? join<float>(*a, cos, sin, st)
                        : a->t.dtype == F16 ? join<__half>(*a, cos, sin, st)
                                            : join<__nv_bfloat16>(*a, cos, sin, st);
  HeadTables t{};
  t.cos = cos;
  t.sin = sin;
  t.row_stride = pairs;
  t.rows = a->batch * a->seq;
  t.dtype = a->t.dtype;
  t.pos_stride_batch = a->seq;
  a->t = t;
  return e;
}

cudaError_t qk_rope_axes_launch(const HeadArgs& a, cudaStream_t st) {
  HeadArgs one = a;
  if (const cudaError_t e = join_axes(&one, false, st); e != cudaSuccess) return e;
  return one.t.axes > 1 ? launch_rope<true>(one, st) : qk_rope_launch(one, st);
}

}  // namespace tfo
