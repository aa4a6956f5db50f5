// The rotation of query and key heads at one position for each token (qk_rope.cuh).
#include "qk_rope.cuh"

namespace tfo {

namespace {
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }

// Every vector of `bytes` bytes of a strided [batch, seq, heads, D] tensor is aligned.
bool rows_aligned(const void* x, const HeadArgs& a, int heads, int64_t sb, int64_t ss, int64_t sh, int esz, int bytes) {
  return aligned(x, bytes) && (a.batch <= 1 || sb * esz % bytes == 0) && (a.seq <= 1 || ss * esz % bytes == 0) &&
         (heads <= 1 || sh * esz % bytes == 0);
}
}  // namespace

bool head_vectors_fit(const HeadArgs& a, int e) {
  if (a.batch * a.seq * (a.q.heads + a.k.heads) >= (1ll << 31) - (1 << 20)) return false;  // units are counted in 32 bits
  return a.head_dim % e == 0 && a.head_dim / e <= 64 && (a.pairs ? a.rotary_dim : a.rotary_dim / 2) % e == 0;
}

int head_vector_elems(const HeadArgs& a, bool backward) {
  const int esz = a.dtype == F32 ? 4 : 2;
  for (int bytes = 16; bytes >= 8; bytes /= 2) {
    const int e = bytes / esz;
    if (!head_vectors_fit(a, e)) continue;
    const int tsz = a.t.dtype == F32 ? 4 : 2;
    const int tb = std::min(16, (a.pairs ? e / 2 : e) * tsz);
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

bool head_streams(const HeadArgs& a, int elems) { return head_warps4(a, elems) >= static_cast<int64_t>(num_sms()) * 24; }

cudaError_t qk_rope_launch(const HeadArgs& a, cudaStream_t st) {
  return a.t.axes > 1 ? qk_rope_axes_launch(a, st) : launch_rope<false>(a, st);
}

}  // namespace tfo
