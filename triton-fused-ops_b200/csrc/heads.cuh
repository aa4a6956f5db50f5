// Shared by the kernels that work on single heads (qk_rope.cu,
// qk_rope_backward.cu): how a head's columns are spread over lanes, the
// rotary table rows, and the lookup of a token's position.
//
// A head of D columns is E-element vectors (16 or 8 bytes). L = half of them
// (rounded up) lanes hold two each, va and vb, chosen so that every rotated
// pair lies in one lane (no lane exchanges values for the rotation) and the
// lanes' va, and their vb, lie next to each other (whole 32-byte sectors):
//   half layout (column i pairs with i + R/2), h = R / (2E) vector pairs:
//     lane p <  h: va = p,             vb = p + h
//     lane p >= h: va = 2h + (p - h),  vb = va + (L - h)     (not rotated)
//   pair layout (column 2i pairs with 2i + 1): va = p, vb = p + L.
#pragma once

#include "capi_internal.h"
#include "common.cuh"

namespace tfo {

// ---- E elements of T as one register vector ------------------------------
template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };

template <typename T> struct Pair16;
template <> struct Pair16<__half> {
  __device__ static float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  __device__ static uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Pair16<__nv_bfloat16> {
  __device__ static float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ static uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename T, int E> struct HeadVec {
  static constexpr int kBytes = E * static_cast<int>(sizeof(T));
  static constexpr int kWords = kBytes / 4;
  using Raw = typename RawVec<kBytes>::type;
  __device__ static Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ static Raw zero() {
    Raw r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    return r;
  }
  __device__ static void unpack(const Raw& r, F2 (&f)[E / 2]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = f2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      } else {
        const float2 p = Pair16<T>::unpack(w[i]);
        f[i] = f2(p.x, p.y);
      }
    }
  }
  __device__ static void store(T* p, const F2 (&f)[E / 2]) {
    Raw r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(f[i].x);
        w[2 * i + 1] = __float_as_uint(f[i].y);
      } else {
        w[i] = Pair16<T>::pack(f[i].x, f[i].y);
      }
    }
    *reinterpret_cast<Raw*>(p) = r;
  }
};

// E floats from an array of run-time dtype; `p` + i must be E-vector aligned
// for that dtype (checked on the host).
template <int E>
__device__ __forceinline__ void load_floats(const void* p, int64_t i, int dtype, float (&f)[E]) {
  if constexpr (E == 1) {
    f[0] = load_as_float(p, i, dtype);
  } else if (dtype == F32) {
    const float* q = reinterpret_cast<const float*>(p) + i;
    constexpr int V = E >= 4 ? 4 : 2;
#pragma unroll
    for (int j = 0; j < E; j += V) {
      F2 t[V / 2];
      HeadVec<float, V>::unpack(HeadVec<float, V>::load(q + j), t);
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        f[j + 2 * k] = t[k].x;
        f[j + 2 * k + 1] = t[k].y;
      }
    }
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + i;
    uint32_t w[(E + 1) / 2];
    if constexpr (E == 8) {
      *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(q);
    } else if constexpr (E == 4) {
      *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(q);
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(q);
    }
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      const float2 v = dtype == F16 ? Pair16<__half>::unpack(w[j]) : Pair16<__nv_bfloat16>::unpack(w[j]);
      f[2 * j] = v.x;
      f[2 * j + 1] = v.y;
    }
  }
}

// ---- where a lane's columns lie -------------------------------------------
struct LaneCols {
  int va, vb;        // vector indexes in the head, or -1
  bool rot_a, rot_b;  // whether they are rotated (half layout: both or none)
};
template <bool PAIRS>
__device__ __forceinline__ LaneCols lane_cols(int p, int lanes, int nvec, int rot_vecs) {
  LaneCols c;
  if constexpr (PAIRS) {
    c.va = p;
    c.vb = p + lanes;
    c.rot_a = c.va < rot_vecs;
    c.rot_b = c.vb < rot_vecs;
  } else {
    const int h = rot_vecs >> 1;
    c.va = p < h ? p : h + p;
    c.vb = p < h ? p + h : c.va + lanes - h;
    c.rot_a = c.rot_b = p < h;
  }
  if (c.va >= nvec) c.va = -1;
  if (c.vb >= nvec) c.vb = -1;
  return c;
}

// ---- a token's table row ----------------------------------------------------
// The position of token (b, s): given, or s itself. A given position outside
// the table is recorded in the device error word and returned as -1 (its
// rotated columns become NaN; the table is not read).
__device__ __forceinline__ int64_t token_position(const HeadTables& t, int64_t b, int64_t s, uint32_t* err, bool report) {
  int64_t pos = s;
  if (t.pos_dtype == POS_I64) {
    pos = reinterpret_cast<const int64_t*>(t.positions)[b * t.pos_stride_batch + s * t.pos_stride_seq];
  } else if (t.pos_dtype == POS_I32) {
    pos = reinterpret_cast<const int32_t*>(t.positions)[b * t.pos_stride_batch + s * t.pos_stride_seq];
  }
  if (pos < 0 || pos >= t.rows) {
    if (report) set_error(err, ERR_BAD_POSITION);
    pos = -1;
  }
  return pos;
}

// cos and signed sin of a lane's pairs: of its E pairs (half layout), or of
// va's E/2 pairs and then vb's (pair layout). Entries of pairs that are not
// rotated stay unset and are not used.
template <int E, bool PAIRS>
__device__ __forceinline__ void lane_table(const HeadTables& t, int64_t pos, const LaneCols& col, bool inverse, float (&c)[E],
                                           float (&s)[E]) {
  if (pos < 0) {
#pragma unroll
    for (int j = 0; j < E; ++j) c[j] = s[j] = __int_as_float(0x7fffffff);
    return;
  }
  const int64_t row = pos * t.row_stride;
  if constexpr (PAIRS) {
    constexpr int H = E / 2;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      if (v == 0 ? !col.rot_a : !col.rot_b) continue;
      float x[H], y[H];
      const int64_t at = row + (v == 0 ? col.va : col.vb) * H;
      load_floats<H>(t.cos, at, t.dtype, x);
      load_floats<H>(t.sin, at, t.dtype, y);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        c[v * H + j] = x[j];
        s[v * H + j] = y[j];
      }
    }
  } else if (col.rot_a) {
    load_floats<E>(t.cos, row + col.va * E, t.dtype, c);
    load_floats<E>(t.sin, row + col.va * E, t.dtype, s);
  }
  if (inverse) {
#pragma unroll
    for (int j = 0; j < E; ++j) s[j] = -s[j];
  }
}

// A lane's rotation with weights: (u, v) -> (u wu c - v wv s, u wu s + v wv c)
// as one product and one multiply-add per output on packed pairs of columns,
// out = own * p + partner * q, where the partner of vector a is vector b (half
// layout) or the pair's other column (pair layout). Where nothing is rotated
// only p = w is used (a product with a zero q would turn a neighbour's
// infinity into NaN).
template <int E, bool PAIRS>
struct WeightedRotation {
  F2 pa[E / 2], qa[E / 2], pb[E / 2], qb[E / 2];
  __device__ void set(const float (&c)[E], const float (&s)[E], const float (&wa)[E], const float (&wb)[E],
                      const LaneCols& col) {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      const int i = 2 * j;
      pa[j] = f2(wa[i], wa[i + 1]);
      pb[j] = f2(wb[i], wb[i + 1]);
      if constexpr (PAIRS) {
        if (col.rot_a) {
          pa[j] = f2(wa[i] * c[j], wa[i + 1] * c[j]);
          qa[j] = f2(-wa[i + 1] * s[j], wa[i] * s[j]);
        }
        if (col.rot_b) {
          pb[j] = f2(wb[i] * c[E / 2 + j], wb[i + 1] * c[E / 2 + j]);
          qb[j] = f2(-wb[i + 1] * s[E / 2 + j], wb[i] * s[E / 2 + j]);
        }
      } else if (col.rot_a) {
        const F2 c2 = f2(c[i], c[i + 1]), s2 = f2(s[i], s[i + 1]);
        qa[j] = mul2(pb[j], f2(-s[i], -s[i + 1]));
        qb[j] = mul2(pa[j], s2);
        pa[j] = mul2(pa[j], c2);
        pb[j] = mul2(pb[j], c2);
      }
    }
  }
  __device__ void apply(F2 (&a)[E / 2], F2 (&b)[E / 2], const LaneCols& col) const {
    if constexpr (PAIRS) {
      one(a, pa, qa, col.rot_a);
      one(b, pb, qb, col.rot_b);
    } else if (col.rot_a) {
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const F2 u = a[j];
        a[j] = fma2(b[j], qa[j], mul2(u, pa[j]));
        b[j] = fma2(u, qb[j], mul2(b[j], pb[j]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        a[j] = mul2(a[j], pa[j]);
        b[j] = mul2(b[j], pb[j]);
      }
    }
  }

 private:
  __device__ static void one(F2 (&v)[E / 2], const F2 (&p)[E / 2], const F2 (&q)[E / 2], bool rotated) {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      const F2 u = v[j];
      v[j] = mul2(u, p[j]);
      if (rotated) v[j] = fma2(f2(u.y, u.x), q[j], v[j]);
    }
  }
};

// A lane's rotation without weights; columns that are not rotated are left as they are.
template <int E, bool PAIRS>
struct PlainRotation {
  F2 c[E / 2], s[E / 2];
  __device__ void set(const float (&cv)[E], const float (&sv)[E]) {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      c[j] = f2(cv[2 * j], cv[2 * j + 1]);
      s[j] = f2(sv[2 * j], sv[2 * j + 1]);
    }
  }
  __device__ void apply(F2 (&a)[E / 2], F2 (&b)[E / 2], const LaneCols& col) const {
    if constexpr (PAIRS) {
      if (col.rot_a) one(a, 0);
      if (col.rot_b) one(b, E / 2);
    } else if (col.rot_a) {
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const F2 u = a[j], vs = mul2(b[j], s[j]);
        a[j] = fma2(u, c[j], f2(-vs.x, -vs.y));
        b[j] = fma2(u, s[j], mul2(b[j], c[j]));
      }
    }
  }

 private:
  __device__ void one(F2 (&v)[E / 2], int at) const {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      const float cj = (at + j) % 2 ? c[(at + j) / 2].y : c[(at + j) / 2].x;
      const float sj = (at + j) % 2 ? s[(at + j) / 2].y : s[(at + j) / 2].x;
      const F2 u = v[j];
      v[j] = f2(u.x * cj - u.y * sj, u.x * sj + u.y * cj);
    }
  }
};

// n / d for n < 2^31 by one wide multiplication (host-made constants).
struct FastDiv {
  uint32_t m;
  int shift;
  __host__ static FastDiv make(uint32_t d) {
    int s = 0;
    while ((1ull << s) < d) ++s;
    return FastDiv{static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), 31 + s};
  }
  __device__ uint32_t div(uint32_t n) const { return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> shift); }
};

// ---- lane groups ----------------------------------------------------------
// A head takes L = ceil(vectors / 2) neighbouring lanes; a warp holds 32 / L
// such groups, and what lanes are left over idle (they take part in shuffles).
// L need not be a power of two: heads of 80 columns fill 30 of 32 lanes.
struct LaneGroup {
  int lanes;  // L
  int p;      // this lane's place in its group
  int base;   // first lane of the group
  int group;  // of the warp
  bool spare;
  __device__ explicit LaneGroup(int l) : lanes(l) {
    const int lane = threadIdx.x & 31;
    group = lane / l;
    spare = group >= 32 / l;
    if (spare) group = 0;
    base = group * l;
    p = spare ? 0 : lane - base;
  }
  template <int O> __device__ static float xor_add(float v) { return v + __shfl_xor_sync(0xffffffffu, v, O); }
  // Sum over the group's lanes, the same bits in each of them: a tree for 4, 8 and
  // 16 lanes, else (1 to 32, the widest heads) a shuffle for each.
  __device__ float sum(float v) const {
    if (lanes == 8) return xor_add<1>(xor_add<2>(xor_add<4>(v)));
    if (lanes == 16) return xor_add<1>(xor_add<2>(xor_add<4>(xor_add<8>(v))));
    if (lanes == 4) return xor_add<1>(xor_add<2>(v));
    float t = 0.f;
    for (int i = 0; i < lanes; ++i) t += __shfl_sync(0xffffffffu, v, base + i);
    return t;
  }
  // Sums side by side: their shuffles overlap.
  template <int O, int N> __device__ static void xor_add(float (&v)[N]) {
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = __shfl_xor_sync(0xffffffffu, v[i], O);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += o[i];
  }
  template <int N> __device__ void sum(float (&v)[N]) const {
    if (lanes == 8 || lanes == 16 || lanes == 4) {
      if (lanes == 16) xor_add<8>(v);
      if (lanes >= 8) xor_add<4>(v);
      xor_add<2>(v);
      xor_add<1>(v);
    } else {
      float t[N] = {};
      for (int i = 0; i < lanes; ++i) {
#pragma unroll
        for (int k = 0; k < N; ++k) t[k] += __shfl_sync(0xffffffffu, v[k], base + i);
      }
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = t[k];
    }
  }
};

// CTAs [0, q_ctas) of a streaming launch take the queries, the rest the keys.
struct SideSplit {
  int q_ctas, k_ctas;
};

// ---- a lane group's stream of heads ------------------------------------------
// A lane group takes "units" of NH neighbouring heads of one token, a fixed
// step apart, so that the groups of a launch read neighbouring memory at a
// time. Each lane copies its own vectors of the units ahead into a ring in
// shared memory with cp.async and later reads them back itself: the loads in
// flight cost no registers, need no barrier and do not depend on occupancy. IN
// tensors of the same shape are streamed side by side. Lanes without columns
// keep zeros.
template <typename T, int E, int NH, int STAGES, int IN, bool FULL>
struct HeadStream {
  using V = HeadVec<T, E>;
  using Raw = typename V::Raw;
  static constexpr int kThreads = 256;
  static constexpr size_t kSmemBytes = static_cast<size_t>(STAGES) * IN * NH * 2 * kThreads * sizeof(Raw);

  struct Input {
    const T* x;  // at the lane's first vector
    int64_t stride_batch, stride_seq, stride_head;
  };
  Raw* ring;  // this thread's first slot
  Input in[IN];
  int vb_offset;  // elements from the lane's first vector to its second
  bool has_a, has_b;
  FastDiv by_seq, by_chunks;
  uint32_t seq, chunks, units, unit_step;
  int heads;
  uint32_t load_unit;  // the next unit to load, and its stage
  int load_stage;

  __device__ Raw* slot(int stage, int i, int h, int v) { return ring + (((stage * IN + i) * NH + h) * 2 + v) * kThreads; }

  // `first`, `step`: the group's units. Fills all stages but the last.
  __device__ void start(void* smem, uint32_t first, uint32_t step) {
    ring = reinterpret_cast<Raw*>(smem) + threadIdx.x;
    if (!FULL && !(has_a && has_b)) {
#pragma unroll 1
      for (int i = 0; i < STAGES * IN * NH * 2; ++i) ring[i * kThreads] = V::zero();
    }
    load_unit = first;
    unit_step = step;
    load_stage = 0;
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) load();
  }

  // Issues the loads of the next unit (nothing past the last) as one cp.async group.
  __device__ void load() {
    if (load_unit < units) {
      const uint32_t token = by_chunks.div(load_unit);
      const uint32_t b = by_seq.div(token);
      const uint32_t s = token - b * seq;
      const int h0 = static_cast<int>(load_unit - token * chunks) * NH;
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        const T* row = in[i].x + b * in[i].stride_batch + s * in[i].stride_seq + h0 * in[i].stride_head;
#pragma unroll
        for (int h = 0; h < NH; ++h, row += in[i].stride_head) {
          if (h0 + h >= heads) break;
          if (FULL || has_a) copy(slot(load_stage, i, h, 0), row);
          if (FULL || has_b) copy(slot(load_stage, i, h, 1), row + vb_offset);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    load_stage = load_stage + 1 == STAGES ? 0 : load_stage + 1;
    load_unit += unit_step;
  }

  // Waits for the oldest unit in flight.
  __device__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }

 private:
  __device__ static void copy(Raw* dst, const T* src) {
    if constexpr (sizeof(Raw) == 16) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    } else {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    }
  }
};

}  // namespace tfo
