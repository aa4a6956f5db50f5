// Shared by the kernels that work on single heads (qk_rope.cu,
// qk_rope_backward.cu): how a head's columns are spread over lanes, the
// rotary table rows, and the lookup of a token's position.
//
// A head of D columns is E-element vectors (16 or 8 bytes). Each lane holds
// two of them, va and vb, chosen so that every rotated pair lies in one lane
// and no lane exchanges values for the rotation:
//   half layout (column i pairs with i + R/2), h = R / (2E) vector pairs:
//     lane p <  h: va = p,                vb = p + h
//     lane p >= h: va = 2h + 2(p - h),    vb = va + 1     (not rotated)
//   pair layout (column 2i pairs with 2i + 1): va = 2p, vb = 2p + 1.
// In both layouts lane p uses the table columns [p*E, p*E + E).
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
  __device__ static void unpack(const Raw& r, float (&f)[E]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 p = Pair16<T>::unpack(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    }
  }
  __device__ static void store(T* p, const float (&f)[E]) {
    Raw r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(f[i]);
      } else {
        w[i] = Pair16<T>::pack(f[2 * i], f[2 * i + 1]);
      }
    }
    *reinterpret_cast<Raw*>(p) = r;
  }
};

// E floats from an array of run-time dtype; `p` + i must be E-vector aligned
// for that dtype (checked on the host).
template <int E>
__device__ __forceinline__ void load_floats(const void* p, int64_t i, int dtype, float (&f)[E]) {
  if (dtype == F32) {
    const float* q = reinterpret_cast<const float*>(p) + i;
    constexpr int V = E >= 4 ? 4 : 2;
#pragma unroll
    for (int j = 0; j < E; j += V) {
      float t[V];
      HeadVec<float, V>::unpack(HeadVec<float, V>::load(q + j), t);
#pragma unroll
      for (int k = 0; k < V; ++k) f[j + k] = t[k];
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
  int va, vb;      // vector indexes in the head, or -1
  int rotated;     // of the lane's two vectors' pairs: 0 none, 1 va only (pair layout), 2 both
};
template <bool PAIRS>
__device__ __forceinline__ LaneCols lane_cols(int p, int nvec, int rot_vecs) {
  LaneCols c;
  if constexpr (PAIRS) {
    c.va = 2 * p;
    c.vb = 2 * p + 1;
    c.rotated = min(2, max(0, rot_vecs - 2 * p));
  } else {
    const int h = rot_vecs >> 1;
    c.va = p < h ? p : 2 * p;
    c.vb = p < h ? p + h : 2 * p + 1;
    c.rotated = p < h ? 2 : 0;
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

// cos and signed sin of a lane's table columns. Entries of pairs that are not
// rotated stay unset: rotate_lane() does not use them.
template <int E>
__device__ __forceinline__ void lane_table(const HeadTables& t, int64_t pos, int p, int rotated, bool inverse,
                                           float (&c)[E], float (&s)[E]) {
  if (pos < 0) {
#pragma unroll
    for (int j = 0; j < E; ++j) c[j] = s[j] = __int_as_float(0x7fffffff);
    return;
  }
  const int64_t at = pos * t.row_stride + p * E;
  if (rotated == 2) {
    load_floats<E>(t.cos, at, t.dtype, c);
    load_floats<E>(t.sin, at, t.dtype, s);
  } else if (rotated == 1) {  // the first of the pair layout's two vectors: half the columns
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      c[j] = load_as_float(t.cos, at + j, t.dtype);
      s[j] = load_as_float(t.sin, at + j, t.dtype);
    }
  }
  if (inverse) {
#pragma unroll
    for (int j = 0; j < E; ++j) s[j] = -s[j];
  }
}

// Rotates a lane's two vectors in place: (u, v) -> (u c - v s, u s + v c) for
// each pair. Columns that are not rotated are left as they are (a product with
// cos = 1 and sin = 0 would turn a neighbour's infinity into NaN).
template <int E, bool PAIRS>
__device__ __forceinline__ void rotate_lane(float (&a)[E], float (&b)[E], const float (&c)[E], const float (&s)[E],
                                            int rotated) {
  if (rotated == 0) return;
  if constexpr (PAIRS) {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      const float u = a[2 * j], v = a[2 * j + 1];
      a[2 * j] = u * c[j] - v * s[j];
      a[2 * j + 1] = u * s[j] + v * c[j];
    }
    if (rotated == 2) {
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const float u = b[2 * j], v = b[2 * j + 1];
        b[2 * j] = u * c[E / 2 + j] - v * s[E / 2 + j];
        b[2 * j + 1] = u * s[E / 2 + j] + v * c[E / 2 + j];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float u = a[j], v = b[j];
      a[j] = u * c[j] - v * s[j];
      b[j] = u * s[j] + v * c[j];
    }
  }
}

// Sum over the `lanes` (a power of two) lanes of a head's group.
__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace tfo
