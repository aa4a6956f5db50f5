// Shared by the kernels of the residual stream (residual_norm.cu,
// residual_norm_backward.cu): how a row is spread over threads, the stream of
// rows through shared memory, sums over a row, and the parameters' columns.
//
// A row of `hidden` columns is chunks of E columns (16 bytes of x, or one
// column where rows are not whole aligned 16-byte vectors). T threads (whole
// warps) take a row, thread t its chunks t, t + T, ... (V of them): a group.
// A CTA holds several groups when rows are short, each with rows of its own
// and a named barrier for its sums.
#pragma once

#include "heads.cuh"
#include "philox.cuh"

namespace tfo {

constexpr int kRowThreads = 512;   // most threads of a CTA
constexpr int kMaxRowWarps = 16;   // of a group

// How a launch spreads the rows.
struct RowPlan {
  int threads;  // T
  int groups;   // of a CTA
};

// ---- sums over a row --------------------------------------------------------
// Sums over a group's threads, the same bits in each. `red`: this group's
// kMaxRowWarps * N floats, the parts of warps that are not there zero; two
// sums in a row must use different ones.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int warps, int warp, int barrier) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    float w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = __shfl_xor_sync(0xffffffffu, v[j], o);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += w[j];
  }
  if (warps == 1) return;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) red[j * kMaxRowWarps + warp] = v[j];
  }
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float4 s = *reinterpret_cast<const float4*>(red + j * kMaxRowWarps);
#pragma unroll
    for (int i = 4; i < kMaxRowWarps; i += 4) {
      const float4 p = *reinterpret_cast<const float4*>(red + j * kMaxRowWarps + i);
      s.x += p.x, s.y += p.y, s.z += p.z, s.w += p.w;
    }
    v[j] = (s.x + s.y) + (s.z + s.w);
  }
}

// ---- chunks -----------------------------------------------------------------
// E columns of T as pairs of floats at `f`, from and to memory (E == 1: half a pair).
template <typename T, int E> struct Chunk {
  static constexpr int kVecs = E * static_cast<int>(sizeof(T)) / 16;  // 16-byte vectors
  static_assert(E % (16 / static_cast<int>(sizeof(T))) == 0, "whole vectors");
  __device__ static void unpack(const uint4 (&r)[kVecs], F2* f) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const uint32_t w[4] = {r[v].x, r[v].y, r[v].z, r[v].w};
      if constexpr (sizeof(T) == 4) {
        f[2 * v] = f2(__uint_as_float(w[0]), __uint_as_float(w[1]));
        f[2 * v + 1] = f2(__uint_as_float(w[2]), __uint_as_float(w[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 p = Pair16<T>::unpack(w[i]);
          f[4 * v + i] = f2(p.x, p.y);
        }
      }
    }
  }
  __device__ static void store(T* p, const F2* f) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      uint4 r;
      if constexpr (sizeof(T) == 4) {
        r = make_uint4(__float_as_uint(f[2 * v].x), __float_as_uint(f[2 * v].y), __float_as_uint(f[2 * v + 1].x),
                       __float_as_uint(f[2 * v + 1].y));
      } else {
        r = make_uint4(Pair16<T>::pack(f[4 * v].x, f[4 * v].y), Pair16<T>::pack(f[4 * v + 1].x, f[4 * v + 1].y),
                       Pair16<T>::pack(f[4 * v + 2].x, f[4 * v + 2].y), Pair16<T>::pack(f[4 * v + 3].x, f[4 * v + 3].y));
      }
      reinterpret_cast<uint4*>(p)[v] = r;
    }
  }
};

__device__ __forceinline__ float& lane_of(F2* f, int i) { return i & 1 ? f[i >> 1].y : f[i >> 1].x; }

// Which columns this thread takes.
template <int E, int V> struct RowCols {
  static constexpr int N = E * V;        // columns
  static constexpr int P = (N + 1) / 2;  // pairs of them
  static_assert(E > 1 || V % 2 == 0, "whole pairs");
  int first, step, hidden;
  __device__ RowCols(int t, int threads, int h) : first(t * E), step(threads * E), hidden(h) {}
  __device__ int col(int k) const { return first + k * step; }
  __device__ bool has(int k) const { return col(k) < hidden; }

  // p's columns of a sequence (otherwise: of a parameter that is not there, and past the row).
  __device__ void param(const RowParam& p, int64_t seq, float otherwise, F2 (&f)[P]) const {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = otherwise;
      if (p.p != nullptr && has(k)) load_floats<E>(p.p, seq * p.seq_stride + col(k), p.dtype, v);
#pragma unroll
      for (int j = 0; j < E; ++j) lane_of(f, k * E + j) = v[j];
    }
  }
  template <typename T> __device__ void store(T* row, F2 (&f)[P]) const {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (!has(k)) continue;
      if constexpr (E == 1) row[col(k)] = Ty<T>::from_f(lane_of(f, k));
      else Chunk<T, E>::store(row + col(k), f + k * E / 2);
    }
  }
  // Which of this thread's columns of row r are kept.
  __device__ uint32_t kept(const DropoutArgs& d, const DropKey& key, int64_t r) const {
    if (d.all) return 0u;
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (has(k)) bits |= key.kept<E>(static_cast<uint64_t>(r * hidden + col(k))) << (k * E);
    return bits;
  }
  __device__ static void drop(uint32_t bits, F2 (&f)[P]) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (!(bits >> (2 * j) & 1)) f[j].x = 0.f;
      if (!(bits >> (2 * j + 1) & 1)) f[j].y = 0.f;
    }
  }
};

// ---- a group's stream of rows -----------------------------------------------
// A thread's chunks of the rows ahead, of NX tensors of TX and NR of TR. Whole
// 16-byte vectors (E > 1) go through a ring in shared memory by cp.async, each
// thread writing and reading its own slots: no barrier, and the loads in flight
// cost no registers. Single columns (E == 1) are held in registers, a row ahead.
template <typename TX, typename TR, int E, int V, int NX, int NR, int STAGES>
struct RowStream {
  static constexpr int kTensors = NX + NR;
  static constexpr int kVecsX = E == 1 ? 0 : Chunk<TX, E == 1 ? 16 : E>::kVecs;
  static constexpr int kVecsR = E == 1 ? 0 : Chunk<TR, E == 1 ? 16 : E>::kVecs;
  static constexpr int kVecsRow = V * (NX * kVecsX + NR * kVecsR);  // of a thread and row
  static constexpr size_t smem_bytes(int threads) { return static_cast<size_t>(STAGES) * kVecsRow * threads * 16; }

  const void* base[kTensors];  // NULL: zeros
  int64_t stride[kTensors];    // elements between rows
  uint4* ring;                 // this thread's first slot
  int slots;                   // threads of the CTA: distance of a thread's slots
  int64_t next, end;
  int load_stage, stage;
  float ahead[E == 1 ? kTensors * V : 1], now[E == 1 ? kTensors * V : 1];

  __device__ uint4* slot(int st, int v) const { return ring + (st * kVecsRow + v) * slots; }
  static __device__ constexpr int first_vec(int i) { return i < NX ? i * V * kVecsX : NX * V * kVecsX + (i - NX) * V * kVecsR; }

  __device__ void start(const RowCols<E, V>& cols, uint4* smem, int64_t r0, int64_t r1) {
    next = r0;
    end = r1;
    load_stage = 0;
    stage = STAGES - 1;
    if constexpr (E > 1) {
      ring = smem + threadIdx.x;
      slots = blockDim.x;
      // what no copy ever fills stays zero
      bool full = cols.has(V - 1);
#pragma unroll
      for (int i = 0; i < kTensors; ++i) full = full && base[i] != nullptr;
      if (!full) {
#pragma unroll 1
        for (int i = 0; i < STAGES * kVecsRow; ++i) ring[i * slots] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll 1
      for (int i = 0; i < STAGES - 1; ++i) load(cols);
    } else {
      load(cols);
    }
  }
  // The next row: its values are there for get(), and the loads of a later one are under way.
  __device__ void advance(const RowCols<E, V>& cols) {
    if constexpr (E > 1) {
      load(cols);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < kTensors * V; ++i) now[i] = ahead[i];
      load(cols);
    }
  }
  template <int I> __device__ void get(F2 (&f)[RowCols<E, V>::P]) const {
    using T = std::conditional_t<(I < NX), TX, TR>;
    if constexpr (E > 1) {
      constexpr int n = Chunk<T, E>::kVecs;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        uint4 r[n];
#pragma unroll
        for (int v = 0; v < n; ++v) r[v] = *slot(stage, first_vec(I) + k * n + v);
        Chunk<T, E>::unpack(r, f + k * E / 2);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) lane_of(f, k) = now[I * V + k];
    }
  }

 private:
  __device__ void load(const RowCols<E, V>& cols) {
    if (next < end) {
#pragma unroll
      for (int i = 0; i < kTensors; ++i) {
        if (base[i] == nullptr) {
          if constexpr (E == 1) {
#pragma unroll
            for (int k = 0; k < V; ++k) ahead[i * V + k] = 0.f;
          }
          continue;
        }
        if (i < NX) copy<TX, kVecsX>(cols, i);
        else copy<TR, kVecsR>(cols, i);
      }
    }
    ++next;
    if constexpr (E > 1) {
      load_stage = load_stage + 1 == STAGES ? 0 : load_stage + 1;
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  template <typename T, int VECS> __device__ void copy(const RowCols<E, V>& cols, int i) {
    const T* row = static_cast<const T*>(base[i]) + next * stride[i];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if constexpr (E == 1) {
        ahead[i * V + k] = cols.has(k) ? Ty<T>::to_f(row[cols.col(k)]) : 0.f;
      } else if (cols.has(k)) {
#pragma unroll
        for (int v = 0; v < VECS; ++v)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           smem_u32(slot(load_stage, first_vec(i) + k * VECS + v))),
                       "l"(reinterpret_cast<const uint4*>(row + cols.col(k)) + v)
                       : "memory");
      }
    }
  }
};

// ---- host: which rows are whole aligned vectors ------------------------------
inline int row_elem_bytes(int dtype) { return dtype == F32 ? 4 : 2; }
inline bool row_aligned(const void* p, int64_t stride, int64_t rows, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || stride * row_elem_bytes(dtype) % 16 == 0);
}
// Columns of a chunk with which the vector kernels can take these rows: 16 bytes of x, or 1.
inline int row_chunk(const ResidualArgs& a, bool backward) {
  const int e = 16 / row_elem_bytes(a.x_dtype);
  bool ok = a.hidden % e == 0;
  const int64_t h = a.hidden;
  ok = ok && row_aligned(a.x, a.x_stride, a.rows, a.x_dtype) && row_aligned(a.res, a.res_stride, a.rows, a.res_dtype);
  if (backward) {
    ok = ok && row_aligned(a.dy, a.dy_stride, a.rows, a.x_dtype) && row_aligned(a.dh, a.dh_stride, a.rows, a.res_dtype);
    ok = ok && row_aligned(a.dx, h, a.rows, a.x_dtype) && row_aligned(a.dres, h, a.rows, a.res_dtype);
  } else {
    ok = ok && row_aligned(a.h, h, a.rows, a.res_dtype) && row_aligned(a.y, h, a.rows, a.x_dtype);
  }
  for (const RowParam* p : {&a.branch_weight, &a.gate, &a.weight, &a.shift})
    ok = ok && (p->p == nullptr || (reinterpret_cast<uintptr_t>(p->p) % 16 == 0 &&
                                    p->seq_stride * row_elem_bytes(p->dtype) % std::min(16, e * row_elem_bytes(p->dtype)) == 0));
  return ok ? e : 1;
}
// T for V chunks of E columns a thread (0: the row does not fit).
inline int row_threads(int hidden, int e, int v) {
  const int64_t need = (static_cast<int64_t>(hidden) + e * v - 1) / (e * v);
  const int64_t t = (need + 31) / 32 * 32;
  return t <= kRowThreads ? static_cast<int>(t) : 0;
}

}  // namespace tfo
