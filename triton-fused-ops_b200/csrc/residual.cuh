// Shared by the kernels of the residual stream (residual_norm.cu,
// residual_norm_backward.cu): how a row is spread over threads, the stream of
// rows through shared memory, sums over a row, and the parameters' columns.
//
// A row of `hidden` columns is chunks of E columns (16 bytes of the wider of x
// and the stream, or one column where rows are not whole aligned vectors). T threads (whole
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
//
// One value: a tree of shuffles, the warps' parts through shared memory, a tree
// again over as many lanes. Four values: each step of the tree also halves how
// many of them a lane carries, so that all four take 6 shuffles instead of 20
// and end in 8 lanes each (as after a reading of the parts), then one shuffle a value.
__device__ __forceinline__ float lanes_sum(float v, int from) {  // over the lanes that differ in bits below `from` * 2
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o <= from) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void row_sum(float (&v)[1], float* red, int warps, int warp, int barrier) {
  v[0] = lanes_sum(v[0], 16);
  if (warps == 1) return;
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[warp] = v[0];
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
  if (warps > 8) v[0] = lanes_sum(red[lane & 15], 8);
  else if (warps > 4) v[0] = lanes_sum(red[lane & 7], 4);
  else v[0] = lanes_sum(red[lane & 3], 2);
}
__device__ __forceinline__ void row_sum(float (&v)[4], float* red, int warps, int warp, int barrier) {
  const int lane = threadIdx.x & 31;
  const bool up = lane & 16, right = lane & 8;
  float a = up ? v[2] : v[0], b = up ? v[3] : v[1];
  a += __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16);
  b += __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 16);
  float mine = right ? b : a;
  mine += __shfl_xor_sync(0xffffffffu, right ? a : b, 8);
  mine = lanes_sum(mine, 4);  // of value lane / 8
  if (warps > 1) {
    if ((lane & 7) == 0) red[(lane >> 3) * kMaxRowWarps + warp] = mine;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
    const float2 p = *reinterpret_cast<const float2*>(red + (lane >> 3) * kMaxRowWarps + (lane & 7) * 2);
    mine = lanes_sum(p.x + p.y, 4);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __shfl_sync(0xffffffffu, mine, 8 * j);
}

// ---- chunks -----------------------------------------------------------------
// E columns of T as pairs of floats at `f`, from and to memory in vectors of 16 or 8 bytes.
template <typename T, int E> struct Chunk {
  static constexpr int kBytes = E * static_cast<int>(sizeof(T));
  static constexpr int kVecBytes = kBytes < 16 ? 8 : 16;
  static constexpr int kVecs = kBytes / kVecBytes;
  static_assert(kVecs * kVecBytes == kBytes, "whole vectors");
  static constexpr int kVecCols = E / kVecs;
  using Vec = HeadVec<T, kVecCols>;
  __device__ static void unpack(const typename Vec::Raw& r, F2* f) {
    F2 t[kVecCols / 2];
    Vec::unpack(r, t);
#pragma unroll
    for (int i = 0; i < kVecCols / 2; ++i) f[i] = t[i];
  }
  __device__ static void store(T* p, const F2* f) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      F2 t[kVecCols / 2];
#pragma unroll
      for (int i = 0; i < kVecCols / 2; ++i) t[i] = f[v * kVecCols / 2 + i];
      Vec::store(p + v * kVecCols, t);
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
    for (int k = 0; k < V; ++k) bits |= key.kept<E>(static_cast<uint64_t>(r * hidden + col(k))) << (k * E);
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
  using ChunkX = Chunk<TX, E == 1 ? 16 : E>;
  using ChunkR = Chunk<TR, E == 1 ? 16 : E>;
  static constexpr int kBytesX = V * ChunkX::kBytes, kBytesR = V * ChunkR::kBytes;  // of a thread and row
  static constexpr int kRowBytes = E == 1 ? 0 : NX * kBytesX + NR * kBytesR;
  static constexpr size_t smem_bytes(int threads) { return static_cast<size_t>(STAGES) * kRowBytes * threads; }

  const void* base[kTensors];  // NULL: zeros
  int64_t stride[kTensors];    // elements between rows
  uint32_t ring;               // shared memory
  uint32_t stage_bytes;
  int64_t next, end;
  int load_stage, stage;
  float ahead[E == 1 ? kTensors * V : 1], now[E == 1 ? kTensors * V : 1];

  // Vector v of tensor i in a stage: the CTA's threads side by side.
  template <int VEC_BYTES> __device__ uint32_t slot(int st, int i, int v) const {
    const int before = (i < NX ? i * kBytesX : NX * kBytesX + (i - NX) * kBytesR) + v * VEC_BYTES;
    return ring + st * stage_bytes + before * blockDim.x + threadIdx.x * VEC_BYTES;
  }

  __device__ void start(const RowCols<E, V>& cols, void* smem, int64_t r0, int64_t r1) {
    next = r0;
    end = r1;
    load_stage = 0;
    stage = STAGES - 1;
    if constexpr (E > 1) {
      ring = smem_u32(smem);
      stage_bytes = kRowBytes * blockDim.x;
      // what no copy ever fills stays zero
#pragma unroll
      for (int i = 0; i < kTensors; ++i) {
        if (i < NX) clear<ChunkX>(cols, i);
        else clear<ChunkR>(cols, i);
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
    if constexpr (E > 1) {
      using C = std::conditional_t<(I < NX), ChunkX, ChunkR>;
#pragma unroll
      for (int v = 0; v < V * C::kVecs; ++v) {
        typename C::Vec::Raw r;
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
        const uint32_t at = slot<C::kVecBytes>(stage, I, v);
        if constexpr (C::kVecBytes == 16)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
        else
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
        C::unpack(r, f + v * C::kVecCols / 2);
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
        if (i < NX) copy<TX, ChunkX>(cols, i);
        else copy<TR, ChunkR>(cols, i);
      }
    }
    ++next;
    if constexpr (E > 1) {
      load_stage = load_stage + 1 == STAGES ? 0 : load_stage + 1;
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  template <typename T, class C> __device__ void copy(const RowCols<E, V>& cols, int i) {
    const T* row = static_cast<const T*>(base[i]) + next * stride[i];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if constexpr (E == 1) {
        ahead[i * V + k] = cols.has(k) ? Ty<T>::to_f(row[cols.col(k)]) : 0.f;
      } else if (cols.has(k)) {
#pragma unroll
        for (int v = 0; v < C::kVecs; ++v) {
          const uint32_t to = slot<C::kVecBytes>(load_stage, i, k * C::kVecs + v);
          const T* from = row + cols.col(k) + v * C::kVecCols;
          if constexpr (C::kVecBytes == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
        }
      }
    }
  }
  template <class C> __device__ void clear(const RowCols<E, V>& cols, int i) {
    if (cols.has(V - 1) && base[i] != nullptr) return;
#pragma unroll 1
    for (int v = 0; v < V * C::kVecs * STAGES; ++v) {
      const uint32_t at = slot<C::kVecBytes>(v / (V * C::kVecs), i, v % (V * C::kVecs));
      if constexpr (C::kVecBytes == 16)
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
      else
        asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(at), "r"(0u) : "memory");
    }
  }
};

// Rows ahead in shared memory: as many as a full CTA has room for, four at most.
template <typename TX, typename TR> constexpr int row_stages(int cols, int nx, int nr) {
  const int row = cols * (nx * static_cast<int>(sizeof(TX)) + nr * static_cast<int>(sizeof(TR))) * kRowThreads;
  const int n = 208 * 1024 / row;
  return n < 1 ? 1 : n > 4 ? 4 : n;
}

// ---- host: which rows are whole aligned vectors ------------------------------
inline int row_elem_bytes(int dtype) { return dtype == F32 ? 4 : 2; }
// Columns of a vector chunk: 16 bytes of the wider type.
template <typename TX, typename TR> constexpr int kRowChunk = 16 / (sizeof(TX) > sizeof(TR) ? sizeof(TX) : sizeof(TR));
// Columns of a chunk with which the kernels can take these rows: kRowChunk, or 1.
inline int row_chunk(const ResidualArgs& a, bool backward) {
  const int e = 16 / std::max(row_elem_bytes(a.x_dtype), row_elem_bytes(a.res_dtype));
  bool ok = a.hidden % e == 0;
  auto aligned = [&](const void* p, int64_t stride, int dtype) {
    const int bytes = e * row_elem_bytes(dtype);
    ok = ok && reinterpret_cast<uintptr_t>(p) % bytes == 0 && (a.rows <= 1 || stride * row_elem_bytes(dtype) % bytes == 0);
  };
  aligned(a.x, a.x_stride, a.x_dtype);
  aligned(a.res, a.res_stride, a.res_dtype);
  if (backward) {
    aligned(a.dy, a.dy_stride, a.x_dtype);
    aligned(a.dh, a.dh_stride, a.res_dtype);
    aligned(a.dx, a.hidden, a.x_dtype);
    aligned(a.dres, a.hidden, a.res_dtype);
  } else {
    aligned(a.h, a.hidden, a.res_dtype);
    aligned(a.y, a.hidden, a.x_dtype);
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
