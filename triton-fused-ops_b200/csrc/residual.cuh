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

// `count` things over `parts` of them as evenly as can be, the first ones one more (no division on the device).
struct Split {
  uint32_t each, more;
  static Split make(int64_t count, int64_t parts) {
    return Split{static_cast<uint32_t>(count / parts), static_cast<uint32_t>(count % parts)};
  }
  __device__ uint32_t first(uint32_t part) const { return part * each + min(part, more); }
};

// How a launch spreads the rows.
struct RowPlan {
  int threads;      // T
  int groups;       // of a CTA
  int64_t step[4];  // bytes between the rows of the streamed tensors
  int present;      // a bit for each of them that is there (the others are zeros)
  Split share;      // rows (backward: items) of the launch's groups
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

// Which columns this thread takes, in blocks of up to 8 of them (whole chunks).
template <int E, int V> struct RowCols {
  static constexpr int N = E * V;         // columns
  static constexpr int B = N < 8 ? N : 8;  // of a block
  static constexpr int BLOCKS = N / B;
  static constexpr int BP = B / 2;  // pairs of a block
  static_assert(B % 2 == 0 && B % E == 0 && N % B == 0, "whole pairs and chunks");
  int first, step, hidden;
  __device__ RowCols(int t, int threads, int h) : first(t * E), step(threads * E), hidden(h) {}
  __device__ int col(int k) const { return first + k * step; }
  __device__ bool has(int k) const { return col(k) < hidden; }

  // Block b of p's columns of a sequence (otherwise: of a parameter that is not there, and past the row).
  __device__ void param(const RowParam& p, int64_t seq, float otherwise, int b, F2 (&f)[BP]) const {
#pragma unroll
    for (int k = 0; k < B / E; ++k) {
      float v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = otherwise;
      const int at = b * (B / E) + k;
      if (p.p != nullptr && has(at)) load_floats<E>(p.p, seq * p.seq_stride + col(at), p.dtype, v);
#pragma unroll
      for (int j = 0; j < E; ++j) lane_of(f, k * E + j) = v[j];
    }
  }
  // scale * gate * w1 (* 1 / (1 - p)): what a normed branch is multiplied by.
  __device__ void branch_coefficient(const ResidualArgs& a, int64_t seq, int b, F2 (&c)[BP]) const {
    F2 g[BP];
    param(a.branch_weight, seq, 1.f, b, c);
    param(a.gate, seq, 1.f, b, g);
    const float s = a.dropped ? a.scale * a.drop.scale : a.scale;
#pragma unroll
    for (int j = 0; j < BP; ++j) c[j] = mul2(mul2(c[j], g[j]), f2(s, s));
  }
  // Block b to this thread's first column of a row.
  template <typename T> __device__ void store(T* mine, int b, F2 (&f)[BP]) const {
#pragma unroll
    for (int k = 0; k < B / E; ++k) {
      const int at = b * (B / E) + k;
      if (!has(at)) continue;
      if constexpr (E == 1) mine[at * step] = Ty<T>::from_f(lane_of(f, k));
      else Chunk<T, E>::store(mine + at * step, f + k * E / 2);
    }
  }
  // Which of this thread's columns are kept in the row whose first element has this index.
  __device__ uint32_t kept(const DropoutArgs& d, const DropKey& key, uint64_t row) const {
    if (d.all) return 0u;
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) bits |= key.kept<E>(row + static_cast<uint32_t>(col(k))) << (k * E);
    return bits;
  }
  __device__ static void drop(uint32_t bits, int b, F2 (&f)[BP]) {
#pragma unroll
    for (int j = 0; j < BP; ++j) {
      if (!(bits >> (b * B + 2 * j) & 1)) f[j].x = 0.f;
      if (!(bits >> (b * B + 2 * j + 1) & 1)) f[j].y = 0.f;
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
  // Slots lie as for a full CTA, so that all but the stage of an address is known when this is compiled.
  static constexpr uint32_t kStageBytes = kRowBytes * kRowThreads;
  static constexpr size_t kSmemBytes = static_cast<size_t>(STAGES) * kStageBytes;

  const char* at[kTensors];  // this thread's first column of the next row to load
  int left;                  // rows to load
  uint32_t ring, write, read;  // shared memory: all stages, and the stages to fill and to read
  float ahead[E == 1 ? kTensors * V : 1], now[E == 1 ? kTensors * V : 1];

  // Vector v of tensor i in a stage: the CTA's threads side by side.
  static __device__ constexpr uint32_t offset(int i, int v, int vec_bytes) {
    return ((i < NX ? i * kBytesX : NX * kBytesX + (i - NX) * kBytesR) + v * vec_bytes) * kRowThreads;
  }

  template <typename T> __device__ void set(int i, const void* base, int64_t row, int64_t step, const RowCols<E, V>& cols) {
    at[i] = static_cast<const char*>(base) + row * step + cols.first * static_cast<int>(sizeof(T));
  }
  // After set() of each tensor: `rows` rows from there.
  __device__ void start(const RowCols<E, V>& cols, const RowPlan& plan, void* smem, int rows) {
    left = rows;
    if constexpr (E > 1) {
      ring = write = smem_u32(smem);
      read = ring + (STAGES - 1) * kStageBytes;
      // what no copy ever fills stays zero
#pragma unroll
      for (int i = 0; i < kTensors; ++i) {
        if (cols.has(V - 1) && (plan.present >> i & 1)) continue;
        if (i < NX) clear<ChunkX>(i);
        else clear<ChunkR>(i);
      }
#pragma unroll 1
      for (int i = 0; i < STAGES - 1; ++i) load(cols, plan);
    } else {
      load(cols, plan);
    }
  }
  // The next row: its values are there for get(), and the loads of a later one are under way.
  __device__ void advance(const RowCols<E, V>& cols, const RowPlan& plan) {
    if constexpr (E > 1) {
      load(cols, plan);
      read = next_stage(read);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < kTensors * V; ++i) now[i] = ahead[i];
      load(cols, plan);
    }
  }
  // Block b of tensor I.
  template <int I> __device__ void get(int b, F2 (&f)[RowCols<E, V>::BP]) const {
    constexpr int CHUNKS = RowCols<E, V>::B / E;
    if constexpr (E > 1) {
      using C = std::conditional_t<(I < NX), ChunkX, ChunkR>;
      const uint32_t mine = read + threadIdx.x * C::kVecBytes;
#pragma unroll
      for (int v = 0; v < CHUNKS * C::kVecs; ++v) {
        typename C::Vec::Raw r;
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
        const uint32_t from = mine + offset(I, b * CHUNKS * C::kVecs + v, C::kVecBytes);
        if constexpr (C::kVecBytes == 16)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(from));
        else
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from));
        C::unpack(r, f + v * C::kVecCols / 2);
      }
    } else {
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) lane_of(f, k) = now[I * V + b * CHUNKS + k];
    }
  }

 private:
  __device__ uint32_t next_stage(uint32_t st) const {
    return st == ring + (STAGES - 1) * kStageBytes ? ring : st + kStageBytes;
  }
  __device__ void load(const RowCols<E, V>& cols, const RowPlan& plan) {
    if (left > 0) {
#pragma unroll
      for (int i = 0; i < kTensors; ++i) {
        if (!(plan.present >> i & 1)) {
          if constexpr (E == 1) {
#pragma unroll
            for (int k = 0; k < V; ++k) ahead[i * V + k] = 0.f;
          }
          continue;
        }
        if (i < NX) copy<TX, ChunkX>(cols, i);
        else copy<TR, ChunkR>(cols, i);
        at[i] += plan.step[i];
      }
    }
    --left;
    if constexpr (E > 1) {
      write = next_stage(write);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  template <typename T, class C> __device__ void copy(const RowCols<E, V>& cols, int i) {
    const T* from = reinterpret_cast<const T*>(at[i]);
    const uint32_t to = write + threadIdx.x * C::kVecBytes;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if constexpr (E == 1) {
        ahead[i * V + k] = cols.has(k) ? Ty<T>::to_f(from[k * cols.step]) : 0.f;
      } else if (cols.has(k)) {
#pragma unroll
        for (int v = 0; v < C::kVecs; ++v) {
          if constexpr (C::kVecBytes == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + offset(i, k * C::kVecs + v, 16)),
                         "l"(from + k * cols.step + v * C::kVecCols)
                         : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to + offset(i, k * C::kVecs + v, 8)),
                         "l"(from + k * cols.step + v * C::kVecCols)
                         : "memory");
        }
      }
    }
  }
  template <class C> __device__ void clear(int i) const {
#pragma unroll 1
    for (int st = 0; st < STAGES; ++st) {
      const uint32_t mine = ring + st * kStageBytes + threadIdx.x * C::kVecBytes;
#pragma unroll
      for (int v = 0; v < V * C::kVecs; ++v) {
        if constexpr (C::kVecBytes == 16)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(mine + offset(i, v, 16)), "r"(0u) : "memory");
        else
          asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(mine + offset(i, v, 8)), "r"(0u) : "memory");
      }
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
