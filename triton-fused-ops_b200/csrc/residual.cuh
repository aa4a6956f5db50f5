// Shared by the kernels of the residual stream (residual_norm.cu,
// residual_norm_backward.cu): how a row is spread over threads, the stream of
// rows through shared memory, sums over a row, and the parameters' columns.
//
// A row of `hidden` columns is chunks of E columns: 16 bytes of the wider of x
// and the stream. Rows need not be whole aligned vectors: if they are not (SHIFTED),
// a chunk is read as the two aligned vectors that it lies in, and a warp puts its
// outputs together into aligned vectors (15992 rows of 1001 bf16: 50 us, a column a thread 113). T threads (whole
// warps) take a row, thread t its chunks t, t + T, ... (V of them): a group.
// A CTA holds several groups when rows are short, each with rows of its own
// and a named barrier for its sums.
#pragma once

#include <initializer_list>

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
  const char* base[4];  // the streamed tensors
  uint32_t step[4];     // bytes between their rows
  int present;      // a bit for each of them that is there (the others are zeros)
  // The rows (backward: items) of the launch's groups: a run for each or, with a stride, every so manyth one, so that all
  // groups read side by side (8192 x 4096: bf16 forward 49 -> 46 us, fp32 backward of 4096 rows 74 -> 69).
  Split share;
  uint32_t stride;  // 0: runs
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
// E columns of T, one vector of 16 or 8 bytes, as pairs of floats.
template <typename T, int E> struct Chunk {
  static constexpr int kBytes = E * static_cast<int>(sizeof(T));
  static constexpr int kWords = kBytes / 4;
  static_assert(kBytes == 16 || kBytes == 8, "one vector");
  using Vec = HeadVec<T, E>;
  using Raw = typename Vec::Raw;
  __device__ static void unpack(const Raw& r, F2* f) {
    F2 t[E / 2];
    Vec::unpack(r, t);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) f[i] = t[i];
  }
  __device__ static Raw pack(const F2* f) {
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
    return r;
  }
  // The vector that starts `bytes` (less than a vector) into two of them side by side.
  __device__ static Raw joined(const Raw& low, const Raw& high, uint32_t bytes) {
    uint32_t w[2 * kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      w[i] = reinterpret_cast<const uint32_t*>(&low)[i];
      w[kWords + i] = reinterpret_cast<const uint32_t*>(&high)[i];
    }
    if constexpr (kWords == 4) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = bytes & 8 ? w[i + 2] : w[i];
    }
#pragma unroll
    for (int i = 0; i < kWords + 1; ++i) w[i] = bytes & 4 ? w[i + 1] : w[i];
    Raw r;
    uint32_t* o = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < kWords; ++i) o[i] = sizeof(T) == 4 ? w[i] : __funnelshift_r(w[i], w[i + 1], (bytes & 3) * 8);
    return r;
  }
};

__device__ __forceinline__ float& lane_of(F2* f, int i) { return i & 1 ? f[i >> 1].y : f[i >> 1].x; }

// Which columns this thread takes, in blocks of up to 8 of them (whole chunks).
template <int E, int V, bool SHIFTED> struct RowCols {
  static constexpr int N = E * V;         // columns
  static constexpr int B = N < 8 ? N : 8;  // of a block
  static constexpr int BLOCKS = N / B;
  static constexpr int BP = B / 2;  // pairs of a block
  static constexpr int BC = B / E;  // chunks of a block
  static_assert(B % 2 == 0 && B % E == 0 && N % B == 0, "whole pairs and chunks");
  int first, step, hidden;
  __device__ RowCols(int t, int threads, int h) : first(t * E), step(threads * E), hidden(h) {}
  __device__ int col(int k) const { return first + k * step; }
  __device__ bool has(int k) const { return col(k) < hidden; }
  // How many of chunk k's columns there are: all or none but in SHIFTED rows.
  __device__ int count(int k) const { return min(max(hidden - col(k), 0), E); }

  // Block b of p's columns of a sequence (otherwise: of a parameter that is not there, and past the row).
  __device__ void param(const RowParam& p, int64_t seq, float otherwise, int b, F2 (&f)[BP]) const {
#pragma unroll
    for (int k = 0; k < BC; ++k) {
      float v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = otherwise;
      const int at = b * BC + k;
      if (p.p != nullptr && has(at)) {
        const int64_t i = seq * p.seq_stride + col(at);
        if constexpr (SHIFTED) {
          const int n = count(at);
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (j < n) v[j] = load_as_float(p.p, i + j, p.dtype);
        } else {
          load_floats<E>(p.p, i, p.dtype, v);
        }
      }
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
  // Block b to a row. The whole warp takes part.
  template <typename T> __device__ void store(T* row, int b, F2 (&f)[BP]) const {
    using C = Chunk<T, E>;
#pragma unroll
    for (int k = 0; k < BC; ++k) {
      const int at = b * BC + k;
      const typename C::Raw own = C::pack(f + k * E / 2);
      T* to = row + col(at);
      const uint32_t shift = SHIFTED ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to)) % C::kBytes : 0u;
      if (!SHIFTED || (shift == 0 && hidden % E == 0)) {
        if (has(at)) *reinterpret_cast<typename C::Raw*>(to) = own;
        continue;
      }
      // The aligned vector in which this chunk begins: the lane before's last columns and this one's first.
      const int lane = threadIdx.x & 31, n = count(at);
      const int head = static_cast<int>((C::kBytes - shift) / sizeof(T));  // own columns in that vector
      typename C::Raw before;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&own);
      uint32_t* u = reinterpret_cast<uint32_t*>(&before);
#pragma unroll
      for (int i = 0; i < C::kWords; ++i) u[i] = __shfl_up_sync(0xffffffffu, w[i], 1);
      const typename C::Raw joined = shift == 0 ? own : C::joined(before, own, C::kBytes - shift);
      auto* vector = reinterpret_cast<typename C::Raw*>(reinterpret_cast<char*>(to) - shift);
      if (col(at) - lane * E + 32 * E <= hidden) {
        // Whole chunks in all lanes. The E columns that are left, the first lane's first ones and the last lane's last
        // ones, by a lane each.
        if (shift == 0 || lane > 0) *vector = joined;
        const int from = lane < head ? 0 : 31;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < C::kWords; ++i) {
          const uint32_t got = __shfl_sync(0xffffffffu, w[i], from);
          if (lane * static_cast<int>(sizeof(T)) / 4 == i) word = got;
        }
        if (shift != 0 && lane < E) {
          T* one = to + (from - lane) * E + lane;
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(one) = word;
          else *reinterpret_cast<uint16_t*>(one) = static_cast<uint16_t>(lane & 1 ? word >> 16 : word);
        }
        __syncwarp();
        continue;
      }
      // The row's end: a lane without the columns for its vector, the first one and the last of the row give theirs one by
      // one.
      const bool whole = n >= head && (shift == 0 || lane > 0);
      const bool next = __shfl_down_sync(0xffffffffu, static_cast<int>(whole), 1) && lane < 31;
      if (whole) *vector = joined;
      if (!whole || !next) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j < n && (j < head ? !whole : !next)) to[j] = Ty<T>::from_f(lane_of(f, k * E + j));
      }
      __syncwarp();
    }
  }
  // Block b to a row of floats (aligned rows).
  __device__ void store_floats(float* row, int b, const F2 (&f)[BP]) const {
#pragma unroll
    for (int k = 0; k < BC; ++k) {
      const int at = b * BC + k;
      if (!has(at)) continue;
#pragma unroll
      for (int j = 0; j < E / 4; ++j)
        reinterpret_cast<float4*>(row + col(at))[j] =
            make_float4(f[k * E / 2 + 2 * j].x, f[k * E / 2 + 2 * j].y, f[k * E / 2 + 2 * j + 1].x, f[k * E / 2 + 2 * j + 1].y);
    }
  }
  // Which of this thread's columns are kept in the row whose first element has this index.
  __device__ uint32_t kept(const DropoutArgs& d, const DropKey& key, uint64_t row) const {
    if (d.all) return 0u;
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const uint64_t i = row + static_cast<uint32_t>(col(k));
      // whole blocks of words, of which the chunk begins in the first one
      if constexpr (SHIFTED) bits |= (key.kept<E + 4>(i & ~uint64_t{3}) >> (i & 3) & ((1u << E) - 1)) << (k * E);
      else bits |= key.kept<E>(i) << (k * E);
    }
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
// A thread's chunks of the rows ahead, of NX tensors of TX and NR of TR, through a
// ring in shared memory by cp.async, each thread writing and reading its own
// slots: no barrier, and the loads in flight cost no registers. SHIFTED: two
// aligned vectors for each chunk, of which only those are read that hold a column
// of it (so none lies outside the row's first and last aligned vector).
template <typename TX, typename TR, int E, int V, bool SHIFTED, int NX, int NR, int STAGES>
struct RowStream {
  using Cols = RowCols<E, V, SHIFTED>;
  static constexpr int kTensors = NX + NR;
  static constexpr int VECS = SHIFTED ? 2 : 1;  // of a chunk
  using ChunkX = Chunk<TX, E>;
  using ChunkR = Chunk<TR, E>;
  static constexpr int kBytesX = V * VECS * ChunkX::kBytes, kBytesR = V * VECS * ChunkR::kBytes;  // of a thread and row
  static constexpr int kRowBytes = NX * kBytesX + NR * kBytesR;
  // Slots lie as for a full CTA, so that all but the stage of an address is known when this is compiled.
  static constexpr uint32_t kStageBytes = kRowBytes * kRowThreads;
  static constexpr size_t kSmemBytes = static_cast<size_t>(STAGES) * kStageBytes;
  template <int I> using ChunkOf = std::conditional_t<(I < NX), ChunkX, ChunkR>;

  uint32_t next, end, by;      // rows to load
  // Two tensors' next rows as pointers that walk on; with four they would cost registers that the rest needs, and are
  // made from the row's index (8192 x 5120 forward 70 us without walking, 66 with it; fp32 4096 x 4096 backward 84 with it, 69 without).
  static constexpr bool WALK = kTensors == 2;
  const char* at[WALK ? kTensors : 1];
  uint32_t ring, write, read;  // shared memory: all stages, and the stages to fill and to read

  // Vector v of tensor i in a stage: the CTA's threads side by side.
  static __device__ constexpr uint32_t offset(int i, int v, int vec_bytes) {
    return ((i < NX ? i * kBytesX : NX * kBytesX + (i - NX) * kBytesR) + v * vec_bytes) * kRowThreads;
  }

  // Rows from `first` on, before `last`, `step` apart.
  __device__ void start(const Cols& cols, const RowPlan& plan, void* smem, uint32_t first, uint32_t last, uint32_t step) {
    next = first;
    end = last;
    by = step;
    if constexpr (WALK) {
#pragma unroll
      for (int i = 0; i < kTensors; ++i)
        at[i] = plan.base[i] + static_cast<uint64_t>(first) * plan.step[i] + cols.first * (i < NX ? sizeof(TX) : sizeof(TR));
    }
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
  }
  // The next row: its values are there for get(), and the loads of a later one are under way.
  __device__ void advance(const Cols& cols, const RowPlan& plan) {
    load(cols, plan);
    read = next_stage(read);
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
  }
  // Block b of tensor I of `row`, the one that advance() has brought.
  template <int I> __device__ void get(const Cols& cols, const RowPlan& plan, uint32_t row, int b, F2 (&f)[Cols::BP]) const {
    using C = ChunkOf<I>;
    // bytes into the first of a chunk's aligned vectors, the same for all chunks
    const uint32_t shift =
        SHIFTED ? (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(plan.base[I])) + row * plan.step[I]) % C::kBytes : 0u;
    const uint32_t mine = read + threadIdx.x * C::kBytes;
#pragma unroll
    for (int k = 0; k < Cols::BC; ++k) {
      const int at_chunk = b * Cols::BC + k;
      typename C::Raw r = fetch<C>(mine + offset(I, at_chunk * VECS, C::kBytes));
      if constexpr (SHIFTED) {
        r = C::joined(r, fetch<C>(mine + offset(I, at_chunk * VECS + 1, C::kBytes)), shift);
        C::unpack(r, f + k * E / 2);
        const int n = cols.count(at_chunk);
        if (n < E) {  // the next row's columns, or nobody's
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (j >= n) lane_of(f, k * E + j) = 0.f;
        }
      } else {
        C::unpack(r, f + k * E / 2);
      }
    }
  }

 private:
  template <class C> static __device__ typename C::Raw fetch(uint32_t from) {
    typename C::Raw r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    if constexpr (C::kBytes == 16)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from));
    else
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from));
    return r;
  }
  __device__ uint32_t next_stage(uint32_t st) const {
    return st == ring + (STAGES - 1) * kStageBytes ? ring : st + kStageBytes;
  }
  __device__ void load(const Cols& cols, const RowPlan& plan) {
    if (next < end) {
#pragma unroll
      for (int i = 0; i < kTensors; ++i) {
        if (!(plan.present >> i & 1)) continue;
        const char* from;
        if constexpr (WALK) {
          from = at[i];
          at[i] += static_cast<uint64_t>(plan.step[i]) * by;
        } else {
          from = plan.base[i] + static_cast<uint64_t>(next) * plan.step[i] + cols.first * (i < NX ? sizeof(TX) : sizeof(TR));
        }
        if (i < NX) copy<TX, ChunkX>(cols, i, from);
        else copy<TR, ChunkR>(cols, i, from);
      }
    }
    next += by;
    write = next_stage(write);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  template <class C> static __device__ void copy_vector(uint32_t to, const void* from) {
    if constexpr (C::kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
  }
  template <typename T, class C> __device__ void copy(const Cols& cols, int i, const char* mine) {
    const uint32_t to = write + threadIdx.x * C::kBytes;
    const uint32_t into = SHIFTED ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(mine)) % C::kBytes : 0u;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (!cols.has(k)) continue;
      const T* from = reinterpret_cast<const T*>(mine - into) + k * cols.step;
      copy_vector<C>(to + offset(i, k * VECS, C::kBytes), from);
      if (SHIFTED && into + cols.count(k) * static_cast<int>(sizeof(T)) > C::kBytes)
        copy_vector<C>(to + offset(i, k * VECS + 1, C::kBytes), from + E);
    }
  }
  template <class C> __device__ void clear(int i) const {
#pragma unroll 1
    for (int st = 0; st < STAGES; ++st) {
      const uint32_t mine = ring + st * kStageBytes + threadIdx.x * C::kBytes;
#pragma unroll
      for (int v = 0; v < V * VECS; ++v) {
        if constexpr (C::kBytes == 16)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(mine + offset(i, v, 16)), "r"(0u) : "memory");
        else
          asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(mine + offset(i, v, 8)), "r"(0u) : "memory");
      }
    }
  }
};

// Rows ahead in shared memory: as many as a full CTA has room for, four at most.
template <typename TX, typename TR> constexpr int row_stages(int cols, int nx, int nr, bool shifted) {
  const int row = (shifted ? 2 : 1) * cols * (nx * static_cast<int>(sizeof(TX)) + nr * static_cast<int>(sizeof(TR))) * kRowThreads;
  const int n = 208 * 1024 / row;
  return n < 1 ? 1 : n > 4 ? 4 : n;
}

// ---- host: which rows are whole aligned vectors ------------------------------
inline int row_elem_bytes(int dtype) { return dtype == F32 ? 4 : 2; }
// Columns of a chunk: 16 bytes of the wider type.
template <typename TX, typename TR> constexpr int kRowChunk = 16 / (sizeof(TX) > sizeof(TR) ? sizeof(TX) : sizeof(TR));
// The streamed tensors of a launch: their steps have to be 32-bit numbers of bytes.
inline bool set_tensors(RowPlan* plan, std::initializer_list<std::pair<const void*, int64_t>> tensors) {
  int i = 0;
  for (const auto& [p, step] : tensors) {
    if (p != nullptr && step > UINT32_MAX) return false;
    plan->base[i] = static_cast<const char*>(p);
    plan->step[i] = static_cast<uint32_t>(step);
    plan->present |= (p != nullptr ? 1 : 0) << i++;
  }
  return true;
}
// Whether rows and parameters are whole aligned vectors of chunks.
inline bool rows_aligned(const ResidualArgs& a, bool backward) {
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
  return ok;
}
// T for V chunks of E columns a thread (0: the row does not fit).
inline int row_threads(int hidden, int e, int v) {
  const int64_t need = (static_cast<int64_t>(hidden) + e * v - 1) / (e * v);
  const int64_t t = (need + 31) / 32 * 32;
  return t <= kRowThreads ? static_cast<int>(t) : 0;
}

}  // namespace tfo
