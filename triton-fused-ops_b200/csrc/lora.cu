// Low-rank adapters of many requests beside a shared projection.
//
//   out[t] = base[t] + scaling[i] * B[i] (A[i] x[t]),   i = ids[t]
//   x [tokens, K], A [adapters, rank, K], B [adapters, N, rank];
//   i < 0: out[t] = base[t]; i >= adapters: NaN, and the device error word.
//
// Two steps with the low-rank values v = A x in fp32 between them:
//   shrink: v = the sum over K, cut into parts that are added in a fixed order
//   expand: out = base + B (scaling * v)
// Rows that use the same adapter are grouped into tiles, so that an adapter's
// matrices are read once per tile and not once per row:
//   up to 256 tokens, one launch (lora_small_kernel): row i leads a tile if 0,
//     16, 32, ... rows before it use the same adapter, which every CTA finds
//     out from the ids; a cluster of CTAs shares a tile, each shrinks a part of
//     K, reads the others' sums through distributed shared memory and expands a
//     part of the columns;
//   more: a one-CTA kernel sorts the rows by adapter into tiles of 64, then two
//     kernels stream x and A, and base and B, through shared memory.
// A row's result does not depend on the rows beside it in its tile.
//
// Both products run on m16n8 tensor instructions with rows of a tile as M.
// They are far from the tensor rate (2 * rank flops for each byte of x); what
// bounds them is reading x, A and B once and the output traffic, so operands
// go from global memory straight into fragments: the order of the summed index
// inside a product is free, and with thread q of four taking the 16 bytes
// [16 q, 16 q + 16) of a 64-byte chunk on both sides, every load is a whole
// vector. Likewise the output columns of four instructions are dealt out so
// that a thread ends up with eight neighbouring ones.
//
// Rounding: products and sums are fp32. v enters the second product as the sum
// of two values of x's type, hi + lo (16 bits of bf16, 22 of fp16 relative to
// the row's largest value, by which the row is scaled to stay in fp16's
// range); fp32 operands are split into two tf32 values on both sides and the
// three larger products are added. The result is rounded once.
#include "heads.cuh"

namespace tfo {

constexpr int kSmallTokens = 256;  // at most: each CTA reads all ids (one per thread)
constexpr int kSmallRows = 16, kSmallWarps = 8, kMaxCluster = 8;
constexpr int kLargeRows = 64, kLargeThreads = 128;

__host__ __device__ constexpr int chunk_elems(int esize) { return 64 / esize; }  // summed elements per 64-byte chunk
// Ranks as the expand step holds them: a power of two of chunks.
inline int64_t padded_rank(int64_t rank, int esize) {
  int64_t r = chunk_elems(esize);
  while (r < rank) r *= 2;
  return r;
}

// ---- tensor instructions ------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x = hi + lo in two tf32 values (an infinity or NaN is all in hi).
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(x)));
  const float h = __uint_as_float(hi);
  const float rest = fabsf(h) <= 3.402823466e38f ? __uint_as_float(x) - h : 0.f;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
}

// d += the product over one 64-byte chunk: a0 / a1 are rows g and g + 8 of the
// first operand, b is row g of the second (lane = 4 g + q, q-th 16 bytes).
template <typename T> struct Chunk;
template <> struct Chunk<__half> {
  __device__ static void mma(float (&d)[4], const uint4& a0, const uint4& a1, const uint4& b) {
    mma_f16(d, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
    mma_f16(d, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
  }
};
template <> struct Chunk<__nv_bfloat16> {
  __device__ static void mma(float (&d)[4], const uint4& a0, const uint4& a1, const uint4& b) {
    mma_bf16(d, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
    mma_bf16(d, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
  }
};
template <> struct Chunk<float> {
  __device__ static void mma(float (&d)[4], const uint4& a0, const uint4& a1, const uint4& b) {
    half(d, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
    half(d, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
  }
  __device__ static void half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                              uint32_t b1) {
    uint32_t h[6], l[6];
    split_tf32(a0, h[0], l[0]);
    split_tf32(a1, h[1], l[1]);
    split_tf32(a2, h[2], l[2]);
    split_tf32(a3, h[3], l[3]);
    split_tf32(b0, h[4], l[4]);
    split_tf32(b1, h[5], l[5]);
    mma_tf32(d, l[0], l[1], l[2], l[3], h[4], h[5]);
    mma_tf32(d, h[0], h[1], h[2], h[3], l[4], l[5]);
    mma_tf32(d, h[0], h[1], h[2], h[3], h[4], h[5]);
  }
};

// 16 bytes at row + i, elements at or past `limit` (and a NULL row) as zeros.
// `width`: elements that rows are aligned to and a multiple of (a vector of 16
// bytes, of 8, or 1).
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const T* row, int64_t i, int64_t limit, int width) {
  constexpr int E = 16 / sizeof(T);
  if (row == nullptr || i >= limit) return make_uint4(0, 0, 0, 0);
  if (width == E) return *reinterpret_cast<const uint4*>(row + i);
  if (width == E / 2) {
    const uint2 lo = *reinterpret_cast<const uint2*>(row + i);
    const uint2 hi = i + E / 2 < limit ? *reinterpret_cast<const uint2*>(row + i + E / 2) : make_uint2(0, 0);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  alignas(16) T t[E];
#pragma unroll
  for (int j = 0; j < E; ++j) t[j] = i + j < limit ? row[i + j] : Ty<T>::from_f(0.f);
  return *reinterpret_cast<const uint4*>(t);
}

// ---- tiles of rows with the same adapter ------------------------------------------
struct LoraPlan {  // of many tokens, in the workspace
  int* perm;       // rows, by group
  int4* tiles;     // {group, first, count, 0}; first indexes perm
  int* num_tiles;
};

// Group of a row: its adapter, `adapters` for none, `adapters` + 1 for an id past the end.
__device__ __forceinline__ int row_group(const LoraArgs& a, int64_t t) {
  const int64_t id = a.ids_dtype == POS_I64 ? reinterpret_cast<const int64_t*>(a.ids)[t]
                                            : reinterpret_cast<const int32_t*>(a.ids)[t];
  const int n = static_cast<int>(a.adapters);
  return id < 0 ? n : id >= n ? n + 1 : static_cast<int>(id);
}

struct Tile {
  int group, count;  // count 0: nothing to do
};

// The tile that row `lead` leads, by the whole CTA (256 threads, tokens <= 256); rows gets its rows.
__device__ __forceinline__ Tile find_tile(const LoraArgs& a, int lead, int* rows, int* scratch) {
  const int t = threadIdx.x;
  const int tokens = static_cast<int>(a.tokens);
  const int group = t < tokens ? row_group(a, t) : -1;
  if (t == lead) scratch[8] = group;
  __syncthreads();
  const int want = scratch[8];
  const bool same = group == want;
  if (__syncthreads_count(same && t < lead) % kSmallRows != 0) return Tile{want, 0};
  const uint32_t votes = __ballot_sync(0xffffffffu, same && t >= lead);
  if ((t & 31) == 0) scratch[t >> 5] = __popc(votes);
  __syncthreads();
  int before = __popc(votes & ((1u << (t & 31)) - 1)), all = 0;
  for (int w = 0; w < kSmallWarps; ++w) {
    if (w < t >> 5) before += scratch[w];
    all += scratch[w];
  }
  if (same && t >= lead && before < kSmallRows) rows[before] = t;
  __syncthreads();
  return Tile{want, min(all, kSmallRows)};
}

// A tile of the sorted rows, by the whole CTA.
__device__ __forceinline__ Tile planned_tile(const LoraPlan& plan, int* rows) {
  if (static_cast<int>(blockIdx.x) >= *plan.num_tiles) return Tile{0, 0};
  const int4 t = plan.tiles[blockIdx.x];
  if (threadIdx.x < t.z) rows[threadIdx.x] = plan.perm[t.y + threadIdx.x];
  __syncthreads();
  return Tile{t.x, t.z};
}

// Sorts the rows by group (the order inside a group is free) and cuts the
// groups into tiles. One CTA, whose threads hold kHeld ids each: their loads
// are in flight together, and up to 8192 rows are read once.
constexpr int kHeld = 8, kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const LoraArgs a, LoraPlan plan) {
  extern __shared__ int bins[];  // [groups] rows of each, then the next free place
  __shared__ int carry[2], sum_rows[32], sum_tiles[32];
  griddep_launch_dependents();
  griddep_wait();
  const int groups = static_cast<int>(a.adapters) + 2;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int tokens = static_cast<int>(a.tokens);
  int held[kHeld];
  auto load = [&](int first) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int64_t i = static_cast<int64_t>(first) + j * kPlanThreads + t;
      held[j] = i < tokens ? row_group(a, i) : -1;
    }
  };
  constexpr int kStep = kHeld * kPlanThreads;
  load(0);
  for (int i = t; i < groups; i += kPlanThreads) bins[i] = 0;
  if (t < 2) carry[t] = 0;
  __syncthreads();
  for (int64_t first = 0; first < tokens; first += kStep) {
    if (first > 0) load(static_cast<int>(first));
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (first + j * kPlanThreads + (t & ~31) >= tokens) break;
      const uint32_t peers = __match_any_sync(0xffffffffu, held[j]);
      if (held[j] >= 0 && lane == __ffs(peers) - 1) atomicAdd(&bins[held[j]], __popc(peers));
    }
  }
  __syncthreads();
  // exclusive prefix sums of rows and tiles over the groups
  for (int first = 0; first < groups; first += kPlanThreads) {
    const int g = first + t;
    const int count = g < groups ? bins[g] : 0;
    const int ntiles = (count + kLargeRows - 1) / kLargeRows;
    int r = count, n = ntiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int pr = __shfl_up_sync(0xffffffffu, r, o), pn = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) {
        r += pr;
        n += pn;
      }
    }
    if (lane == 31) {
      sum_rows[warp] = r;
      sum_tiles[warp] = n;
    }
    __syncthreads();
    int before_r = carry[0], before_n = carry[1];
    for (int w = 0; w < warp; ++w) {
      before_r += sum_rows[w];
      before_n += sum_tiles[w];
    }
    const int row0 = before_r + r - count, tile0 = before_n + n - ntiles;
    if (g < groups) {
      bins[g] = row0;
      for (int i = 0; i < ntiles; ++i)
        plan.tiles[tile0 + i] = make_int4(g, row0 + i * kLargeRows, min(kLargeRows, count - i * kLargeRows), 0);
    }
    __syncthreads();
    if (t == kPlanThreads - 1) {
      carry[0] = before_r + r;
      carry[1] = before_n + n;
    }
    __syncthreads();
  }
  if (t == 0) *plan.num_tiles = carry[1];
  for (int64_t first = 0; first < tokens; first += kStep) {
    if (tokens > kStep) load(static_cast<int>(first));
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int64_t i = first + j * kPlanThreads + t;
      if (i - lane >= tokens) break;
      const int g = held[j];
      const uint32_t peers = __match_any_sync(0xffffffffu, g);
      const int leader = __ffs(peers) - 1;
      int at = 0;
      if (g >= 0 && lane == leader) at = atomicAdd(&bins[g], __popc(peers));
      at = __shfl_sync(0xffffffffu, at, leader);
      if (g >= 0) plan.perm[at + __popc(peers & ((1u << lane) - 1))] = static_cast<int>(i);
    }
  }
}

// ---- streaming through shared memory -------------------------------------------------
// Tiles are rows of `nch` 64-byte chunks. Eight lanes that read 16 bytes each
// touch two rows of different parity; an even number of chunks would put those
// on the same banks, so the chunks of odd rows are swapped in pairs.
__device__ __forceinline__ uint32_t tile_offset(int row, int nch, int chunk, int quarter) {
  const int c = (nch & 1) ? chunk : chunk ^ (row & 1);
  return static_cast<uint32_t>((row * nch + c) * 64 + quarter * 16);
}
// 16 bytes from global to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// ---- shrink: v = A x ---------------------------------------------------------------
// grid: (tiles, splits of K, blocks of 8 NT ranks); a warp has 16 rows.
__device__ __forceinline__ void split_range(int64_t units, int splits, int split, int* first, int* last) {
  *first = static_cast<int>(units * split / splits);
  *last = static_cast<int>(units * (split + 1) / splits);
}

template <int NT>
__device__ __forceinline__ void store_v(const Tile& tile, const int* rows, float* v, int64_t v_rank, int r0, int m0, int g,
                                        int q, const float (&acc)[NT][4]) {
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = r0 + j * 8 + 2 * q;
    if (r >= v_rank) continue;  // v_rank is a multiple of 16
    if (m0 + g < tile.count)
      *reinterpret_cast<float2*>(v + static_cast<int64_t>(rows[m0 + g]) * v_rank + r) = make_float2(acc[j][0], acc[j][1]);
    if (m0 + g + 8 < tile.count)
      *reinterpret_cast<float2*>(v + static_cast<int64_t>(rows[m0 + g + 8]) * v_rank + r) = make_float2(acc[j][2], acc[j][3]);
  }
}

// x and A in steps of 128 bytes of K, STAGES deep.
template <typename T, int NT, int STAGES>
__global__ void __launch_bounds__(kLargeThreads) lora_shrink_kernel(const LoraArgs a, LoraPlan plan, float* __restrict__ v,
                                                                    int splits, int64_t v_rank) {
  constexpr int E = 16 / sizeof(T), KS = 128 / sizeof(T);
  constexpr int kXBytes = kLargeRows * 128, kStage = kXBytes + 8 * NT * 128;
  __shared__ int rows[kLargeRows];
  extern __shared__ __align__(128) uint8_t smem[];
  griddep_launch_dependents();
  griddep_wait();
  const Tile tile = planned_tile(plan, rows);
  if (tile.count == 0 || tile.group >= a.adapters) return;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int k0, k1;
  split_range((a.k + KS - 1) / KS, splits, blockIdx.y, &k0, &k1);
  // this thread's copies: 16 bytes `vec` of every sixteenth row
  const int vec = t & 7, row0 = t >> 3;
  const int r0 = blockIdx.z * 8 * NT;
  const T* x = static_cast<const T*>(a.x) + vec * E;
  const T* w = static_cast<const T*>(a.a) + (static_cast<int64_t>(tile.group) * a.rank + r0) * a.k + vec * E;
  const T* xp[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) xp[i] = x + static_cast<int64_t>(rows[min(row0 + 16 * i, tile.count - 1)]) * a.x_stride;
  const uint32_t base = smem_u32(smem);
  auto load = [&](int step, int stage) {
    if (step < k1) {
      const int64_t at = static_cast<int64_t>(step) * KS;
      const bool in = at + vec * E < a.k;
      const uint32_t dst = base + stage * kStage;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = row0 + 16 * i;
        copy16(dst + tile_offset(r, 2, vec >> 2, vec & 3), in ? xp[i] + at : a.x, in && r < tile.count);
      }
#pragma unroll
      for (int i = 0; i < NT / 2; ++i) {
        const int r = row0 + 16 * i;
        const bool ok = in && r0 + r < a.rank;
        copy16(dst + kXBytes + tile_offset(r, 2, vec >> 2, vec & 3), ok ? w + r * a.k + at : a.a, ok);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(k0 + i, i);
  const int g = lane >> 2, q = lane & 3, m0 = warp * 16;
  float acc[NT][4] = {};
  int stage = 0;
  for (int step = k0; step < k1; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();  // the step's bytes are there, and the stage before it is free
    load(step + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
    if (m0 < tile.count) {
      const uint8_t* xs = smem + stage * kStage;
      const uint8_t* as = xs + kXBytes;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 a0 = lds16(xs + tile_offset(m0 + g, 2, c, q)), a1 = lds16(xs + tile_offset(m0 + g + 8, 2, c, q));
#pragma unroll
        for (int j = 0; j < NT; ++j) Chunk<T>::mma(acc[j], a0, a1, lds16(as + tile_offset(j * 8 + g, 2, c, q)));
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  store_v<NT>(tile, rows, v + static_cast<int64_t>(blockIdx.y) * a.tokens * v_rank, v_rank, r0, m0, g, q, acc);
}

// Any alignment of x and A: elements straight into fragments.
template <typename T, int NT>
__global__ void __launch_bounds__(kLargeThreads) lora_shrink_any_kernel(const LoraArgs a, LoraPlan plan,
                                                                        float* __restrict__ v, int splits, int64_t v_rank) {
  constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  __shared__ int rows[kLargeRows];
  griddep_launch_dependents();
  griddep_wait();
  const Tile tile = planned_tile(plan, rows);
  if (tile.count == 0 || tile.group >= a.adapters) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q = lane & 3, m0 = warp * 16;
  if (m0 >= tile.count) return;
  const T* x = static_cast<const T*>(a.x);
  const T* x0 = m0 + g < tile.count ? x + static_cast<int64_t>(rows[m0 + g]) * a.x_stride : nullptr;
  const T* x1 = m0 + g + 8 < tile.count ? x + static_cast<int64_t>(rows[m0 + g + 8]) * a.x_stride : nullptr;
  const int r0 = blockIdx.z * 8 * NT;
  const T* w[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = r0 + j * 8 + g;
    w[j] = r < a.rank ? static_cast<const T*>(a.a) + (static_cast<int64_t>(tile.group) * a.rank + r) * a.k : nullptr;
  }
  int c0, c1;
  split_range((a.k + C - 1) / C, splits, blockIdx.y, &c0, &c1);
  float acc[NT][4] = {};
  for (int c = c0; c < c1; ++c) {
    const int64_t i = static_cast<int64_t>(c) * C + q * E;
    const uint4 a0 = load_chunk<T>(x0, i, a.k, 1), a1 = load_chunk<T>(x1, i, a.k, 1);
#pragma unroll
    for (int j = 0; j < NT; ++j) Chunk<T>::mma(acc[j], a0, a1, load_chunk<T>(w[j], i, a.k, 1));
  }
  store_v<NT>(tile, rows, v + static_cast<int64_t>(blockIdx.y) * a.tokens * v_rank, v_rank, r0, m0, g, q, acc);
}

// ---- expand: out = base + B v ------------------------------------------------------
// Eight neighbouring values of a row, as raw 16-byte vectors.
template <typename T> struct Eight {
  static constexpr int W = 8 * sizeof(T) / 16;
  uint4 u[W];
};
template <typename T>
__device__ __forceinline__ void load_eight(Eight<T>& e, const T* p) {
#pragma unroll
  for (int i = 0; i < Eight<T>::W; ++i) e.u[i] = reinterpret_cast<const uint4*>(p)[i];
}
// out = e + f, whole vectors
template <typename T>
__device__ __forceinline__ void store_sum(T* out, const Eight<T>& e, bool with_base, const float (&f)[8]) {
  using V = HeadVec<T, 16 / sizeof(T)>;
  constexpr int H = 8 / sizeof(T);  // pairs of a 16-byte vector
#pragma unroll
  for (int i = 0; i < Eight<T>::W; ++i) {
    F2 t[H];
    V::unpack(e.u[i], t);
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const float x = f[2 * (i * H + j)], y = f[2 * (i * H + j) + 1];
      t[j] = with_base ? f2(t[j].x + x, t[j].y + y) : f2(x, y);
    }
    V::store(out + i * (16 / sizeof(T)), t);
  }
}
// out = base + f element by element, `limit` of the eight at most
template <typename T>
__device__ __forceinline__ void store_each(T* out, const T* base, int64_t limit, const float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < limit) out[j] = Ty<T>::from_f(base != nullptr ? Ty<T>::to_f(base[j]) + f[j] : f[j]);
  }
}

// Rows without a product: copied from base (or zero), or NaN for a bad id.
template <typename T>
__device__ __forceinline__ void fill_rows(const LoraArgs& a, const Tile& tile, const int* rows, int64_t col0, int64_t col1,
                                          bool vec, uint32_t* err) {
  const bool bad = tile.group > a.adapters;
  if (bad && threadIdx.x == 0) set_error(err, ERR_BAD_ADAPTER);
  if (col0 >= col1 || (!bad && a.base == a.out)) return;  // left as they are
  const T fill = Ty<T>::from_f(bad ? __int_as_float(0x7fffffff) : 0.f);
  const int per_row = static_cast<int>((col1 - col0 + 7) / 8);
  for (int i = threadIdx.x; i < per_row * tile.count; i += blockDim.x) {
    const int64_t row = rows[i / per_row], col = col0 + i % per_row * 8;
    const T* base = a.base != nullptr && !bad ? static_cast<const T*>(a.base) + row * a.base_stride + col : nullptr;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + col;
    if (vec && base != nullptr) {
      Eight<T> e;
      load_eight(e, base);
#pragma unroll
      for (int j = 0; j < Eight<T>::W; ++j) reinterpret_cast<uint4*>(out)[j] = e.u[j];
    } else {
      for (int j = 0; j < 8 && col + j < col1; ++j) out[j] = base != nullptr ? base[j] : fill;
    }
  }
}

// Stages the tile's v as operands in shared memory: hi and lo (16-bit types;
// fp32 as it is), [M][stride] elements. sum(m, r) gives four neighbouring
// values of row m, summed and scaled. fp16 rows are scaled by a power of two
// to below 2 (row_scale takes it back; `sums` holds them meanwhile); rows past
// the tile and ranks past the end are zero.
template <typename T, int M, typename Sum>
__device__ __forceinline__ void stage_v(const Tile& tile, int rank, int vr, int stride, T* hi, T* lo, float* sums,
                                        float* row_scale, unsigned* row_max, Sum sum) {
  constexpr bool SPLIT = sizeof(T) == 2;
  constexpr bool SCALED = std::is_same<T, __half>::value;
  const int quads = vr / 4, threads = blockDim.x;
  if constexpr (SCALED) {
    for (int m = threadIdx.x; m < M; m += threads) row_max[m] = 0;
    __syncthreads();
  }
  auto put = [&](int m, int r, const float (&t)[4], float down) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = SCALED ? t[j] * down : t[j];
      const T h = Ty<T>::from_f(x);
      hi[m * stride + r + j] = h;
      if constexpr (SPLIT) {
        const float hf = Ty<T>::to_f(h);
        lo[m * stride + r + j] = Ty<T>::from_f(fabsf(hf) <= 3.402823466e38f ? x - hf : 0.f);  // infinities are all in hi
      }
    }
  };
#pragma unroll 2
  for (int i = threadIdx.x; i < M * quads; i += threads) {
    const int m = i / quads, r = i % quads * 4;
    float t[4] = {};
    if (m < tile.count && r < rank) {
      const float4 u = sum(m, r);
      t[0] = u.x;
      t[1] = r + 1 < rank ? u.y : 0.f;  // ranks past the end hold nothing
      t[2] = r + 2 < rank ? u.z : 0.f;
      t[3] = r + 3 < rank ? u.w : 0.f;
    }
    if constexpr (SCALED) {
      *reinterpret_cast<float4*>(sums + m * vr + r) = make_float4(t[0], t[1], t[2], t[3]);
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) most = !(fabsf(t[j]) <= most) ? fabsf(t[j]) : most;  // NaN stays
      if (most != 0.f) atomicMax(row_max + m, __float_as_uint(most));  // ordered like the floats; NaN above all
    } else {
      put(m, r, t, 1.f);
    }
  }
  __syncthreads();
  if constexpr (SCALED) {
    for (int m = threadIdx.x; m < M; m += threads) {
      const float most = __uint_as_float(row_max[m]);
      row_scale[m] = most > 0.f && most <= 1.7e38f ? ldexpf(1.f, min(126, max(-126, ilogbf(most)))) : 1.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < M * quads; i += threads) {
      const int m = i / quads, r = i % quads * 4;
      const float4 u = *reinterpret_cast<const float4*>(sums + m * vr + r);
      const float t[4] = {u.x, u.y, u.z, u.w};
      put(m, r, t, 1.f / row_scale[m]);
    }
    __syncthreads();
  }
}

// v of a sorted tile's row from the splits' parts, in order.
struct SumParts {
  const float* v;
  const int* rows;
  int64_t part;  // elements from one split's part to the next
  int splits, vr;
  float scale;
  __device__ float4 operator()(int m, int r) const {
    const float* p = v + static_cast<int64_t>(rows[m]) * vr + r;
    float4 u = *reinterpret_cast<const float4*>(p);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) {
      const float4 w = *reinterpret_cast<const float4*>(p + k * part);
      u.x += w.x;
      u.y += w.y;
      u.z += w.z;
      u.w += w.w;
    }
    return make_float4(u.x * scale, u.y * scale, u.z * scale, u.w * scale);
  }
};

// The product over chunk c of 16 staged rows (hi0 / lo0: this lane's place in
// row g) with 32 rows of B given by bf(j, chunk): adds to acc.
template <typename T, typename LoadB>
__device__ __forceinline__ void expand_chunk(float (&acc)[4][4], const T* hi0, const T* lo0, int stride, int c, LoadB bf) {
  constexpr int C = chunk_elems(sizeof(T));
  uint4 b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = bf(j, c);
  const uint4 a0 = *reinterpret_cast<const uint4*>(hi0 + c * C);
  const uint4 a1 = *reinterpret_cast<const uint4*>(hi0 + 8 * stride + c * C);
#pragma unroll
  for (int j = 0; j < 4; ++j) Chunk<T>::mma(acc[j], a0, a1, b[j]);
  if constexpr (sizeof(T) == 2) {
    const uint4 l0 = *reinterpret_cast<const uint4*>(lo0 + c * C);
    const uint4 l1 = *reinterpret_cast<const uint4*>(lo0 + 8 * stride + c * C);
#pragma unroll
    for (int j = 0; j < 4; ++j) Chunk<T>::mma(acc[j], l0, l1, b[j]);
  }
}
// The same with the rows' few chunks kept in registers.
template <typename T, int NCH>
struct StagedRows {
  uint4 h0[NCH], h1[NCH], l0[NCH], l1[NCH];
  __device__ void load(const T* hi0, const T* lo0, int stride) {
    constexpr int C = chunk_elems(sizeof(T));
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      h0[c] = *reinterpret_cast<const uint4*>(hi0 + c * C);
      h1[c] = *reinterpret_cast<const uint4*>(hi0 + 8 * stride + c * C);
      l0[c] = *reinterpret_cast<const uint4*>(lo0 + c * C);
      l1[c] = *reinterpret_cast<const uint4*>(lo0 + 8 * stride + c * C);
    }
  }
  template <typename LoadB>
  __device__ void expand(float (&acc)[4][4], LoadB bf) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 b = bf(j, c);
        Chunk<T>::mma(acc[j], h0[c], h1[c], b);
        Chunk<T>::mma(acc[j], l0[c], l1[c], b);
      }
    }
  }
};
// This thread's eight columns of row g and of row g + 8.
__device__ __forceinline__ void block_values(const float (&acc)[4][4], float s0, float s1, float (&f0)[8], float (&f1)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f0[2 * j] = acc[j][0] * s0;
    f0[2 * j + 1] = acc[j][1] * s0;
    f1[2 * j] = acc[j][2] * s1;
    f1[2 * j + 1] = acc[j][3] * s1;
  }
}
// The column of a block of 32 that instruction 0 computes in row g of B;
// instruction j: 2 j further.
__device__ __forceinline__ int block_column(int g) { return (g >> 1) * 8 + (g & 1); }

// base and B in steps of 128 bytes of a row (64 or 32 columns), STAGES deep;
// NCH: 64-byte chunks of a row of B (up to two: v stays in registers).
// grid: (tiles, ranges of `range` columns); a warp has 16 rows.
template <typename T, int NCH, int STAGES>
__global__ void __launch_bounds__(kLargeThreads) lora_expand_kernel(const LoraArgs a, LoraPlan plan,
                                                                    const float* __restrict__ v, int splits,
                                                                    int64_t v_rank, int64_t range, uint32_t* err) {
  constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  constexpr int NS = 128 / sizeof(T);  // columns of a step
  constexpr int M = kLargeRows;
  constexpr bool SCALED = std::is_same<T, __half>::value;
  __shared__ int rows[M];
  __shared__ float row_scale[M];
  __shared__ unsigned row_max[M];
  extern __shared__ __align__(128) uint8_t smem[];
  griddep_launch_dependents();
  griddep_wait();
  const Tile tile = planned_tile(plan, rows);
  if (tile.count == 0) return;
  const int64_t col0 = blockIdx.y * range, col1 = min(a.n, col0 + range);
  if (tile.group >= a.adapters) {
    fill_rows<T>(a, tile, rows, col0, col1, true, err);
    return;
  }
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  constexpr int vr = NCH * C, stride = vr + E;
  constexpr int kBase = M * 128, kStage = kBase + NS * NCH * 64;
  T* hi = reinterpret_cast<T*>(smem + STAGES * kStage);
  T* lo = hi + M * stride;

  // this thread's copies of a step: 16 bytes `vec` of every sixteenth row of
  // base, and of every kBStep-th row of B
  const int vec = t & 7, row0 = t >> 3;
  constexpr int kBVecs = NCH * 4, kBStep = kBVecs > kLargeThreads ? 1 : kLargeThreads / kBVecs;
  static_assert(kBVecs <= kLargeThreads, "a row of B has at most one vector for each thread");
  const int b_vec = t % kBVecs, b_row0 = t / kBVecs;
  const bool with_base = a.base != nullptr;
  const T* bp[4];
  bool has_row[4];
  uint32_t base_dst[4];
  const uint32_t ring = smem_u32(smem);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row0 + 16 * i;
    has_row[i] = r < tile.count;
    bp[i] = static_cast<const T*>(a.base) + static_cast<int64_t>(rows[has_row[i] ? r : 0]) * a.base_stride + col0 + vec * E;
    base_dst[i] = ring + tile_offset(r, 2, vec >> 2, vec & 3);
  }
  const T* b = static_cast<const T*>(a.b) + (static_cast<int64_t>(tile.group) * a.n + col0 + b_row0) * a.rank + b_vec * E;
  const bool b_in = b_vec * E < a.rank;
  const int64_t b_step = static_cast<int64_t>(kBStep) * a.rank;
  const int cols = static_cast<int>(col1 - col0);
  const int steps = (cols + NS - 1) / NS;
  auto load = [&](int step, int stage) {
    if (step < steps) {
      const int col = step * NS;
      const uint32_t at = stage * kStage;
      if (with_base) {
        const bool in = col + vec * E < cols;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = in && has_row[i];
          copy16(base_dst[i] + at, ok ? bp[i] + col : a.base, ok);
        }
      }
      const T* src = b + static_cast<int64_t>(col) * a.rank;
#pragma unroll
      for (int r = 0; r < NS; r += kBStep, src += b_step) {
        const bool ok = b_in && col + r + b_row0 < cols;
        copy16(ring + at + kBase + tile_offset(r + b_row0, NCH, b_vec >> 2, b_vec & 3), ok ? src : a.b, ok);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(i, i);
  const SumParts sum{v, rows, a.tokens * v_rank, splits, vr, a.scaling != nullptr ? a.scaling[tile.group] : 1.f};
  stage_v<T, M>(tile, static_cast<int>(a.rank), vr, stride, hi, lo, reinterpret_cast<float*>(lo + M * stride), row_scale,
                row_max, sum);
  const int g = lane >> 2, q = lane & 3, m0 = warp * 16;
  const bool in0 = m0 + g < tile.count, in1 = m0 + g + 8 < tile.count;
  const float s0 = SCALED ? row_scale[m0 + g] : 1.f, s1 = SCALED ? row_scale[m0 + g + 8] : 1.f;
  const T* hi0 = hi + (m0 + g) * stride + q * E;
  const T* lo0 = lo + (m0 + g) * stride + q * E;
  T* out0 = static_cast<T*>(a.out) + static_cast<int64_t>(rows[in0 ? m0 + g : 0]) * a.out_stride + col0 + q * 8;
  T* out1 = static_cast<T*>(a.out) + static_cast<int64_t>(rows[in1 ? m0 + g + 8 : 0]) * a.out_stride + col0 + q * 8;
  constexpr bool HELD = NCH <= 2 && sizeof(T) == 2;
  StagedRows<T, HELD ? NCH : 1> held;
  if constexpr (HELD) held.load(hi0, lo0, stride);
  int stage = 0;
  for (int step = 0; step < steps; ++step, out0 += NS, out1 += NS) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();  // the step's bytes are there, and the stage before it is free
    load(step + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
    const uint8_t* es = smem + stage * kStage;
    const uint8_t* bs = es + kBase;
    if (m0 < tile.count) {
#pragma unroll
      for (int blk = 0; blk < NS / 32; ++blk) {
        float acc[4][4] = {};
        auto bf = [&](int j, int c) { return lds16(bs + tile_offset(blk * 32 + block_column(g) + 2 * j, NCH, c, q)); };
        if constexpr (HELD) {
          held.expand(acc, bf);
        } else {
#pragma unroll 2
          for (int c = 0; c < NCH; ++c) expand_chunk<T>(acc, hi0, lo0, stride, c, bf);
        }
        float f0[8], f1[8];
        block_values(acc, s0, s1, f0, f1);
        if (step * NS + blk * 32 + q * 8 < cols) {
          Eight<T> e0, e1;
#pragma unroll
          for (int i = 0; i < Eight<T>::W; ++i) {
            const int w = (blk * 4 + q) * Eight<T>::W + i;  // 16-byte vector of the row
            e0.u[i] = lds16(es + tile_offset(m0 + g, 2, w >> 2, w & 3));
            e1.u[i] = lds16(es + tile_offset(m0 + g + 8, 2, w >> 2, w & 3));
          }
          if (in0) store_sum<T>(out0 + blk * 32, e0, with_base, f0);
          if (in1) store_sum<T>(out1 + blk * 32, e1, with_base, f1);
        }
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Any alignment: B, base and out element by element. Grid as above.
template <typename T>
__global__ void __launch_bounds__(kLargeThreads) lora_expand_any_kernel(const LoraArgs a, LoraPlan plan,
                                                                        const float* __restrict__ v, int splits,
                                                                        int64_t v_rank, int64_t range, int b_width,
                                                                        uint32_t* err) {
  constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  constexpr int M = kLargeRows;
  constexpr bool SCALED = std::is_same<T, __half>::value;
  __shared__ int rows[M];
  __shared__ float row_scale[M];
  __shared__ unsigned row_max[M];
  extern __shared__ __align__(128) uint8_t smem[];
  griddep_launch_dependents();
  griddep_wait();
  const Tile tile = planned_tile(plan, rows);
  if (tile.count == 0) return;
  const int64_t col0 = blockIdx.y * range, col1 = min(a.n, col0 + range);
  if (tile.group >= a.adapters) {
    fill_rows<T>(a, tile, rows, col0, col1, false, err);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int vr = static_cast<int>(v_rank);
  const int stride = vr + E;
  T* hi = reinterpret_cast<T*>(smem);
  T* lo = hi + M * stride;
  const SumParts sum{v, rows, a.tokens * v_rank, splits, vr, a.scaling != nullptr ? a.scaling[tile.group] : 1.f};
  stage_v<T, M>(tile, static_cast<int>(a.rank), vr, stride, hi, lo, reinterpret_cast<float*>(lo + M * stride), row_scale,
                row_max, sum);
  const int g = lane >> 2, q = lane & 3, m0 = warp * 16;
  if (m0 >= tile.count) return;
  const bool in0 = m0 + g < tile.count, in1 = m0 + g + 8 < tile.count;
  const int64_t t0 = rows[in0 ? m0 + g : 0], t1 = rows[in1 ? m0 + g + 8 : 0];
  const float s0 = SCALED ? row_scale[m0 + g] : 1.f, s1 = SCALED ? row_scale[m0 + g + 8] : 1.f;
  const T* hi0 = hi + (m0 + g) * stride + q * E;
  const T* lo0 = lo + (m0 + g) * stride + q * E;
  const T* b = static_cast<const T*>(a.b) + static_cast<int64_t>(tile.group) * a.n * a.rank;
  const T* base = static_cast<const T*>(a.base);
  T* out = static_cast<T*>(a.out);
  for (int64_t n0 = col0; n0 < col1; n0 += 32) {
    float acc[4][4] = {};
    for (int c = 0; c < vr / C; ++c) {
      expand_chunk<T>(acc, hi0, lo0, stride, c, [&](int j, int k) {
        const int64_t col = n0 + block_column(g) + 2 * j;
        return load_chunk<T>(col < a.n ? b + col * a.rank : nullptr, k * C + q * E, a.rank, b_width);
      });
    }
    float f0[8], f1[8];
    block_values(acc, s0, s1, f0, f1);
    const int64_t at = n0 + q * 8, left = a.n - at;
    if (in0) store_each<T>(out + t0 * a.out_stride + at, base ? base + t0 * a.base_stride + at : nullptr, left, f0);
    if (in1) store_each<T>(out + t1 * a.out_stride + at, base ? base + t1 * a.base_stride + at : nullptr, left, f1);
  }
}

// ---- few tokens: one launch ------------------------------------------------------------
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 16 bytes to a cluster address; their arrival is counted by the mbarrier at `bar` in the same CTA.
__device__ __forceinline__ void push16(uint32_t addr, float4 v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
               "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)), "r"(__float_as_uint(v.w)),
               "r"(bar)
               : "memory");
}

struct SmallWidths {  // elements that rows are aligned to: of x and A, of B; whole vectors of out and base
  int k, b;
  bool n;
};

// A cluster of CTAs (grid.x / tokens of them) takes the tile that row
// blockIdx.x / cluster leads. Its CTA c shrinks part c of K (a warp a part of
// that), sends its sums to all CTAs of the cluster, and expands part c of the
// columns. What such a launch takes is a chain of memory latencies (ids, x and
// A, the exchange), so every load is issued as early as its address is known:
// BATCH chunks of x and A at a time, the first B rows and base values before
// the exchange, and each next block's before the one at hand is computed.
template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(256) lora_small_kernel(const LoraArgs a, int cluster, SmallWidths given, int64_t v_rank,
                                                         uint32_t* err) {
  // aligned calls (VEC) are compiled without the other widths: a launch this short waits for its instructions too
  const SmallWidths width = VEC ? SmallWidths{16 / sizeof(T), 16 / sizeof(T), true} : given;
  constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  constexpr int M = kSmallRows, RB = 8 * NT;  // ranks of a pass
  constexpr int BATCH = NT == 2 ? 4 : NT == 4 ? 2 : 1;
  constexpr bool SCALED = std::is_same<T, __half>::value;
  __shared__ int rows[M], scratch[9];
  __shared__ float row_scale[M];
  __shared__ unsigned row_max[M];
  __shared__ uint64_t received;
  extern __shared__ __align__(128) uint8_t smem[];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  if (t == 0) {
    mbar_init(&received, 1);
    fence_mbar_init();
  }
  __syncwarp();
  cluster_arrive();  // the barriers of the cluster's CTAs exist when all have arrived
  griddep_launch_dependents();
  griddep_wait();
  const int lead = static_cast<int>(blockIdx.x) / cluster, part = static_cast<int>(blockIdx.x) % cluster;
  const Tile tile = find_tile(a, lead, rows, scratch);
  if (tile.count == 0) {  // of the whole cluster
    cluster_wait();
    return;
  }
  const int64_t blocks = (a.n + 31) / 32;
  const int64_t col0 = blocks * part / cluster * 32, col1 = min(a.n, blocks * (part + 1) / cluster * 32);
  if (tile.group >= a.adapters) {
    fill_rows<T>(a, tile, rows, col0, col1, width.n, err);
    __syncwarp();
    cluster_wait();
    return;
  }
  const int g = lane >> 2, q = lane & 3;
  const int vr = static_cast<int>(v_rank), rank = static_cast<int>(a.rank);
  const int stride = vr + E, quads = (rank + 3) / 4;
  float* parts = reinterpret_cast<float*>(smem);  // [cluster][M][vr]: the CTAs' parts of v
  T* hi = reinterpret_cast<T*>(smem + sizeof(float) * cluster * M * vr);
  T* lo = hi + M * stride;
  float* staged = reinterpret_cast<float*>(lo + (sizeof(T) == 2 ? M * stride : 0));  // [M][vr] for fp16
  auto* red = reinterpret_cast<float(*)[M][RB + 4]>(staged + (SCALED ? M * vr : 0));  // [kSmallWarps]
  if (t == 0) mbar_arrive_expect_tx(&received, static_cast<uint32_t>(cluster * tile.count * quads * 16));
  const bool in0 = g < tile.count, in1 = g + 8 < tile.count;
  const int64_t t0 = rows[in0 ? g : 0], t1 = rows[in1 ? g + 8 : 0];
  // shrink
  const T* x0 = in0 ? static_cast<const T*>(a.x) + t0 * a.x_stride : nullptr;
  const T* x1 = in1 ? static_cast<const T*>(a.x) + t1 * a.x_stride : nullptr;
  int c0, c1;
  split_range((a.k + C - 1) / C, cluster * kSmallWarps, part * kSmallWarps + warp, &c0, &c1);
  const uint32_t my_part = smem_u32(parts + part * M * vr), bar = smem_u32(&received);
  for (int r0 = 0; r0 < rank; r0 += RB) {
    const T* w[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = r0 + j * 8 + g;
      w[j] = r < rank ? static_cast<const T*>(a.a) + (static_cast<int64_t>(tile.group) * rank + r) * a.k : nullptr;
    }
    float acc[NT][4] = {};
    for (int c = c0; c < c1; c += BATCH) {
      uint4 x0c[BATCH], x1c[BATCH], wc[BATCH][NT];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int64_t at = c + i < c1 ? static_cast<int64_t>(c + i) * C + q * E : a.k;  // past the end: zeros
        x0c[i] = load_chunk<T>(x0, at, a.k, width.k);
        x1c[i] = load_chunk<T>(x1, at, a.k, width.k);
#pragma unroll
        for (int j = 0; j < NT; ++j) wc[i][j] = load_chunk<T>(w[j], at, a.k, width.k);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j) Chunk<T>::mma(acc[j], x0c[i], x1c[i], wc[i][j]);
      }
    }
    if (r0 > 0) __syncthreads();  // the pass before has been read
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      *reinterpret_cast<float2*>(&red[warp][g][j * 8 + 2 * q]) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(&red[warp][g + 8][j * 8 + 2 * q]) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    if (r0 == 0) cluster_wait();
    const int here = min(RB / 4, quads - r0 / 4);  // quads of this pass
    for (int i = t; i < tile.count * here; i += 256) {
      const int m = i / here, r = i % here * 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kSmallWarps; ++k) {
        const float4 u = *reinterpret_cast<const float4*>(&red[k][m][r]);
        s.x += u.x;
        s.y += u.y;
        s.z += u.z;
        s.w += u.w;
      }
      const uint32_t dst = my_part + (m * vr + r0 + r) * 4;
      for (int k = 0; k < cluster; ++k) push16(mapa_shared(dst, k), s, mapa_shared(bar, k));
    }
  }
  // the first block of this warp's columns, ahead of the exchange
  const T* b = static_cast<const T*>(a.b) + static_cast<int64_t>(tile.group) * a.n * rank;
  const T* base0 = a.base != nullptr ? static_cast<const T*>(a.base) + t0 * a.base_stride + q * 8 : nullptr;
  const T* base1 = a.base != nullptr ? static_cast<const T*>(a.base) + t1 * a.base_stride + q * 8 : nullptr;
  auto b_chunk = [&](int64_t n0, int j, int c) {
    const int64_t col = n0 + block_column(g) + 2 * j;
    return load_chunk<T>(col < col1 ? b + col * rank : nullptr, c * C + q * E, rank, width.b);
  };
  struct Block {
    uint4 b[4];
    Eight<T> e0, e1;
  };
  auto load_block = [&](Block& k, int64_t n0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) k.b[j] = b_chunk(n0, j, 0);
    if (width.n && base0 != nullptr && n0 + q * 8 < col1) {
      if (in0) load_eight(k.e0, base0 + n0);
      if (in1) load_eight(k.e1, base1 + n0);
    }
  };
  const int64_t first = col0 + warp * 32;
  Block next{};
  load_block(next, first);
  const float scale = a.scaling != nullptr ? a.scaling[tile.group] : 1.f;
  if (!mbar_wait(&received, 0, err, ERR_WAIT_TIMEOUT_OTHER)) return;
  // v: the parts of the cluster's CTAs in order
  stage_v<T, M>(tile, rank, vr, stride, hi, lo, staged, row_scale, row_max, [&](int m, int r) {
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < cluster; ++k) {
      const float4 w = *reinterpret_cast<const float4*>(parts + (k * M + m) * vr + r);
      u.x += w.x;
      u.y += w.y;
      u.z += w.z;
      u.w += w.w;
    }
    return make_float4(u.x * scale, u.y * scale, u.z * scale, u.w * scale);
  });
  const float s0 = SCALED ? row_scale[g] : 1.f, s1 = SCALED ? row_scale[g + 8] : 1.f;
  const T* hi0 = hi + g * stride + q * E;
  const T* lo0 = lo + g * stride + q * E;
  T* out0 = static_cast<T*>(a.out) + t0 * a.out_stride + q * 8;
  T* out1 = static_cast<T*>(a.out) + t1 * a.out_stride + q * 8;
  for (int64_t n0 = first; n0 < col1; n0 += kSmallWarps * 32) {
    const Block now = next;
    if (n0 + kSmallWarps * 32 < col1) load_block(next, n0 + kSmallWarps * 32);
    float acc[4][4] = {};
    expand_chunk<T>(acc, hi0, lo0, stride, 0, [&](int j, int) { return now.b[j]; });
    for (int c = 1; c < vr / C; ++c) expand_chunk<T>(acc, hi0, lo0, stride, c, [&](int j, int k) { return b_chunk(n0, j, k); });
    float f0[8], f1[8];
    block_values(acc, s0, s1, f0, f1);
    const int64_t left = col1 - n0 - q * 8;
    if (width.n) {
      if (left > 0 && in0) store_sum<T>(out0 + n0, now.e0, base0 != nullptr, f0);
      if (left > 0 && in1) store_sum<T>(out1 + n0, now.e1, base1 != nullptr, f1);
    } else {
      if (in0) store_each<T>(out0 + n0, base0 != nullptr ? base0 + n0 : nullptr, left, f0);
      if (in1) store_each<T>(out1 + n0, base1 != nullptr ? base1 + n0 : nullptr, left, f1);
    }
  }
}

// ---- host ----------------------------------------------------------------------------
namespace {
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

bool small_call(int64_t tokens) { return tokens <= kSmallTokens; }

struct Launch {  // of many tokens
  int64_t tiles;   // upper bound
  int64_t likely;  // tiles to expect
  int splits;
  int64_t v_rank;
  size_t v_bytes, perm_bytes, tile_bytes;
  size_t total() const { return v_bytes + perm_bytes + tile_bytes + 256; }
};

Launch plan_launch(int64_t tokens, int64_t adapters, int64_t rank, int64_t k, int dtype) {
  const int esize = dtype == F32 ? 4 : 2;
  Launch l{};
  l.tiles = tokens / kLargeRows + std::min(tokens, adapters + 2);
  l.likely = (tokens + kLargeRows - 1) / kLargeRows;
  l.v_rank = padded_rank(rank, esize);
  // about four CTAs for every SM, and at least four steps of 128 bytes for a CTA
  const int64_t steps = (k * esize + 127) / 128;
  const int64_t ctas = static_cast<int64_t>(num_sms()) * 4;
  l.splits = static_cast<int>(std::min<int64_t>({16, std::max<int64_t>(1, steps / 4), std::max<int64_t>(1, ctas / l.likely)}));
  l.v_bytes = round256(sizeof(float) * l.splits * tokens * l.v_rank);
  l.perm_bytes = round256(sizeof(int) * tokens);
  l.tile_bytes = round256(sizeof(int4) * l.tiles);
  return l;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_grid(void (*kernel)(KArgs...), dim3 grid, int block, int cluster, size_t smem, cudaStream_t st,
                        Args&&... args) {
  // a little more than asked for: the limit without the attribute includes the kernel's static arrays
  if (const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem + 4096); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Elements that rows of `length` starting at p (and `stride` apart) are aligned to: 16 bytes' worth, 8's, or 1.
template <typename T>
int row_width(const void* p, int64_t length, int64_t stride) {
  for (int e = 16 / sizeof(T); e > static_cast<int>(4 / sizeof(T)); e /= 2) {
    if (reinterpret_cast<uintptr_t>(p) % (e * sizeof(T)) == 0 && length % e == 0 && stride % e == 0) return e;
  }
  return 1;
}

template <typename T>
bool output_vectors(const LoraArgs& a) {
  constexpr int E = 16 / sizeof(T);
  const bool one = a.tokens == 1;
  return a.n % 8 == 0 && aligned16(a.out) && (one || a.out_stride % E == 0) &&
         (a.base == nullptr || (aligned16(a.base) && (one || a.base_stride % E == 0)));
}

template <typename T>
cudaError_t launch_small(const LoraArgs& a, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const int64_t v_rank = padded_rank(a.rank, sizeof(T));
  const int kw = std::min(row_width<T>(a.x, a.k, a.tokens == 1 ? 0 : a.x_stride), row_width<T>(a.a, a.k, 0));
  const SmallWidths width{kw, row_width<T>(a.b, a.rank, 0), output_vectors<T>(a)};
  // enough CTAs that a warp has about two chunks of K and two blocks of columns
  const int64_t chunks = (a.k + chunk_elems(sizeof(T)) - 1) / chunk_elems(sizeof(T));
  const int64_t want = std::max(chunks / (2 * kSmallWarps), a.n / (2 * 32 * kSmallWarps));
  int cluster = 1;
  while (cluster < kMaxCluster && cluster < want && 2 * cluster * a.tokens <= 2 * num_sms() && 2 * cluster * v_rank <= 512)
    cluster *= 2;
  const size_t smem = kSmallRows * (sizeof(float) * v_rank * cluster + (sizeof(T) == 2 ? 2 : 1) * sizeof(T) * (v_rank + E) +
                                    (std::is_same<T, __half>::value ? sizeof(float) * v_rank : 0));
  auto launch = [&](auto* kernel, int nt) {
    const size_t red = sizeof(float) * kSmallWarps * kSmallRows * (8 * nt + 4);
    return launch_grid(kernel, dim3(static_cast<unsigned>(a.tokens * cluster)), 256, cluster, smem + red, st, a, cluster,
                       width, v_rank, error_word_ptr());
  };
  const bool vec = width.k == E && width.b == E && width.n;
  if (a.rank <= 16) return vec ? launch(lora_small_kernel<T, 2, true>, 2) : launch(lora_small_kernel<T, 2, false>, 2);
  if (a.rank <= 32) return vec ? launch(lora_small_kernel<T, 4, true>, 4) : launch(lora_small_kernel<T, 4, false>, 4);
  return vec ? launch(lora_small_kernel<T, 8, true>, 8) : launch(lora_small_kernel<T, 8, false>, 8);
}

template <typename T>
cudaError_t launch_large(const LoraArgs& a, void* ws, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T), STAGES = 4;
  const Launch l = plan_launch(a.tokens, a.adapters, a.rank, a.k, a.dtype);
  char* p = static_cast<char*>(ws);
  float* v = reinterpret_cast<float*>(p);
  LoraPlan plan{};
  plan.perm = reinterpret_cast<int*>(p + l.v_bytes);
  plan.tiles = reinterpret_cast<int4*>(p + l.v_bytes + l.perm_bytes);
  plan.num_tiles = reinterpret_cast<int*>(p + l.v_bytes + l.perm_bytes + l.tile_bytes);
  cudaError_t e = launch_grid(lora_plan_kernel, dim3(1), kPlanThreads, 0, sizeof(int) * static_cast<size_t>(a.adapters + 2),
                              st, a, plan);
  if (e != cudaSuccess) return e;

  const bool vec_k = row_width<T>(a.x, a.k, a.x_stride) == E && row_width<T>(a.a, a.k, 0) == E;
  auto shrink = [&](auto* kernel, auto* any, int nt, int stages) {
    const dim3 grid(static_cast<unsigned>(l.tiles), static_cast<unsigned>(l.splits),
                    static_cast<unsigned>((a.rank + 8 * nt - 1) / (8 * nt)));
    return vec_k ? launch_grid(kernel, grid, kLargeThreads, 0, static_cast<size_t>(stages) * (kLargeRows + 8 * nt) * 128, st,
                               a, plan, v, l.splits, l.v_rank)
                 : launch_grid(any, grid, kLargeThreads, 0, 0, st, a, plan, v, l.splits, l.v_rank);
  };
  if (a.rank <= 16) {
    e = shrink(lora_shrink_kernel<T, 2, STAGES>, lora_shrink_any_kernel<T, 2>, 2, STAGES);
  } else if (a.rank <= 32) {
    e = shrink(lora_shrink_kernel<T, 4, STAGES>, lora_shrink_any_kernel<T, 4>, 4, STAGES);
  } else {
    e = shrink(lora_shrink_kernel<T, 8, STAGES>, lora_shrink_any_kernel<T, 8>, 8, STAGES);
  }
  if (e != cudaSuccess) return e;

  const int b_width = row_width<T>(a.b, a.rank, 0);
  const int64_t unit = 128 / sizeof(T);  // columns of a step
  const int64_t units = (a.n + unit - 1) / unit;
  const int64_t ranges = std::min<int64_t>(units, std::max<int64_t>(1, num_sms() * 4 / l.likely));
  const int64_t range = (units + ranges - 1) / ranges * unit;
  const dim3 grid(static_cast<unsigned>(l.tiles), static_cast<unsigned>((a.n + range - 1) / range));
  // hi and lo, and for fp16 the fp32 sums that they are made from
  const size_t staged = kLargeRows * ((sizeof(T) == 2 ? 2 : 1) * sizeof(T) * (l.v_rank + E) +
                                      (std::is_same<T, __half>::value ? sizeof(float) * l.v_rank : 0));
  if (b_width == E && output_vectors<T>(a)) {
    auto expand = [&](auto* kernel, int stages) {
      const size_t stage = kLargeRows * 128 + unit * l.v_rank * sizeof(T);
      return launch_grid(kernel, grid, kLargeThreads, 0, stages * stage + staged, st, a, plan, static_cast<const float*>(v),
                         l.splits, l.v_rank, range, error_word_ptr());
    };
    const int64_t chunks = l.v_rank * static_cast<int64_t>(sizeof(T)) / 64;
    if (chunks == 1) return expand(lora_expand_kernel<T, 1, 3>, 3);
    if (chunks == 2) return expand(lora_expand_kernel<T, 2, 3>, 3);
    if (chunks == 4) return expand(lora_expand_kernel<T, 4, 3>, 3);
    if constexpr (sizeof(T) == 4) {
      if (chunks == 16) return expand(lora_expand_kernel<T, 16, 2>, 2);
    }
    return expand(lora_expand_kernel<T, 8, 2>, 2);  // fp16: 217 KB with two stages
  }
  return launch_grid(lora_expand_any_kernel<T>, grid, kLargeThreads, 0, staged, st, a, plan, static_cast<const float*>(v),
                     l.splits, l.v_rank, range, b_width, error_word_ptr());
}

template <typename T>
cudaError_t launch_type(const LoraArgs& a, void* ws, cudaStream_t st) {
  return small_call(a.tokens) ? launch_small<T>(a, st) : launch_large<T>(a, ws, st);
}
}  // namespace

size_t lora_workspace_bytes(int64_t tokens, int64_t adapters, int64_t rank, int64_t k, int dtype) {
  return small_call(tokens) ? 0 : plan_launch(tokens, adapters, rank, k, dtype).total();
}

cudaError_t lora_launch(const LoraArgs& a, void* ws, cudaStream_t st) {
  if (a.dtype == F16) return launch_type<__half>(a, ws, st);
  if (a.dtype == BF16) return launch_type<__nv_bfloat16>(a, ws, st);
  return launch_type<float>(a, ws, st);
}

}  // namespace tfo
