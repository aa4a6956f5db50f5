// Low-rank adapters of many requests beside a shared projection.
//
//   out[t] = base[t] + scaling[i] * B[i] (A[i] x[t]),   i = ids[t]
//   x [tokens, K], A [adapters, rank, K], B [adapters, N, rank];
//   i < 0: out[t] = base[t]; i >= adapters: NaN, and the device error word.
//
// Two steps with the low-rank values v = A x in fp32 between them:
//   shrink: v[split, t, :] = the sum over a part of K
//   expand: v = scaling * sum over splits, out = base + B v
// Rows that use the same adapter are grouped into tiles, so that an adapter's
// matrices are read once per tile and not once per row:
//   few tokens: every CTA finds its own tile of 16 rows from the ids (row i
//     leads a tile if 0, 16, 32, ... rows before it use the same adapter);
//   many: a one-CTA kernel sorts the rows by adapter into tiles of 64 first.
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
#include "capi_internal.h"
#include "common.cuh"

namespace tfo {

constexpr int kSmallTokens = 256;  // at most: each CTA reads all ids (one per thread)
constexpr int kSmallRows = 16, kSmallWarps = 8;
constexpr int kLargeRows = 64, kLargeWarps = 4;

__host__ __device__ constexpr int chunk_elems(int esize) { return 64 / esize; }  // summed elements per 64-byte chunk
__host__ __device__ inline int64_t padded_rank(int64_t rank, int esize) {
  const int c = chunk_elems(esize);
  return (rank + c - 1) / c * c;
}

// ---- tensor instructions ------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
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
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_chunk(const T* row, int64_t i, int64_t limit) {
  constexpr int E = 16 / sizeof(T);
  if (row == nullptr || i >= limit) return make_uint4(0, 0, 0, 0);
  if constexpr (VEC) return *reinterpret_cast<const uint4*>(row + i);  // limit is a multiple of E
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

template <bool SMALL>
__device__ __forceinline__ Tile this_tile(const LoraArgs& a, const LoraPlan& plan, int* rows, int* scratch) {
  if constexpr (SMALL) {
    return find_tile(a, blockIdx.x, rows, scratch);
  } else {
    if (static_cast<int>(blockIdx.x) >= *plan.num_tiles) return Tile{0, 0};
    const int4 t = plan.tiles[blockIdx.x];
    if (threadIdx.x < t.z) rows[threadIdx.x] = plan.perm[t.y + threadIdx.x];
    __syncthreads();
    return Tile{t.x, t.z};
  }
}

// Sorts the rows by group (the order inside a group is free) and cuts the
// groups into tiles. One CTA; bins: [groups] in shared memory.
__global__ void __launch_bounds__(1024) lora_plan_kernel(const LoraArgs a, LoraPlan plan) {
  extern __shared__ int bins[];  // [groups] counts, then the next free place; [groups] tiles
  __shared__ int carry[2], warp_sum_rows[32], warp_sum_tiles[32];
  griddep_launch_dependents();
  griddep_wait();
  const int groups = static_cast<int>(a.adapters) + 2;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  for (int i = t; i < groups; i += 1024) bins[i] = 0;
  if (t < 2) carry[t] = 0;
  __syncthreads();
  const int tokens = static_cast<int>(a.tokens);
  for (int first = 0; first < tokens; first += 1024) {
    const int i = first + t;
    const int g = i < tokens ? row_group(a, i) : -1;
    const uint32_t peers = __match_any_sync(0xffffffffu, g);
    if (g >= 0 && lane == __ffs(peers) - 1) atomicAdd(&bins[g], __popc(peers));
  }
  __syncthreads();
  // exclusive prefix sums of rows and tiles over the groups, 1024 groups at a time
  for (int first = 0; first < groups; first += 1024) {
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
      warp_sum_rows[warp] = r;
      warp_sum_tiles[warp] = n;
    }
    __syncthreads();
    int before_r = carry[0], before_n = carry[1];
    for (int w = 0; w < warp; ++w) {
      before_r += warp_sum_rows[w];
      before_n += warp_sum_tiles[w];
    }
    const int row0 = before_r + r - count, tile0 = before_n + n - ntiles;
    if (g < groups) {
      bins[g] = row0;
      for (int i = 0; i < ntiles; ++i)
        plan.tiles[tile0 + i] = make_int4(g, row0 + i * kLargeRows, min(kLargeRows, count - i * kLargeRows), 0);
    }
    __syncthreads();
    if (t == 1023) {
      carry[0] = before_r + r;
      carry[1] = before_n + n;
    }
    __syncthreads();
  }
  if (t == 0) *plan.num_tiles = carry[1];
  for (int first = 0; first < tokens; first += 1024) {
    const int i = first + t;
    const int g = i < tokens ? row_group(a, i) : -1;
    const uint32_t peers = __match_any_sync(0xffffffffu, g);
    const int leader = __ffs(peers) - 1;
    int at = 0;
    if (g >= 0 && lane == leader) at = atomicAdd(&bins[g], __popc(peers));
    at = __shfl_sync(0xffffffffu, at, leader);
    if (g >= 0) plan.perm[at + __popc(peers & ((1u << lane) - 1))] = i;
  }
}

// ---- shrink: v = A x ---------------------------------------------------------------
// grid: (tiles, splits of K, blocks of 8 NT ranks). Few tokens: the warps share
// the tile's 16 rows and take parts of the split; many: 16 rows each.
template <typename T, int NT, bool SMALL, bool VEC>
__global__ void __launch_bounds__(SMALL ? 256 : 128) lora_shrink_kernel(const LoraArgs a, LoraPlan plan,
                                                                        float* __restrict__ v, int splits,
                                                                        int64_t v_rank) {
  constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  __shared__ int rows[kLargeRows], scratch[9];
  griddep_launch_dependents();
  griddep_wait();
  const Tile tile = this_tile<SMALL>(a, plan, rows, scratch);
  if (tile.count == 0 || tile.group >= a.adapters) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q = lane & 3;
  const int m0 = SMALL ? 0 : warp * 16;
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
  const int64_t chunks = (a.k + C - 1) / C;
  const int64_t parts = SMALL ? static_cast<int64_t>(splits) * kSmallWarps : splits;
  const int64_t part = SMALL ? static_cast<int64_t>(blockIdx.y) * kSmallWarps + warp : blockIdx.y;
  const int c0 = static_cast<int>(chunks * part / parts), c1 = static_cast<int>(chunks * (part + 1) / parts);
  float acc[NT][4] = {};
  if (SMALL || m0 < tile.count) {
#pragma unroll 2
    for (int c = c0; c < c1; ++c) {
      const int64_t i = static_cast<int64_t>(c) * C + q * E;
      const uint4 a0 = load_chunk<T, VEC>(x0, i, a.k), a1 = load_chunk<T, VEC>(x1, i, a.k);
      uint4 b[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j] = load_chunk<T, VEC>(w[j], i, a.k);
#pragma unroll
      for (int j = 0; j < NT; ++j) Chunk<T>::mma(acc[j], a0, a1, b[j]);
    }
  }
  v += static_cast<int64_t>(blockIdx.y) * a.tokens * v_rank + r0;
  if constexpr (SMALL) {
    // the warps' parts, added in order
    __shared__ float red[kSmallWarps][16][8 * NT + 2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      red[warp][g][j * 8 + 2 * q] = acc[j][0];
      red[warp][g][j * 8 + 2 * q + 1] = acc[j][1];
      red[warp][g + 8][j * 8 + 2 * q] = acc[j][2];
      red[warp][g + 8][j * 8 + 2 * q + 1] = acc[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tile.count * 8 * NT; i += 256) {
      const int m = i / (8 * NT), r = i % (8 * NT);
      if (r0 + r >= v_rank) continue;
      float t = 0.f;
#pragma unroll
      for (int s = 0; s < kSmallWarps; ++s) t += red[s][m][r];
      v[static_cast<int64_t>(rows[m]) * v_rank + r] = t;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = j * 8 + 2 * q;
      if (r0 + r >= v_rank) continue;  // v_rank is a multiple of 16
      if (m0 + g < tile.count)
        *reinterpret_cast<float2*>(v + static_cast<int64_t>(rows[m0 + g]) * v_rank + r) = make_float2(acc[j][0], acc[j][1]);
      if (m0 + g + 8 < tile.count)
        *reinterpret_cast<float2*>(v + static_cast<int64_t>(rows[m0 + g + 8]) * v_rank + r) =
            make_float2(acc[j][2], acc[j][3]);
    }
  }
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
// out = base + f (f alone without a base), columns at or past `limit` left out.
template <typename T, bool VEC>
__device__ __forceinline__ void store_eight(T* out, const Eight<T>& loaded, const T* base, int64_t limit, const float (&f)[8]) {
  if (limit <= 0) return;
  if constexpr (VEC) {
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < Eight<T>::W; ++i) reinterpret_cast<uint4*>(t)[i] = loaded.u[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = Ty<T>::from_f(base != nullptr ? Ty<T>::to_f(t[j]) + f[j] : f[j]);
#pragma unroll
    for (int i = 0; i < Eight<T>::W; ++i) reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(t)[i];
  } else {
    for (int j = 0; j < 8 && j < limit; ++j)
      out[j] = Ty<T>::from_f(base != nullptr ? Ty<T>::to_f(base[j]) + f[j] : f[j]);
  }
}

// Rows without a product: copied from base (or zero), or NaN for a bad id.
template <typename T, bool VEC>
__device__ __forceinline__ void fill_rows(const LoraArgs& a, const Tile& tile, const int* rows, int64_t col0, int64_t col1,
                                          uint32_t* err) {
  const bool bad = tile.group > a.adapters;
  if (bad && threadIdx.x == 0) set_error(err, ERR_BAD_ADAPTER);
  if (!bad && a.base == a.out) return;  // left as they are
  const float fill = bad ? __int_as_float(0x7fffffff) : 0.f;
  const float f[8] = {fill, fill, fill, fill, fill, fill, fill, fill};
  const int per_row = static_cast<int>((col1 - col0 + 7) / 8);
  for (int i = threadIdx.x; i < per_row * tile.count; i += blockDim.x) {
    const int64_t row = rows[i / per_row], col = col0 + i % per_row * 8;
    const T* base = a.base != nullptr ? static_cast<const T*>(a.base) + row * a.base_stride + col : nullptr;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + col;
    if constexpr (VEC) {
      if (!bad && base != nullptr) {  // bit for bit
        Eight<T> e;
        load_eight(e, base);
#pragma unroll
        for (int j = 0; j < Eight<T>::W; ++j) reinterpret_cast<uint4*>(out)[j] = e.u[j];
        continue;
      }
    }
    if (!bad && base != nullptr) {
      for (int j = 0; j < 8 && col + j < col1; ++j) out[j] = base[j];
    } else {
      Eight<T> none{};
      store_eight<T, VEC>(out, none, nullptr, col1 - col, f);
    }
  }
}

// The tile's v, summed over the splits and scaled, as operands in shared
// memory: hi and lo (SPLIT: 16-bit types), [M][stride]. fp16 rows are scaled by
// a power of two to at most 2 (row_scale takes it back), rows past the tile
// are zero.
template <typename T, int M, int THREADS>
__device__ __forceinline__ void stage_v(const LoraArgs& a, const Tile& tile, const int* rows, const float* __restrict__ v,
                                        int splits, int vr, int stride, T* hi, T* lo, float* sums, float* row_scale,
                                        unsigned* row_max) {
  constexpr bool SPLIT = sizeof(T) == 2;
  constexpr bool SCALED = std::is_same<T, __half>::value;
  const float s = a.scaling != nullptr ? a.scaling[tile.group] : 1.f;
  const int quads = vr / 4;  // a multiple of 4 (fp32) or 8
  const int rank = static_cast<int>(a.rank);
  if constexpr (SCALED) {
    for (int m = threadIdx.x; m < M; m += THREADS) row_max[m] = 0;
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
#pragma unroll 4
  for (int i = threadIdx.x; i < M * quads; i += THREADS) {
    const int m = i / quads, r = i % quads * 4;
    float t[4] = {};
    if (m < tile.count) {
      const float* p = v + static_cast<int64_t>(rows[m]) * vr + r;
      float4 u = *reinterpret_cast<const float4*>(p);
      for (int k = 1; k < splits; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(p + k * a.tokens * vr);
        u.x += w.x;
        u.y += w.y;
        u.z += w.z;
        u.w += w.w;
      }
      // ranks past the end were not written
      t[0] = r < rank ? u.x * s : 0.f;
      t[1] = r + 1 < rank ? u.y * s : 0.f;
      t[2] = r + 2 < rank ? u.z * s : 0.f;
      t[3] = r + 3 < rank ? u.w * s : 0.f;
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
    for (int m = threadIdx.x; m < M; m += THREADS) {
      const float most = __uint_as_float(row_max[m]);
      row_scale[m] = most > 0.f && most <= 1.7e38f ? ldexpf(1.f, min(126, max(-126, ilogbf(most)))) : 1.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < M * quads; i += THREADS) {
      const int m = i / quads, r = i % quads * 4;
      const float4 u = *reinterpret_cast<const float4*>(sums + m * vr + r);
      const float t[4] = {u.x, u.y, u.z, u.w};
      put(m, r, t, 1.f / row_scale[m]);
    }
    __syncthreads();
  }
}

// grid: (tiles, ranges of `range` columns, a multiple of 32). Few tokens: each
// warp takes every eighth block of 32 columns; many: each warp 16 rows.
template <typename T, bool SMALL, bool VEC, bool VECB>
__global__ void __launch_bounds__(SMALL ? 256 : 128) lora_expand_kernel(const LoraArgs a, LoraPlan plan,
                                                                        const float* __restrict__ v, int splits,
                                                                        int64_t v_rank, int64_t range, uint32_t* err) {
  constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  constexpr int M = SMALL ? kSmallRows : kLargeRows;
  constexpr int THREADS = SMALL ? 256 : 128;
  constexpr bool SPLIT = sizeof(T) == 2;                         // v as hi + lo
  constexpr bool SCALED = std::is_same<T, __half>::value;
  __shared__ int rows[kLargeRows], scratch[9];
  __shared__ float row_scale[M];
  __shared__ unsigned row_max[M];
  extern __shared__ __align__(16) uint8_t smem[];
  griddep_launch_dependents();
  griddep_wait();
  const Tile tile = this_tile<SMALL>(a, plan, rows, scratch);
  if (tile.count == 0) return;
  const int64_t col0 = blockIdx.y * range;
  const int64_t col1 = min(a.n, col0 + range);
  if (tile.group >= a.adapters) {
    fill_rows<T, VEC>(a, tile, rows, col0, col1, err);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int vr = static_cast<int>(v_rank);
  const int stride = vr + E;  // 16 bytes of padding
  T* hi = reinterpret_cast<T*>(smem);
  T* lo = hi + M * stride;
  stage_v<T, M, THREADS>(a, tile, rows, v, splits, vr, stride, hi, lo, reinterpret_cast<float*>(lo + M * stride), row_scale,
                         row_max);
  const int g = lane >> 2, q = lane & 3;
  const int m0 = SMALL ? 0 : warp * 16;
  if (m0 >= tile.count) return;
  const bool in0 = m0 + g < tile.count, in1 = m0 + g + 8 < tile.count;
  const int64_t t0 = rows[in0 ? m0 + g : 0], t1 = rows[in1 ? m0 + g + 8 : 0];
  const float s0 = SCALED ? row_scale[m0 + g] : 1.f, s1 = SCALED ? row_scale[m0 + g + 8] : 1.f;
  const T* hi0 = hi + (m0 + g) * stride + q * E;
  const T* lo0 = lo + (m0 + g) * stride + q * E;
  const T* b = static_cast<const T*>(a.b) + static_cast<int64_t>(tile.group) * a.n * a.rank;
  const T* base0 = a.base != nullptr ? static_cast<const T*>(a.base) + t0 * a.base_stride + q * 8 : nullptr;
  const T* base1 = a.base != nullptr ? static_cast<const T*>(a.base) + t1 * a.base_stride + q * 8 : nullptr;
  T* out0 = static_cast<T*>(a.out) + t0 * a.out_stride + q * 8;
  T* out1 = static_cast<T*>(a.out) + t1 * a.out_stride + q * 8;
  // the block's column that instruction j computes in this thread's row g of the second operand
  const int pick = (g >> 1) * 8 + (g & 1);
#pragma unroll 2
  for (int64_t n0 = col0 + (SMALL ? warp * 32 : 0); n0 < col1; n0 += SMALL ? kSmallWarps * 32 : 32) {
    const int64_t left = a.n - n0 - q * 8;  // columns from this thread's first on
    Eight<T> e0{}, e1{};
    if (VEC && base0 != nullptr && left > 0) {
      if (in0) load_eight(e0, base0 + n0);
      if (in1) load_eight(e1, base1 + n0);
    }
    float acc[4][4] = {};
    const T* brow[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t col = n0 + pick + 2 * j;
      brow[j] = col < a.n ? b + col * a.rank : nullptr;
    }
    for (int c = 0; c < vr; c += C) {
      uint4 bf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bf[j] = load_chunk<T, VECB>(brow[j], c + q * E, a.rank);
      const uint4 a0 = *reinterpret_cast<const uint4*>(hi0 + c);
      const uint4 a1 = *reinterpret_cast<const uint4*>(hi0 + 8 * stride + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) Chunk<T>::mma(acc[j], a0, a1, bf[j]);
      if constexpr (SPLIT) {
        const uint4 l0 = *reinterpret_cast<const uint4*>(lo0 + c);
        const uint4 l1 = *reinterpret_cast<const uint4*>(lo0 + 8 * stride + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) Chunk<T>::mma(acc[j], l0, l1, bf[j]);
      }
    }
    float f0[8], f1[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f0[2 * j] = acc[j][0] * s0;
      f0[2 * j + 1] = acc[j][1] * s0;
      f1[2 * j] = acc[j][2] * s1;
      f1[2 * j + 1] = acc[j][3] * s1;
    }
    if (in0) store_eight<T, VEC>(out0 + n0, e0, base0 != nullptr ? base0 + n0 : nullptr, left, f0);
    if (in1) store_eight<T, VEC>(out1 + n0, e1, base1 != nullptr ? base1 + n0 : nullptr, left, f1);
  }
}

// ---- host ----------------------------------------------------------------------------
namespace {
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

struct Launch {
  bool small;
  int64_t tiles;      // upper bound
  int64_t likely;     // tiles to expect
  int splits;
  int64_t v_rank;
  size_t v_bytes, perm_bytes, tile_bytes;
  size_t total() const { return v_bytes + perm_bytes + tile_bytes + 256; }
};

Launch plan_launch(int64_t tokens, int64_t adapters, int64_t rank, int64_t k, int dtype) {
  const int esize = dtype == F32 ? 4 : 2;
  Launch l{};
  l.small = tokens <= kSmallTokens;
  const int64_t groups = std::min(tokens, adapters + 2);
  l.tiles = l.small ? tokens : tokens / kLargeRows + groups;
  l.likely = l.small ? std::min(tokens, adapters) : (tokens + kLargeRows - 1) / kLargeRows;
  l.v_rank = padded_rank(rank, esize);
  const int64_t chunks = (k + chunk_elems(esize) - 1) / chunk_elems(esize);
  // enough CTAs for every SM, and at least two (few tokens) or eight chunks for a warp
  const int64_t ctas = static_cast<int64_t>(num_sms()) * (l.small ? 2 : 4);
  const int64_t most = std::max<int64_t>(1, chunks / (l.small ? 2 * kSmallWarps : 8));
  l.splits = static_cast<int>(std::min<int64_t>({16, most, std::max<int64_t>(1, ctas / l.likely)}));
  l.v_bytes = round256(sizeof(float) * l.splits * tokens * l.v_rank);
  if (!l.small) {
    l.perm_bytes = round256(sizeof(int) * tokens);
    l.tile_bytes = round256(sizeof(int4) * l.tiles);
  }
  return l;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_grid(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, cudaStream_t st, Args&&... args) {
  if (const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename T, bool SMALL>
cudaError_t launch_sized(const LoraArgs& a, const Launch& l, const LoraPlan& plan, float* v, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  constexpr int threads = 32 * (SMALL ? kSmallWarps : kLargeWarps);
  const bool vec_k = a.k % E == 0 && aligned16(a.x) && aligned16(a.a) && (a.tokens == 1 || a.x_stride % E == 0);
  const unsigned tiles = static_cast<unsigned>(l.tiles), splits = static_cast<unsigned>(l.splits);
  cudaError_t e;
#define TFO_SHRINK(NT)                                                                                                \
  e = vec_k ? launch_grid(lora_shrink_kernel<T, NT, SMALL, true>,                                                      \
                          dim3(tiles, splits, static_cast<unsigned>((a.rank + 8 * NT - 1) / (8 * NT))), threads, 0, st, \
                          a, plan, v, l.splits, l.v_rank)                                                              \
            : launch_grid(lora_shrink_kernel<T, NT, SMALL, false>,                                                     \
                          dim3(tiles, splits, static_cast<unsigned>((a.rank + 8 * NT - 1) / (8 * NT))), threads, 0, st, \
                          a, plan, v, l.splits, l.v_rank)
  if (a.rank <= 16) {
    TFO_SHRINK(2);
  } else if (a.rank <= 32) {
    TFO_SHRINK(4);
  } else {
    TFO_SHRINK(8);
  }
#undef TFO_SHRINK
  if (e != cudaSuccess) return e;
  const bool vec_n = a.n % 8 == 0 && aligned16(a.out) && (a.tokens == 1 || a.out_stride % E == 0) &&
                     (a.base == nullptr || (aligned16(a.base) && (a.tokens == 1 || a.base_stride % E == 0)));
  const bool vec_b = a.rank % E == 0 && aligned16(a.b);
  const int64_t unit = SMALL ? 32 * kSmallWarps : 128;  // columns of the shortest range
  const int64_t units = (a.n + unit - 1) / unit;
  const int64_t ranges = std::min(units, std::max<int64_t>(1, num_sms() * (SMALL ? 4 : 6) / l.likely));
  const int64_t range = (units + ranges - 1) / ranges * unit;
  const dim3 grid(tiles, static_cast<unsigned>((a.n + range - 1) / range));
  // hi and lo, and for fp16 the fp32 sums that they are made from
  const size_t smem = (SMALL ? kSmallRows : kLargeRows) *
                      ((sizeof(T) == 2 ? 2 : 1) * sizeof(T) * (l.v_rank + E) +
                       (std::is_same<T, __half>::value ? sizeof(float) * l.v_rank : 0));
  auto expand = [&](auto* kernel) {
    return launch_grid(kernel, grid, threads, smem, st, a, plan, static_cast<const float*>(v), l.splits, l.v_rank, range,
                       error_word_ptr());
  };
  if (vec_n) return vec_b ? expand(lora_expand_kernel<T, SMALL, true, true>) : expand(lora_expand_kernel<T, SMALL, true, false>);
  return vec_b ? expand(lora_expand_kernel<T, SMALL, false, true>) : expand(lora_expand_kernel<T, SMALL, false, false>);
}

template <typename T>
cudaError_t launch_type(const LoraArgs& a, void* ws, cudaStream_t st) {
  const Launch l = plan_launch(a.tokens, a.adapters, a.rank, a.k, a.dtype);
  char* p = static_cast<char*>(ws);
  float* v = reinterpret_cast<float*>(p);
  LoraPlan plan{};
  if (l.small) return launch_sized<T, true>(a, l, plan, v, st);
  plan.perm = reinterpret_cast<int*>(p + l.v_bytes);
  plan.tiles = reinterpret_cast<int4*>(p + l.v_bytes + l.perm_bytes);
  plan.num_tiles = reinterpret_cast<int*>(p + l.v_bytes + l.perm_bytes + l.tile_bytes);
  const cudaError_t e =
      launch_grid(lora_plan_kernel, dim3(1), 1024, sizeof(int) * static_cast<size_t>(a.adapters + 2), st, a, plan);
  return e != cudaSuccess ? e : launch_sized<T, false>(a, l, plan, v, st);
}
}  // namespace

size_t lora_workspace_bytes(int64_t tokens, int64_t adapters, int64_t rank, int64_t k, int dtype) {
  return plan_launch(tokens, adapters, rank, k, dtype).total();
}

cudaError_t lora_launch(const LoraArgs& a, void* ws, cudaStream_t st) {
  if (a.dtype == F16) return launch_type<__half>(a, ws, st);
  if (a.dtype == BF16) return launch_type<__nv_bfloat16>(a, ws, st);
  return launch_type<float>(a, ws, st);
}

}  // namespace tfo
