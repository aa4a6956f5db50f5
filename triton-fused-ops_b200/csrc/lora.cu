// Low-rank adapters of many requests beside a shared projection.
//
//   out[t] = base[t] + scaling[i] * B[i] (A[i] x[t]),   i = ids[t]
//   x [tokens, K], A [adapters, rank, K], B [adapters, N, rank];
//   i < 0: out[t] = base[t]; i >= adapters: NaN, and the device error word.
//
// Two steps with the low-rank values v = A x in fp32 between them:
//   shrink: v = the sum over K, cut into parts that are added in a fixed order
//   expand: out = base + B (scaling * v)
// both in one kernel, v never leaves the SMs.
// Rows that use the same adapter are grouped into tiles, so that an adapter's
// matrices are read once per tile and not once per row:
//   up to 384 tokens, one launch (lora_small_kernel): every CTA finds its tile
//     of up to 16 rows from the ids; a cluster of CTAs shares a tile, each
//     shrinks a part of K, sends its sums to the others' shared memory and
//     expands a part of the columns;
//   more: a kernel of one cluster sorts the rows by adapter into tiles of 64,
//     then a cluster of CTAs takes a tile in the same way, streaming x and A, then
//     base and B, through shared memory (lora_large_kernel).
// A row's result does not depend on the rows beside it in its tile.
//
// Both products run on m16n8 tensor instructions with rows of a tile as M.
// Their floor is memory (x, base and out once, A and B of the adapters that are
// there): a rank of 16 makes 16 flops for each byte. The order of the summed
// index inside a product is free, so thread q of four takes the 16 bytes
// [16 q, 16 q + 16) of a 64-byte chunk on both sides: every operand load, from
// global or shared memory, is a whole vector. Likewise the output columns of
// four instructions are dealt out so that a thread ends up with eight
// neighbouring ones.
//
// Measured (us; 4096 x 4096, bf16): one token of rank 16 4.3; 64 tokens over 32
// adapters 6.6, 256 over 16 8.5; 1024 over 16 17.9; 512 of rank 32 over 16 20.5;
// 8192 tokens of 16 adapters of rank 16 47, of rank 32 51, 63 % of the measured
// copy rate (rank 64 84, rank 128 171: the legacy tensor path's 530 TFLOP/s bounds
// those). fp32: 8192 tokens of rank 16 106, 32 156, 64 312, bound by splitting the
// operands and by three products. A form of the large kernel on tcgen05 (128-row
// tiles copied into swizzled shared memory, v as two values and the outputs in
// tensor memory) took 67 us at rank 32, 98 at 64 and 152 at 128: its steps'
// waits, proxy fences and barriers ran 750 cycles with one CTA on an SM.
//
// Rounding: products and sums are fp32 (long sums by rounded additions, see the
// shrink step and Chunk<float>: a tensor instruction cuts what it adds to). v enters
// the second product as a sum of values of x's type, cut so that they have v's
// sign (stage_v): three of bf16, all 24 bits; two of fp16, 22 bits (rows are scaled
// by a power of two to use fp16's whole range). With two of bf16, 16 bits, 2 of 1000
// outputs were not the nearest value to the 64-bit result, with three and rounded
// sums 1 to 3 of 10000, like an fp32 matrix product's. The third product costs
// where the products bound (8192 tokens of rank 32 47 -> 50 us, 64 72 -> 83, 128
// 135 -> 160); up to 16 ranks half of a chunk's instructions had multiplied zeros,
// and without them three are faster than two were (8192 tokens 48.7 -> 47.2, one
// token 4.6 -> 4.3). fp32 operands are split into two tf32 values on both sides
// and the three larger products are added. The result is rounded once.
#include <map>
#include <mutex>
#include <tuple>

#include "heads.cuh"

namespace tfo {

// At most: each CTA reads all ids (two per thread). Measured over five sets of
// adapters and sizes, this way / sorted: 300 tokens 10-15 / 14-21 us, 400
// 11-19 / 15-22, 512 15-25 / 16-23.
constexpr int kSmallTokens = 384;
constexpr int kSmallRows = 16, kSmallWarps = 8, kMaxCluster = 8;
constexpr int kLargeRows = 64, kLargeThreads = 256;

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
// x = hi + lo in two tf32 values of one sign, both infinite if x is, and neither
// of them zero unless x is (or below 2^-62): an infinity of the other operand then
// has the same sign in every product, where 0 * infinity or infinities of both
// signs would be a NaN. 2^-64 of x in place of a zero lo lies below what a tensor
// instruction keeps beside hi's product, so exact sums stay exact. hi is cut, not
// rounded (lo's sign), and the product of both lo, left out, is 2^-23 of the
// whole on average: results are 2.2e-7 to 3.2e-7 off 64 bits, 1.4e-7 to 2.0e-7
// with a rounded hi.
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = x & 0xffffe000u;  // cut
  const float f = __uint_as_float(x);
  const float rest = fmaxf(fabsf(f - __uint_as_float(hi)), fabsf(f * 0x1p-64f));  // infinity - infinity gives way
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(copysignf(rest, f)));
}

// d += the product over one 64-byte chunk: a0 / a1 are rows g and g + 8 of the
// first operand, b is row g of the second (lane = 4 g + q, q-th 16 bytes).
template <typename T> struct Chunk;
template <> struct Chunk<__half> {
  __device__ static void mma(float (&d)[4], const uint4& a0, const uint4& a1, const uint4& b) {
    mma_f16(d, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
    mma_f16(d, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
  }
  // over half of one, 32 bytes: thread q has the q-th 8
  __device__ static void mma(float (&d)[4], const uint2& a0, const uint2& a1, const uint2& b) {
    mma_f16(d, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
  }
};
template <> struct Chunk<__nv_bfloat16> {
  __device__ static void mma(float (&d)[4], const uint4& a0, const uint4& a1, const uint4& b) {
    mma_bf16(d, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
    mma_bf16(d, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
  }
  // over half of one, 32 bytes: thread q has the q-th 8
  __device__ static void mma(float (&d)[4], const uint2& a0, const uint2& a1, const uint2& b) {
    mma_bf16(d, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
  }
};
template <> struct Chunk<float> {
  // A chunk's sum starts at zero and is added to d by a rounded addition: the
  // tensor instructions cut their sum instead of rounding it, which over a long K
  // is a drift. Error of 1000 tokens of rank 256, K = 1024, against 64 bits 3.8e-6
  // without these additions, 3.2e-7 with them; 8192 tokens of 4096 x 4096, rank
  // 16 161 -> 106 us, 32 164 -> 156, 64 289 -> 312 (with the present split).
  __device__ static void mma(float (&d)[4], const uint4& a0, const uint4& a1, const uint4& b) {
    float t[4] = {};
    half(t, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
    half(t, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] += t[i];
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

// 8 bytes at row + i, likewise.
template <typename T>
__device__ __forceinline__ uint2 load_half(const T* row, int64_t i, int64_t limit, int width) {
  constexpr int E = 8 / sizeof(T);
  if (row == nullptr || i >= limit) return make_uint2(0, 0);
  if (width >= E) return *reinterpret_cast<const uint2*>(row + i);
  alignas(8) T t[E];
#pragma unroll
  for (int j = 0; j < E; ++j) t[j] = i + j < limit ? row[i + j] : Ty<T>::from_f(0.f);
  return *reinterpret_cast<const uint2*>(t);
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

// Tile `index` of at most kSmallTokens rows, by the whole CTA (256 threads of
// kIds rows each); rows gets its rows. A row leads a tile if 0, 16, 32, ...
// rows before it are of its group; tiles are counted in the order of their
// leaders.
constexpr int kIds = (kSmallTokens + 255) / 256;
__device__ __forceinline__ Tile find_tile(const LoraArgs& a, int index, int* rows, int* groups, int* scratch) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int tokens = static_cast<int>(a.tokens);
  int group[kIds], rank[kIds], before[kIds];  // rank: rows of the group before this one
  bool leads[kIds];
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    const int i = k * 256 + t;
    group[k] = i < tokens ? row_group(a, i) : -1;
    if (k * 256 < tokens) groups[i] = group[k];
  }
  if (t == 0) scratch[8 * kIds] = -1;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    rank[k] = before[k] = 0;
    leads[k] = false;
    if (k * 256 >= tokens) continue;
    const int end = k * 256 + t < tokens ? k * 256 + t : 0;
#pragma unroll 8
    for (int i = 0; i + 4 <= end; i += 4) {
      const int4 g = *reinterpret_cast<const int4*>(groups + i);
      rank[k] += (g.x == group[k]) + (g.y == group[k]) + (g.z == group[k]) + (g.w == group[k]);
    }
    for (int i = end & ~3; i < end; ++i) rank[k] += groups[i] == group[k];
    leads[k] = group[k] >= 0 && rank[k] % kSmallRows == 0;
    const uint32_t votes = __ballot_sync(0xffffffffu, leads[k]);
    if (lane == 0) scratch[k * 8 + warp] = __popc(votes);
    before[k] = __popc(votes & ((1u << lane) - 1));
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    if (k * 256 >= tokens) continue;
    for (int w = 0; w < k * 8 + warp; ++w) before[k] += scratch[w];
    if (leads[k] && before[k] == index) {
      scratch[8 * kIds] = k * 256 + t;
      scratch[8 * kIds + 1] = rank[k];
    }
  }
  __syncthreads();
  const int lead = scratch[8 * kIds];
  if (lead < 0) return Tile{0, 0};
  const int want = groups[lead];
  int count = 0;
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    if (k * 256 >= tokens) continue;
    const int place = rank[k] - scratch[8 * kIds + 1];
    const bool mine = group[k] == want && place >= 0 && place < kSmallRows;
    if (mine) rows[place] = k * 256 + t;
    count += __syncthreads_count(mine);
  }
  return Tile{want, count};
}

// A tile of the sorted rows, by the whole CTA.
__device__ __forceinline__ Tile planned_tile(const LoraPlan& plan, int index, int* rows) {
  const int4 t = plan.tiles[index];  // past the last tile: anything, not used
  if (index >= *plan.num_tiles) return Tile{0, 0};
  if (threadIdx.x < t.z) rows[threadIdx.x] = plan.perm[t.y + threadIdx.x];
  __syncthreads();
  return Tile{t.x, t.z};
}

// Sorts the rows by group (the order inside a group is free) and cuts the
// groups into tiles. One cluster of up to eight CTAs, each with a share of the
// rows, whose threads hold kHeld ids each: their loads are in flight together,
// and up to 8192 rows a CTA are read and counted once. The CTAs read each
// other's counts for the places of their rows. Measured: 8192 rows 7.7 us
// (one CTA 7.1 in order, more in random order), 65536 in order 9.7 us (51), in
// random order 14.7 us (101).
constexpr int kHeld = 8, kPlanThreads = 1024;

// Inclusive prefix sums over a warp.
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int p = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += p;
  }
  return v;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// `share`: rows of a CTA.
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const LoraArgs a, LoraPlan plan, int cluster, int64_t share) {
  extern __shared__ int bins[];  // [groups] rows of each in this CTA's share
  __shared__ int carry[2], sum_rows[32], sum_tiles[32];
  griddep_launch_dependents();
  griddep_wait();
  const int groups = static_cast<int>(a.adapters) + 2;
  int* const start = bins + groups;  // [groups] the first place of this CTA's rows
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, cta = static_cast<int>(blockIdx.x);
  const int64_t row0 = min(a.tokens, cta * share), end = min(a.tokens, row0 + share);
  constexpr int kStep = kHeld * kPlanThreads;
  int group[kHeld], place[kHeld];
  auto load = [&](int64_t first) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int64_t i = first + j * kPlanThreads + t;
      group[j] = i < end ? row_group(a, i) : -1;
    }
  };
  // adds the held rows to the bins; place: where the row comes in its bin
  auto count = [&](int* into, int64_t first) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (first + j * kPlanThreads + (t & ~31) >= end) break;
      // requests' rows mostly lie together: a whole warp of one group needs no match
      const bool one = __all_sync(0xffffffffu, group[j] == __shfl_sync(0xffffffffu, group[j], 0));
      const uint32_t peers = one ? 0xffffffffu : __match_any_sync(0xffffffffu, group[j]);
      const int leader = __ffs(peers) - 1;
      int at = 0;
      if (group[j] >= 0 && lane == leader) at = atomicAdd(&into[group[j]], __popc(peers));
      place[j] = __shfl_sync(0xffffffffu, at, leader) + __popc(peers & ((1u << lane) - 1));
    }
  };
  load(row0);
  for (int i = t; i < groups; i += kPlanThreads) bins[i] = 0;
  if (t < 2) carry[t] = 0;
  __syncthreads();
  count(bins, row0);
  for (int64_t first = row0 + kStep; first < end; first += kStep) {
    load(first);
    count(bins, first);
  }
  __syncthreads();
  if (cluster > 1) {
    cluster_arrive();
    cluster_wait();
  }
  // exclusive prefix sums of rows and tiles over the groups, in every CTA
  for (int first = 0; first < groups; first += kPlanThreads) {
    const int g = first + t;
    int rows = 0, before = 0;  // of all CTAs, of those before this one
    if (g < groups) {
      if (cluster == 1) {
        rows = bins[g];
      } else {
        int counts[kMaxCluster];
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
          counts[k] = 0;
          if (k < cluster)
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(counts[k]) : "r"(mapa_shared(smem_u32(bins + g), k)) : "memory");
        }
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
          rows += counts[k];
          before += k < cta ? counts[k] : 0;
        }
      }
    }
    const int tiles = rows / kLargeRows + (rows % kLargeRows != 0);
    const int r = warp_scan(rows, lane), n = warp_scan(tiles, lane);
    if (lane == 31) {
      sum_rows[warp] = r;
      sum_tiles[warp] = n;
    }
    __syncthreads();
    if (warp == 0) {
      const int sr = warp_scan(sum_rows[lane], lane), sn = warp_scan(sum_tiles[lane], lane);
      sum_rows[lane] = sr;
      sum_tiles[lane] = sn;
    }
    __syncthreads();
    const int first_row = carry[0] + (warp > 0 ? sum_rows[warp - 1] : 0) + r - rows;
    const int first_tile = carry[1] + (warp > 0 ? sum_tiles[warp - 1] : 0) + n - tiles;
    if (g < groups) start[g] = first_row + before;
    auto tile = [&](int at, int of, int row, int rows_of, int i) {
      plan.tiles[at + i] = make_int4(of, row + i * kLargeRows, min(kLargeRows, rows_of - i * kLargeRows), 0);
    };
    constexpr int kOwn = 8;  // tiles of a group that its thread writes; those of a longer one by a warp of each CTA
    if (cta == 0 && tiles <= kOwn)
      for (int i = 0; i < tiles; ++i) tile(first_tile, g, first_row, rows, i);
    for (uint32_t left = __ballot_sync(0xffffffffu, tiles > kOwn); left != 0; left &= left - 1) {
      const int src = __ffs(left) - 1;
      const int rows_of = __shfl_sync(0xffffffffu, rows, src), row_of = __shfl_sync(0xffffffffu, first_row, src);
      const int tile_of = __shfl_sync(0xffffffffu, first_tile, src), tiles_of = __shfl_sync(0xffffffffu, tiles, src);
      for (int i = cta * 32 + lane; i < tiles_of; i += cluster * 32) tile(tile_of, g - lane + src, row_of, rows_of, i);
    }
    if (first + kPlanThreads >= groups) {  // the last ones
      if (t == 0 && cta == 0) *plan.num_tiles = carry[1] + sum_tiles[31];
      break;
    }
    __syncthreads();
    if (t == 0) {
      carry[0] += sum_rows[31];
      carry[1] += sum_tiles[31];
    }
    __syncthreads();
  }
  __syncthreads();
  if (cluster > 1) cluster_arrive();  // the other CTAs' counts are read
  // the rows' places; a longer share is counted again, from its groups' first places
  for (int64_t first = row0; first < end; first += kStep) {
    if (share > kStep) {
      load(first);
      count(start, first);
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int64_t i = first + j * kPlanThreads + t;
      if (i < end) plan.perm[share > kStep ? place[j] : start[group[j]] + place[j]] = static_cast<int>(i);
    }
  }
  __syncwarp();
  if (cluster > 1) cluster_wait();
}

// ---- streaming through shared memory -------------------------------------------------
// Tiles are rows of `nch` 64-byte chunks. Eight lanes that read 16 bytes each
// touch two rows of different parity; an even number of chunks would put those
// on the same banks, so the chunks of odd rows are swapped in pairs.
__device__ __forceinline__ uint32_t tile_offset(int row, int nch, int chunk, int quarter) {
  const int c = (nch & 1) ? chunk : chunk ^ (row & 1);
  return static_cast<uint32_t>((row * nch + c) * 64 + quarter * 16);
}
// `bytes` (16 or 0) from global to shared memory, the rest of 16 as zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// Part `part` of 2^log_parts of a range.
__device__ __forceinline__ void split_range(int64_t units, int log_parts, int part, int* first, int* last) {
  *first = static_cast<int>((units * part) >> log_parts);
  *last = static_cast<int>((units * (part + 1)) >> log_parts);
}

// ---- the expand step -----------------------------------------------------------------
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
  const int lane = threadIdx.x & 31, cols = static_cast<int>(col1 - col0);
  constexpr int AHEAD = 4;  // vectors of a lane in flight: one at a time, a CTA of these was the last to end
  for (int m = threadIdx.x >> 5; m < tile.count; m += blockDim.x >> 5) {  // a warp for a row
    const int64_t row = rows[m];
    const T* base = a.base != nullptr && !bad ? static_cast<const T*>(a.base) + row * a.base_stride + col0 : nullptr;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + col0;
    if (vec && base != nullptr) {
      for (int c = lane * 8; c < cols; c += AHEAD * 256) {
        Eight<T> e[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          if (c + j * 256 < cols) load_eight(e[j], base + c + j * 256);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          if (c + j * 256 < cols) {
#pragma unroll
            for (int i = 0; i < Eight<T>::W; ++i) reinterpret_cast<uint4*>(out + c + j * 256)[i] = e[j].u[i];
          }
        }
      }
    } else {
      for (int c = lane; c < cols; c += 32) out[c] = base != nullptr ? base[c] : fill;
    }
  }
}

// The values of x's type that v is split into: v = the sum of them.
template <typename T> constexpr int kSplits = sizeof(T) == 4 ? 1 : std::is_same<T, __nv_bfloat16>::value ? 3 : 2;

// The staged values of v, [M][stride] elements each; a third one lies elsewhere.
template <typename T, int M> struct Staged {
  T *at, *third;
  int stride;
  __device__ T* split(int i) const { return i == 2 ? third : at + i * M * stride; }
  __device__ Staged from(int elements) const { return Staged{at + elements, third + elements, stride}; }
};

// x cut, not rounded, to T's bits.
template <typename T> __device__ __forceinline__ float cut(float x);
template <> __device__ __forceinline__ float cut<__half>(float x) { return __half2float(__float2half_rz(x)); }
template <> __device__ __forceinline__ float cut<__nv_bfloat16>(float x) { return __bfloat162float(__float2bfloat16_rz(x)); }

// Stages the tile's v as operands in shared memory, split into values of one
// sign, of which none is zero unless v is (a zero one becomes 2^-24 of the scaled
// row, or 2^-64 of v) and all are infinite if v is: beside an infinity of B their
// products have one sign, as the whole v's. sum(m, r) gives four neighbouring
// values of row m, summed and scaled. fp16 rows are scaled by a power of two to
// below 2^15, so that values down to 2^-15 of a row's largest keep all their bits
// (row_scale takes it back; `sums`, [M][sums_stride], holds them meanwhile and may
// be what sum(m, r) reads); rows past the tile and ranks past the end are zero.
// OVER_VR: if not 0, vr, and the third of the split values lies over what sum(m, r)
// reads: it is held until all of that has been read (256 threads).
template <typename T, int OVER_VR, int M, typename Sum>
__device__ __forceinline__ void stage_v(const Tile& tile, int rank, int vr, const Staged<T, M>& v, float* sums,
                                        int sums_stride, float* row_scale, unsigned* row_max, Sum sum) {
  constexpr int SPLITS = kSplits<T>;
  constexpr bool OVER = OVER_VR > 0 && SPLITS == 3;
  constexpr int TURNS = OVER ? M * OVER_VR / 4 / 256 : 1;
  static_assert(!OVER || M * OVER_VR / 4 % 256 == 0, "whole turns of the threads");
  uint2 held[TURNS];
  constexpr bool SCALED = std::is_same<T, __half>::value;
  const int shift = 31 - __clz(vr / 4), quads = 1 << shift, threads = blockDim.x;  // vr is a power of two
  if constexpr (SCALED) {
    for (int m = threadIdx.x; m < M; m += threads) row_max[m] = 0;
    __syncthreads();
  }
  // four values of row m, split
  auto put = [&](int m, int r, const float (&t)[4], float down, uint2& third) {
    const int to = m * v.stride + r;
    if constexpr (SPLITS == 1) {
      *reinterpret_cast<float4*>(v.split(0) + to) = make_float4(t[0], t[1], t[2], t[3]);
    } else {
      alignas(8) T part[SPLITS][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = SCALED ? t[j] * down : t[j];
#pragma unroll
        for (int i = 0; i < SPLITS; ++i) {
          float f = i + 1 < SPLITS ? cut<T>(x) : Ty<T>::to_f(Ty<T>::from_f(x));
          if (fabsf(f) <= 3.402823466e38f) x -= f;  // an infinity is all of them
          if (f == 0.f && t[j] != 0.f) f = SCALED ? copysignf(0x1p-24f, t[j]) : 0x1p-64f * t[j];
          part[i][j] = Ty<T>::from_f(f);
        }
      }
#pragma unroll
      for (int i = 0; i < SPLITS; ++i) {
        const uint2 u = *reinterpret_cast<const uint2*>(part[i]);
        if (OVER && i == 2) third = u;
        else *reinterpret_cast<uint2*>(v.split(i) + to) = u;
      }
    }
  };
  auto take = [&](int i, uint2& third) {
    const int m = i >> shift, r = (i & (quads - 1)) * 4;
    float t[4] = {};
    if (m < tile.count && r < rank) {
      const float4 u = sum(m, r);
      t[0] = u.x;
      t[1] = r + 1 < rank ? u.y : 0.f;  // ranks past the end hold nothing
      t[2] = r + 2 < rank ? u.z : 0.f;
      t[3] = r + 3 < rank ? u.w : 0.f;
    }
    if constexpr (SCALED) {
      if (r < sums_stride) *reinterpret_cast<float4*>(sums + m * sums_stride + r) = make_float4(t[0], t[1], t[2], t[3]);
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = fabsf(t[j]);
        if (x <= 3.402823466e38f) most = fmaxf(most, x);  // infinities and NaN need no scale
      }
      if (most != 0.f) atomicMax(row_max + m, __float_as_uint(most));  // ordered like the floats
    } else {
      put(m, r, t, 1.f, third);
    }
  };
  if constexpr (OVER) {
#pragma unroll
    for (int n = 0; n < TURNS; ++n) take(n * 256 + static_cast<int>(threadIdx.x), held[n]);
  } else {
    // Not unrolled: most launches take one turn or two (64 tokens over 32 adapters 7.5 -> 7.3 us).
#pragma unroll 1
    for (int i = threadIdx.x; i < M * quads; i += threads) take(i, held[0]);
  }
  __syncthreads();
  if constexpr (OVER) {
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      const int i = n * 256 + static_cast<int>(threadIdx.x);
      *reinterpret_cast<uint2*>(v.third + (i >> shift) * v.stride + (i & (quads - 1)) * 4) = held[n];
    }
    __syncthreads();
  }
  if constexpr (SCALED) {
    for (int m = threadIdx.x; m < M; m += threads) {
      const float most = __uint_as_float(row_max[m]);
      row_scale[m] = most > 0.f ? ldexpf(1.f, max(-126, ilogbf(most) - 14)) : 1.f;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < M * quads; i += threads) {
      const int m = i >> shift, r = (i & (quads - 1)) * 4;
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < sums_stride) u = *reinterpret_cast<const float4*>(sums + m * sums_stride + r);
      const float t[4] = {u.x, u.y, u.z, u.w};
      put(m, r, t, 1.f / row_scale[m], held[0]);
    }
    __syncthreads();
  }
}

// The parts of v that a cluster's CTAs have sent, [cluster][M][stride], added in order.
template <int M> struct SumParts {
  const float* parts;
  int cluster, stride;
  float scale;
  __device__ float4 operator()(int m, int r) const {
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < cluster; ++k) {
      const float4 w = *reinterpret_cast<const float4*>(parts + (k * M + m) * stride + r);
      u.x += w.x;
      u.y += w.y;
      u.z += w.z;
      u.w += w.w;
    }
    return make_float4(u.x * scale, u.y * scale, u.z * scale, u.w * scale);
  }
};

// The product over chunk c of 16 staged rows (v: this lane's place in row g)
// with 32 rows of B given by bf(j, chunk): adds to acc, the smallest of the
// split values first.
template <typename T, int M, typename LoadB>
__device__ __forceinline__ void expand_chunk(float (&acc)[4][4], const Staged<T, M>& v, int c, LoadB bf) {
  constexpr int C = chunk_elems(sizeof(T));
  uint4 b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = bf(j, c);
#pragma unroll
  for (int i = kSplits<T> - 1; i >= 0; --i) {
    const uint4 a0 = *reinterpret_cast<const uint4*>(v.split(i) + c * C);
    const uint4 a1 = *reinterpret_cast<const uint4*>(v.split(i) + 8 * v.stride + c * C);
#pragma unroll
    for (int j = 0; j < 4; ++j) Chunk<T>::mma(acc[j], a0, a1, b[j]);
  }
}
// What a thread holds of a row in the expand step: the q-th 16 bytes of a chunk
// or, where ranks end with its first half (HALF: 16-bit types, up to 16 ranks), the
// q-th 8 of that half, for which one instruction does instead of two.
template <bool HALF> using Operand = std::conditional_t<HALF, uint2, uint4>;

// expand_chunk's product with the rows' few chunks kept in registers.
template <typename T, int NCH, bool HALF>
struct StagedRows {
  static constexpr int SPLITS = kSplits<T>;
  using Vec = Operand<HALF>;
  static_assert(!HALF || NCH == 1, "half of the only chunk");
  Vec a0[SPLITS][NCH], a1[SPLITS][NCH];
  template <int M>
  __device__ void load(const Staged<T, M>& v) {
    constexpr int C = chunk_elems(sizeof(T));
#pragma unroll
    for (int i = 0; i < SPLITS; ++i) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        a0[i][c] = *reinterpret_cast<const Vec*>(v.split(i) + c * C);
        a1[i][c] = *reinterpret_cast<const Vec*>(v.split(i) + 8 * v.stride + c * C);
      }
    }
  }
  template <typename LoadB>
  __device__ void expand(float (&acc)[4][4], LoadB bf) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Vec b = bf(j, c);
#pragma unroll
        for (int i = SPLITS - 1; i >= 0; --i) Chunk<T>::mma(acc[j], a0[i][c], a1[i][c], b);
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

// ---- clusters ----------------------------------------------------------------------------
// 16 bytes to a cluster address; their arrival is counted by the mbarrier at `bar` in the same CTA.
__device__ __forceinline__ void push16(uint32_t addr, float4 v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
               "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)), "r"(__float_as_uint(v.w)),
               "r"(bar)
               : "memory");
}

// ---- few tokens ----------------------------------------------------------------------------
struct SmallWidths {  // elements that rows are aligned to: of x and A, of B; whole vectors of out and base
  int k, b;
  bool n;
};

// A cluster of CTAs takes a tile. Its CTA c shrinks part c of K (a warp a part
// of that), sends its sums to all CTAs of the cluster, and expands part c of
// the columns. What such a launch takes is a chain of memory latencies (ids, x
// and A, the exchange, B and base), so loads are issued as early as their
// addresses are known: BATCH chunks of x and A at a time, the first B rows and
// base values before the exchange, and each next block's before the one at hand
// is computed. Its instructions are fetched once, too, so the kernel is kept
// short: four chunks or two blocks in flight were 0.2 and 0.3 us slower. One
// token, 4096 x 4096, rank 16, bf16: 4.3 us, of which the launch is 1.5 (two
// launches with v in global memory took 6.3).
template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) lora_small_kernel(const LoraArgs a, int log_cluster, SmallWidths given, int64_t v_rank,
                                                         uint32_t* err) {
  // aligned calls (VEC) are compiled without the other widths: a launch this short waits for its instructions too
  const SmallWidths width = VEC ? SmallWidths{16 / sizeof(T), 16 / sizeof(T), true} : given;
  constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  constexpr int M = kSmallRows, RB = 8 * NT;  // ranks of a pass
  constexpr int BATCH = NT == 8 ? 1 : 2;
  constexpr bool SCALED = std::is_same<T, __half>::value;
  __shared__ int rows[M], scratch[8 * kIds + 2];
  __shared__ __align__(16) int groups[kIds * 256];
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
  const int cluster = 1 << log_cluster, part = static_cast<int>(blockIdx.x) & (cluster - 1);
  const Tile tile = find_tile(a, static_cast<int>(blockIdx.x) >> log_cluster, rows, groups, scratch);
  if (tile.count == 0) {  // of the whole cluster
    cluster_wait();
    return;
  }
  int block0, block1;
  split_range((a.n + 31) / 32, log_cluster, part, &block0, &block1);
  const int64_t col0 = static_cast<int64_t>(block0) * 32, col1 = min(a.n, static_cast<int64_t>(block1) * 32);
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
  T* const staged = reinterpret_cast<T*>(smem + sizeof(float) * cluster * M * vr);
  const Staged<T, M> v{staged, staged + 2 * M * stride, stride};
  auto* red = reinterpret_cast<float(*)[M][RB + 4]>(staged + kSplits<T> * M * stride);  // [kSmallWarps]
  if (t == 0) mbar_arrive_expect_tx(&received, static_cast<uint32_t>(cluster * tile.count * quads * 16));
  const bool in0 = g < tile.count, in1 = g + 8 < tile.count;
  const int64_t t0 = rows[in0 ? g : 0], t1 = rows[in1 ? g + 8 : 0];
  // shrink
  const T* x0 = in0 ? static_cast<const T*>(a.x) + t0 * a.x_stride : nullptr;
  const T* x1 = in1 ? static_cast<const T*>(a.x) + t1 * a.x_stride : nullptr;
  int c0, c1;
  static_assert(kSmallWarps == 8, "a power of two");
  split_range((a.k + C - 1) / C, log_cluster + 3, part * kSmallWarps + warp, &c0, &c1);
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
    for (int i = t; i < tile.count * (RB / 4); i += 256) {
      const int m = i / (RB / 4), r = i % (RB / 4) * 4;
      if (r0 + r >= rank) continue;
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
  constexpr bool HALF = NT == 2 && sizeof(T) == 2;
  auto b_chunk = [&](int64_t n0, int j, int c) {
    const int64_t col = n0 + block_column(g) + 2 * j;
    const T* row = col < col1 ? b + col * rank : nullptr;
    if constexpr (HALF) return load_half<T>(row, q * (E / 2), rank, width.b);
    else return load_chunk<T>(row, c * C + q * E, rank, width.b);
  };
  struct Block {
    Operand<HALF> b[4];
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
  constexpr int kStride = kSmallWarps * 32;
  Block next{};
  load_block(next, first);
  const float scale = a.scaling != nullptr ? a.scaling[tile.group] : 1.f;
  const bool arrived = mbar_wait(&received, 0, err, ERR_WAIT_TIMEOUT_OTHER);
  if (__syncthreads_or(!arrived)) return;
  stage_v<T, 0>(tile, rank, vr, v, parts, vr, row_scale, row_max, SumParts<M>{parts, cluster, vr, scale});
  const float s0 = SCALED ? row_scale[g] : 1.f, s1 = SCALED ? row_scale[g + 8] : 1.f;
  const Staged<T, M> mine = v.from(g * stride + q * (HALF ? E / 2 : E));
  StagedRows<T, 1, HALF> held;
  if constexpr (HALF) held.load(mine);
  T* out0 = static_cast<T*>(a.out) + t0 * a.out_stride + q * 8;
  T* out1 = static_cast<T*>(a.out) + t1 * a.out_stride + q * 8;
  for (int64_t n0 = first; n0 < col1; n0 += kStride) {
    const Block now = next;
    if (n0 + kStride < col1) load_block(next, n0 + kStride);
    float acc[4][4] = {};
    if constexpr (HALF) {
      held.expand(acc, [&](int j, int) { return now.b[j]; });
    } else {
      expand_chunk(acc, mine, 0, [&](int j, int) { return now.b[j]; });
      for (int c = 1; c < vr / C; ++c) expand_chunk(acc, mine, c, [&](int j, int k) { return b_chunk(n0, j, k); });
    }
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

// ---- many tokens ---------------------------------------------------------------------------
// A cluster of CTAs takes a tile of 64 rows that use the same adapter; CTA c of
// it shrinks part c of K and expands part c of the columns. Both steps stream
// through a ring of STAGES stages in shared memory: STEP bytes of K of x's rows
// and A's (RANKS of them at a time), then STEP bytes of columns of base with
// their rows of B. The first columns are on their way while the cluster's CTAs
// exchange their parts of v. Warp w has rows 16 (w % 4) .. + 15; the two halves
// of the warps share the 64-byte chunks of K and the blocks of 32 columns.
// VR: ranks held by the expand step (a power of two of chunks). VEC: x, A, B,
// base and out are whole aligned vectors; else elements are copied one by one.
template <typename T, int RANKS, int VR, int STEP, int STAGES, bool VEC>
struct LargeShape {
  static constexpr int E = 16 / sizeof(T), C = chunk_elems(sizeof(T));
  static constexpr int M = kLargeRows;
  static constexpr int SB = STEP;         // bytes of a row in a step
  static constexpr int KS = SB / sizeof(T);    // elements of K, and columns, of a step
  static constexpr int NCH = VR / C;           // chunks of a row of B
  static constexpr int kRows = M * SB;         // bytes of the tile's rows in a stage
  static constexpr int kShrink = kRows + RANKS * SB, kExpand = kRows + KS * NCH * 64;
  static constexpr int kStage = kShrink > kExpand ? kShrink : kExpand;
  static constexpr int stride = VR + E;
  // v's split values, a third one over the exchanged parts (they are summed by then)
  static constexpr size_t kSplit = sizeof(T) * M * stride, kStaged = (kSplits<T> == 1 ? 1 : 2) * kSplit;
  static_assert(kStaged >= sizeof(float) * M * (RANKS + 4), "the halves' sums fit where v is staged later");
  static constexpr int PR = VR > RANKS && RANKS < 128 ? RANKS : VR;  // ranks of a row of an exchanged part
  static size_t smem(int cluster) {
    return STAGES * kStage + kStaged + std::max(kSplits<T> == 3 ? kSplit : 0, sizeof(float) * cluster * M * PR);
  }
};

template <typename T, int RANKS, int VR, int STEP, int STAGES, bool VEC>
__global__ void __launch_bounds__(kLargeThreads) lora_large_kernel(const LoraArgs a, LoraPlan plan, int log_cluster,
                                                                   uint32_t* err) {
  using S = LargeShape<T, RANKS, VR, STEP, STAGES, VEC>;
  constexpr int E = S::E, M = S::M, KS = S::KS, NCH = S::NCH, NT = RANKS / 8, stride = S::stride;
  constexpr bool SCALED = std::is_same<T, __half>::value;
  __shared__ int rows[M];
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
  const int cluster = 1 << log_cluster, part = static_cast<int>(blockIdx.x) & (cluster - 1);
  const Tile tile = planned_tile(plan, static_cast<int>(blockIdx.x) >> log_cluster, rows);
  const int64_t col_steps = (a.n + KS - 1) / KS;
  int s0i, s1i;
  split_range(col_steps, log_cluster, part, &s0i, &s1i);
  const int64_t col0 = static_cast<int64_t>(s0i) * KS, col1 = min(a.n, static_cast<int64_t>(s1i) * KS);
  if (tile.count == 0 || tile.group >= a.adapters) {  // of the whole cluster
    if (tile.count > 0) fill_rows<T>(a, tile, rows, col0, col1, VEC, err);
    __syncwarp();
    cluster_wait();
    return;
  }
  const int rank = static_cast<int>(a.rank), quads = (rank + 3) / 4;
  uint8_t* ring = smem;
  float* parts = reinterpret_cast<float*>(smem + STAGES * S::kStage + S::kStaged);  // [cluster][M][PR]
  const Staged<T, M> v{reinterpret_cast<T*>(smem + STAGES * S::kStage), reinterpret_cast<T*>(parts), stride};
  auto* halves = reinterpret_cast<float(*)[RANKS + 4]>(v.at);  // until v is staged
  if (t == 0) mbar_arrive_expect_tx(&received, static_cast<uint32_t>(cluster * tile.count * quads * 16));
  const int g = lane >> 2, q = lane & 3;
  const int m0 = (warp & 3) * 16, half = warp >> 2;
  const bool busy = m0 < tile.count;
  const uint32_t ring_at = smem_u32(ring);
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  // This thread's copies of a step: 16 bytes `vec` of every kRowStep-th row.
  // Where they go does not change but for the stage, and the sources move on by
  // a step's bytes: a copy costs a few instructions.
  constexpr int kVecs = S::SB / 16, kRowStep = kLargeThreads / kVecs, kCopies = M / kRowStep, kChunks = S::SB / 64;
  const int vec = t % kVecs, row0 = t / kVecs;
  const uint32_t copy_at = tile_offset(row0, kChunks, vec >> 2, vec & 3);  // rows kRowStep apart have the same parity
  static_assert(kRowStep % 2 == 0, "rows of a thread have one parity");
  auto put = [&](uint32_t at, const T* from, int left) {  // `left` elements exist (none: zeros)
    if constexpr (VEC) {
      copy16(ring_at + at, from, left > 0 ? 16 : 0);
    } else {
      *reinterpret_cast<uint4*>(ring + at) = load_chunk<T>(left > 0 ? from : nullptr, 0, left, 1);
    }
  };

  // ---- shrink
  int k0, k1;
  split_range((a.k + KS - 1) / KS, log_cluster, part, &k0, &k1);
  const uint32_t my_part = smem_u32(parts + part * M * S::PR), bar = smem_u32(&received);
  // a lane's operands in a stage: row m0 + g (and 8 further) of x, row g (and 8, 16, ... further) of A
  constexpr int kHalfChunks = kChunks / 2;
  const uint32_t x_at = tile_offset(m0 + g, kChunks, half * kHalfChunks, q), a_at = S::kRows + tile_offset(g, kChunks, half * kHalfChunks, q);
  for (int r0 = 0; r0 < rank; r0 += RANKS) {
    constexpr int kACopies = (RANKS + kRowStep - 1) / kRowStep;
    const int64_t start = static_cast<int64_t>(k0) * KS + vec * E;
    const T *xp[kCopies], *ap[kACopies];
    bool x_ok[kCopies], a_ok[kACopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = row0 + kRowStep * i;
      x_ok[i] = r < tile.count;
      xp[i] = static_cast<const T*>(a.x) + static_cast<int64_t>(rows[x_ok[i] ? r : 0]) * a.x_stride + start;
    }
#pragma unroll
    for (int i = 0; i < kACopies; ++i) {
      const int r = r0 + row0 + kRowStep * i;
      a_ok[i] = r < rank && row0 + kRowStep * i < RANKS;
      ap[i] = static_cast<const T*>(a.a) + (static_cast<int64_t>(tile.group) * rank + (a_ok[i] ? r : 0)) * a.k + start;
    }
    int left = static_cast<int>(a.k - start), to_load = k1 - k0;
    auto load = [&](uint32_t at) {
      if (to_load > 0) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          put(at + copy_at + i * kRowStep * S::SB, xp[i], x_ok[i] ? left : 0);
          xp[i] += KS;
        }
#pragma unroll
        for (int i = 0; i < kACopies; ++i) {
          if (RANKS % kRowStep == 0 || row0 + kRowStep * i < RANKS)
            put(at + S::kRows + copy_at + i * kRowStep * S::SB, ap[i], a_ok[i] ? left : 0);
          ap[i] += KS;
        }
        left -= KS;
      }
      --to_load;
      commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) load(i * S::kStage);
    // A tensor instruction cuts what it adds to: over 4096 columns 3e-6 of the sum (8192 tokens of rank 64 in fp16:
    // 1 of 100 outputs off by a step, 1 of 700 without it; the time of rank 32 is the same, of 128 160 -> 171 us). So a
    // step's sums start at zero and are added by rounded additions, GROUP at a time where that was faster (an instruction
    // waits for the one before it on the same sum; rank 64 88 -> 84 us, 128 in fp32 168 -> 158, in bf16 171 -> 174).
    constexpr int GROUP = NT == 8 || (NT == 16 && sizeof(T) == 4) ? 4 : 1;
    float acc[NT][4] = {};
    uint32_t now = 0, free = (STAGES - 1) * S::kStage;  // the stage at hand, and the one before it
    for (int step = k0; step < k1; ++step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncthreads();  // the step's bytes are there, and the stage before it is free
      load(free);
      if (busy) {
        const uint8_t* xs = ring + now + x_at;
        const uint8_t* as = ring + now + a_at;
        // the next chunk: 64 bytes on, or where the swap of odd rows puts it
        int on[kHalfChunks];
        uint4 a0[kHalfChunks], a1[kHalfChunks];
#pragma unroll
        for (int h = 0; h < kHalfChunks; ++h) {
          on[h] = h == 0 ? 0 : static_cast<int>(tile_offset(g, kChunks, half * kHalfChunks + h, q)) -
                                   static_cast<int>(tile_offset(g, kChunks, half * kHalfChunks, q));
          a0[h] = lds16(xs + on[h]);
          a1[h] = lds16(xs + on[h] + 8 * S::SB);
        }
#pragma unroll
        for (int j0 = 0; j0 < NT; j0 += GROUP) {
          float t[GROUP][4] = {};
#pragma unroll
          for (int h = 0; h < kHalfChunks; ++h) {
            uint4 b[GROUP];
#pragma unroll
            for (int j = 0; j < GROUP; ++j) b[j] = lds16(as + on[h] + (j0 + j) * 8 * S::SB);
            if constexpr (sizeof(T) == 2) {
#pragma unroll
              for (int j = 0; j < GROUP; ++j)
                Chunk<T>::mma(t[j], make_uint2(a0[h].x, a0[h].y), make_uint2(a1[h].x, a1[h].y), make_uint2(b[j].x, b[j].y));
#pragma unroll
              for (int j = 0; j < GROUP; ++j)
                Chunk<T>::mma(t[j], make_uint2(a0[h].z, a0[h].w), make_uint2(a1[h].z, a1[h].w), make_uint2(b[j].z, b[j].w));
            } else {
#pragma unroll
              for (int j = 0; j < GROUP; ++j) Chunk<T>::mma(t[j], a0[h], a1[h], b[j]);
            }
          }
#pragma unroll
          for (int j = 0; j < GROUP; ++j) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const F2 sum = add2(f2(acc[j0 + j][i], acc[j0 + j][i + 1]), f2(t[j][i], t[j][i + 1]));
              acc[j0 + j][i] = sum.x;
              acc[j0 + j][i + 1] = sum.y;
            }
          }
        }
      }
      free = now;
      now = now + S::kStage == STAGES * S::kStage ? 0 : now + S::kStage;
    }
    // the two halves' sums, then this CTA's part to all CTAs of the cluster
    auto each = [&](auto f) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        f(reinterpret_cast<float2*>(&halves[m0 + g][j * 8 + 2 * q]), acc[j][0], acc[j][1]);
        f(reinterpret_cast<float2*>(&halves[m0 + g + 8][j * 8 + 2 * q]), acc[j][2], acc[j][3]);
      }
    };
    if (busy && half == 1) each([](float2* p, float x, float y) { *p = make_float2(x, y); });
    __syncthreads();
    if (busy && half == 0) {
      each([](float2* p, float x, float y) {
        const float2 o = *p;
        *p = make_float2(x + o.x, y + o.y);
      });
    }
    if (r0 == 0) cluster_wait();
    __syncthreads();
    for (int i = t; i < tile.count * (RANKS / 4); i += kLargeThreads) {
      const int m = i / (RANKS / 4), r = i % (RANKS / 4) * 4;
      if (r0 + r >= rank) continue;
      const float4 u = *reinterpret_cast<const float4*>(&halves[m][r]);
      const uint32_t dst = my_part + (m * S::PR + r0 + r) * 4;
      for (int k = 0; k < cluster; ++k) push16(mapa_shared(dst, k), u, mapa_shared(bar, k));
    }
    __syncthreads();  // before the halves' sums and the ring are written again
  }

  // ---- expand
  const bool with_base = a.base != nullptr;
  const int cols = static_cast<int>(col1 - col0);
  const T* bp[kCopies];
  bool b_row_ok[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const int r = row0 + kRowStep * i;
    b_row_ok[i] = r < tile.count;
    bp[i] = static_cast<const T*>(a.base) + static_cast<int64_t>(rows[b_row_ok[i] ? r : 0]) * a.base_stride + col0 + vec * E;
  }
  // of B: 16 bytes w_vec of every kWStep-th row
  constexpr int kWVecs = NCH * 4, kWStep = kLargeThreads / kWVecs, kWCopies = (KS + kWStep - 1) / kWStep;
  static_assert(kWVecs <= kLargeThreads && kWStep % 2 == 0, "a row of B has at most one vector for each thread");
  const int w_vec = t % kWVecs, w_row0 = t / kWVecs;
  const T* wp = static_cast<const T*>(a.b) + (static_cast<int64_t>(tile.group) * a.n + col0 + w_row0) * rank + w_vec * E;
  const uint32_t w_at = S::kRows + tile_offset(w_row0, NCH, w_vec >> 2, w_vec & 3);
  const int w_left = rank - w_vec * E;
  const int64_t w_step = static_cast<int64_t>(kWStep) * rank, w_on = static_cast<int64_t>(KS) * rank;
  int cols_left = cols;
  auto load = [&](uint32_t at) {
    if (cols_left > 0) {
      if (VEC && with_base) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          put(at + copy_at + i * kRowStep * S::SB, bp[i], b_row_ok[i] ? cols_left - vec * E : 0);
          bp[i] += KS;
        }
      }
      const T* from = wp;
#pragma unroll
      for (int i = 0; i < kWCopies; ++i, from += w_step) {
        const int r = w_row0 + kWStep * i;
        if (KS % kWStep == 0 || r < KS) put(at + w_at + i * kWStep * NCH * 64, from, r < cols_left ? w_left : 0);
      }
      wp += w_on;
    }
    cols_left -= KS;
    commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(i * S::kStage);
  const float scale = a.scaling != nullptr ? a.scaling[tile.group] : 1.f;
  const bool arrived = mbar_wait(&received, 0, err, ERR_WAIT_TIMEOUT_OTHER);
  if (__syncthreads_or(!arrived)) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }
  stage_v<T, VR>(tile, rank, VR, v, parts, S::PR, row_scale, row_max, SumParts<M>{parts, cluster, S::PR, scale});
  const bool in0 = m0 + g < tile.count, in1 = m0 + g + 8 < tile.count;
  const float f0s = SCALED ? row_scale[m0 + g] : 1.f, f1s = SCALED ? row_scale[m0 + g + 8] : 1.f;
  constexpr bool HALF = RANKS == 16 && sizeof(T) == 2;
  const Staged<T, M> mine = v.from((m0 + g) * stride + q * (HALF ? E / 2 : E));
  const int64_t t0 = rows[in0 ? m0 + g : 0], t1 = rows[in1 ? m0 + g + 8 : 0];
  T* out0 = static_cast<T*>(a.out) + t0 * a.out_stride + col0 + q * 8;
  T* out1 = static_cast<T*>(a.out) + t1 * a.out_stride + col0 + q * 8;
  constexpr bool HELD = NCH <= 2 && sizeof(T) == 2;
  StagedRows<T, HELD ? NCH : 1, HALF> held;
  if constexpr (HELD) held.load(mine);
  constexpr int BLOCKS = KS / 32;  // of a step: the halves of the warps share them, or take turns
  const uint32_t b_at = S::kRows + (HALF ? tile_offset(block_column(g), NCH, 0, 0) + q * 8 : tile_offset(block_column(g), NCH, 0, q));
  const uint32_t e_at = (m0 + g) * S::SB;
  uint32_t now = 0, free = (STAGES - 1) * S::kStage;
  const int steps = s1i - s0i;
  for (int step = 0; step < steps; ++step, out0 += KS, out1 += KS) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();  // the step's bytes are there, and the stage before it is free
    load(free);
    if (busy && (BLOCKS > 1 || (step & 1) == half)) {
      constexpr int MINE = BLOCKS > 1 ? BLOCKS / 2 : 1;
      const uint8_t* es = ring + now + e_at;
      float acc[MINE][4][4] = {};
      Eight<T> e0[MINE], e1[MINE];
      // all blocks' operands before the first store, which the compiler would not move them over
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int blk = BLOCKS > 1 ? half * MINE + i : 0;
        const uint8_t* bs = ring + now + b_at + blk * 32 * NCH * 64;
        auto bf = [&](int j, int c) {  // chunk c of an odd row may be swapped
          const int on = (NCH & 1) ? c * 64 : ((c ^ (g & 1)) - (g & 1)) * 64;
          return *reinterpret_cast<const Operand<HALF>*>(bs + j * 2 * NCH * 64 + on);
        };
        if constexpr (HELD) {
          held.expand(acc[i], bf);
        } else {
#pragma unroll 2
          for (int c = 0; c < NCH; ++c) expand_chunk(acc[i], mine, c, bf);
        }
        if constexpr (VEC) {
#pragma unroll
          for (int k = 0; k < Eight<T>::W; ++k) {
            const int w = (blk * 4 + q) * Eight<T>::W + k;  // 16-byte vector of the row; odd rows' chunks are swapped
            const uint32_t off = ((w >> 2) ^ (g & 1)) * 64 + (w & 3) * 16;
            e0[i].u[k] = lds16(es + off);
            e1[i].u[k] = lds16(es + off + 8 * S::SB);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int blk = BLOCKS > 1 ? half * MINE + i : 0;
        float f0[8], f1[8];
        block_values(acc[i], f0s, f1s, f0, f1);
        const int left = cols - step * KS - blk * 32 - q * 8;
        if constexpr (VEC) {
          if (left > 0 && in0) store_sum<T>(out0 + blk * 32, e0[i], with_base, f0);
          if (left > 0 && in1) store_sum<T>(out1 + blk * 32, e1[i], with_base, f1);
        } else {
          const T* base = static_cast<const T*>(a.base);
          const int64_t at = col0 + step * KS + blk * 32 + q * 8;
          if (in0) store_each<T>(out0 + blk * 32, with_base ? base + t0 * a.base_stride + at : nullptr, left, f0);
          if (in1) store_each<T>(out1 + blk * 32, with_base ? base + t1 * a.base_stride + at : nullptr, left, f1);
        }
      }
    }
    free = now;
    now = now + S::kStage == STAGES * S::kStage ? 0 : now + S::kStage;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- host ----------------------------------------------------------------------------
namespace {
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

int log2_of(int cluster) { return cluster == 8 ? 3 : cluster == 4 ? 2 : cluster - 1; }

bool small_call(int64_t tokens) { return tokens <= kSmallTokens; }

struct PlanBytes {  // of many tokens
  int64_t tiles;  // upper bound
  size_t perm, list;
  size_t total() const { return perm + list + 256; }
};
PlanBytes plan_bytes(int64_t tokens, int64_t adapters) {
  PlanBytes p{};
  p.tiles = tokens / kLargeRows + std::min(tokens, adapters + 2);
  p.perm = round256(sizeof(int) * tokens);
  p.list = round256(sizeof(int4) * p.tiles);
  return p;
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

// Clusters of a kernel that are resident at once (the SMs of a cluster share a
// processing cluster: fewer than their CTAs alone would allow).
cudaError_t resident_clusters(const void* kernel, int block, int cluster, size_t smem, int* count) {
  if (const cudaError_t e = ensure_smem_attr(kernel, smem + 4096); e != cudaSuccess) return e;
  int dev = 0;
  cudaGetDevice(&dev);
  static std::mutex mu;
  static std::map<std::tuple<const void*, size_t, int, int>, int> known;
  std::lock_guard<std::mutex> lock(mu);
  const auto [at, fresh] = known.try_emplace(std::make_tuple(kernel, smem, cluster, dev), 0);
  if (fresh) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(cluster));
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (const cudaError_t e = cudaOccupancyMaxActiveClusters(&at->second, kernel, &cfg); e != cudaSuccess) {
      known.erase(at);
      return e;
    }
  }
  *count = at->second;
  return cudaSuccess;
}

// Few clusters: an SM for each CTA, by asking for more than half of its memory
// (two would share one while others idle: 64 tokens over 8 adapters of rank 64
// 10.8 -> 9.0 us, 512 over 4 of rank 16 16.7 -> 14.2; 4096 x 4096).
cudaError_t spread(const void* kernel, int block, int cluster, int64_t clusters, size_t* smem) {
  constexpr size_t kAlone = 120 * 1024;
  if (*smem >= kAlone || clusters * cluster > num_sms()) return cudaSuccess;
  int resident = 0;
  const cudaError_t e = resident_clusters(kernel, block, cluster, kAlone, &resident);
  if (e == cudaSuccess && clusters <= resident) *smem = kAlone;
  return e;
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
  // at most so many tiles, most of them there when the adapters are mixed
  const int64_t tiles = std::min(a.tokens, a.tokens / kSmallRows + a.adapters + 2);
  // enough CTAs that a warp has about two chunks of K and two blocks of
  // columns, about one wave of them, and 32 KB of exchanged sums at most
  const int64_t chunks = (a.k + chunk_elems(sizeof(T)) - 1) / chunk_elems(sizeof(T));
  const int64_t want = std::max(chunks / (2 * kSmallWarps), a.n / (2 * 32 * kSmallWarps));
  int cluster = 1;
  while (cluster < kMaxCluster && cluster < want && 2 * cluster * tiles <= 4 * num_sms() && 2 * cluster * v_rank <= 512)
    cluster *= 2;
  const size_t smem = kSmallRows * (sizeof(float) * v_rank * cluster + kSplits<T> * sizeof(T) * (v_rank + E));
  auto launch = [&](auto* kernel, int nt) {
    size_t bytes = smem + sizeof(float) * kSmallWarps * kSmallRows * (8 * nt + 4);
    if (const cudaError_t e = spread(reinterpret_cast<const void*>(kernel), 256, cluster, tiles, &bytes); e != cudaSuccess) return e;
    return launch_grid(kernel, dim3(static_cast<unsigned>(tiles * cluster)), 256, cluster, bytes, st, a, log2_of(cluster),
                       width, v_rank, error_word_ptr());
  };
  const bool vec = width.k == E && width.b == E && width.n;
  if (a.rank <= 16) return vec ? launch(lora_small_kernel<T, 2, true>, 2) : launch(lora_small_kernel<T, 2, false>, 2);
  if (a.rank <= 32) return vec ? launch(lora_small_kernel<T, 4, true>, 4) : launch(lora_small_kernel<T, 4, false>, 4);
  return vec ? launch(lora_small_kernel<T, 8, true>, 8) : launch(lora_small_kernel<T, 8, false>, 8);
}

// The number of CTAs that share a tile, and the time to expect. The tiles run
// in waves of as many clusters as are resident at once; a tile's time is 5 us
// (first loads, the exchange) and its steps, shared by the cluster. Measured
// for rows of K + N = 8192 bf16 values, alone on a tile: 72 us with 256 bytes a
// step, 83 with 128. Less than a whole wave costs a whole one (4096 x 4096,
// rank 16, 256 bytes: 8192 tokens 50 us, 12000 84, 16384 88), so that more
// CTAs on an SM, or larger clusters, pay where they save a wave (12000 tokens
// with 128 bytes a step 66). The model knows bytes alone, not the products of a
// high rank or of fp32, and loses there: 2048 tokens of 4 adapters of rank 64 took
// 40.2 us by its choice and 36.7 without it.
struct ShapeChoice {
  int cluster = 1;
  double us = 0;
};
template <typename T, int RANKS, int VR, int STEP, int STAGES, bool VEC>
cudaError_t choose_cluster(const LoraArgs& a, int64_t tiles, ShapeChoice* best) {
  using S = LargeShape<T, RANKS, VR, STEP, STAGES, VEC>;
  const void* kernel = reinterpret_cast<const void*>(lora_large_kernel<T, RANKS, VR, STEP, STAGES, VEC>);
  const int64_t steps = (std::max(a.k, a.n) + S::KS - 1) / S::KS;
  const double alone = static_cast<double>(a.k + a.n) * sizeof(T) / 16384 * (STEP >= 256 ? 72 : 83) * (VEC ? 1 : 3);
  constexpr int kFewest = STEP >= 256 ? 4 : VEC ? 2 : 1;  // steps of a CTA
  for (int c = 1; c <= kMaxCluster && (c == 1 || kFewest * c <= steps) && (c == 1 || S::smem(c) <= 216 * 1024); c *= 2) {
    int resident = 0;
    if (const cudaError_t e = resident_clusters(kernel, kLargeThreads, c, S::smem(c), &resident); e != cudaSuccess) return e;
    if (resident == 0 && c > 1) break;  // no room for such a cluster
    const int64_t waves = (tiles + std::max(resident, 1) - 1) / std::max(resident, 1);
    const double sent = static_cast<double>(std::min<int64_t>(tiles, resident)) * c * c * kLargeRows * 4 * a.rank;  // bytes of a wave
    const double us = static_cast<double>(waves) * (5 + 0.35 * (c - 1) + sent / 3e6 + alone / c);
    if (c == 1 || us < best->us) *best = ShapeChoice{c, us};
  }
  return cudaSuccess;
}

template <typename T, int RANKS, int VR, int STEP, int STAGES, bool VEC>
cudaError_t launch_shape(const LoraArgs& a, const PlanBytes& p, const LoraPlan& plan, int64_t tiles, int cluster, cudaStream_t st) {
  using S = LargeShape<T, RANKS, VR, STEP, STAGES, VEC>;
  if (a.rank > S::PR || a.rank > VR) return cudaErrorInvalidValue;  // the exchanged parts' rows would be written past their ends
  auto* kernel = lora_large_kernel<T, RANKS, VR, STEP, STAGES, VEC>;
  size_t smem = S::smem(cluster);
  if (const cudaError_t e = spread(reinterpret_cast<const void*>(kernel), kLargeThreads, cluster, tiles, &smem); e != cudaSuccess)
    return e;
  return launch_grid(kernel, dim3(static_cast<unsigned>(p.tiles * cluster)), kLargeThreads, cluster, smem, st, a, plan,
                     log2_of(cluster), error_word_ptr());
}

// Up to 64 ranks: 128 or 256 bytes of a row a step, whichever is expected to be faster.
template <typename T, int RANKS, int STAGES, bool VEC>
cudaError_t launch_best(const LoraArgs& a, const PlanBytes& p, const LoraPlan& plan, int64_t tiles, cudaStream_t st) {
  constexpr int C = chunk_elems(sizeof(T)), VR = RANKS > C ? RANKS : C;
  ShapeChoice narrow, wide;
  if (const cudaError_t e = choose_cluster<T, RANKS, VR, 128, STAGES, VEC>(a, tiles, &narrow); e != cudaSuccess) return e;
  if (const cudaError_t e = choose_cluster<T, RANKS, VR, 256, 3, VEC>(a, tiles, &wide); e != cudaSuccess) return e;
  if (wide.us < narrow.us) return launch_shape<T, RANKS, VR, 256, 3, VEC>(a, p, plan, tiles, wide.cluster, st);
  return launch_shape<T, RANKS, VR, 128, STAGES, VEC>(a, p, plan, tiles, narrow.cluster, st);
}

// More ranks: in passes of 128. Two stages leave room for clusters of four with
// 128 ranks, three for two.
template <typename T, bool VEC>
cudaError_t launch_ranks(const LoraArgs& a, const PlanBytes& p, const LoraPlan& plan, int64_t tiles, cudaStream_t st) {
  ShapeChoice three, two;
  if (a.rank > 128) {
    if (const cudaError_t e = choose_cluster<T, 128, 256, 128, 2, VEC>(a, tiles, &two); e != cudaSuccess) return e;
    return launch_shape<T, 128, 256, 128, 2, VEC>(a, p, plan, tiles, two.cluster, st);
  }
  if (const cudaError_t e = choose_cluster<T, 128, 128, 128, 3, VEC>(a, tiles, &three); e != cudaSuccess) return e;
  if (const cudaError_t e = choose_cluster<T, 128, 128, 128, 2, VEC>(a, tiles, &two); e != cudaSuccess) return e;
  if (two.us < three.us) return launch_shape<T, 128, 128, 128, 2, VEC>(a, p, plan, tiles, two.cluster, st);
  return launch_shape<T, 128, 128, 128, 3, VEC>(a, p, plan, tiles, three.cluster, st);
}

template <typename T, bool VEC>
cudaError_t launch_tiles(const LoraArgs& a, const PlanBytes& p, const LoraPlan& plan, cudaStream_t st) {
  // the tiles to expect: each group's last one is half full on average
  const int64_t groups = std::min(a.tokens, a.adapters + 1);
  const int64_t tiles = std::max(groups, a.tokens / kLargeRows + groups / 2);
  if (a.rank <= 16) return launch_best<T, 16, 4, VEC>(a, p, plan, tiles, st);
  if (a.rank <= 32) return launch_best<T, 32, 3, VEC>(a, p, plan, tiles, st);  // three stages: two CTAs on an SM in clusters of eight
  if (a.rank <= 64) return launch_best<T, 64, 4, VEC>(a, p, plan, tiles, st);
  return launch_ranks<T, VEC>(a, p, plan, tiles, st);
}

template <typename T>
cudaError_t launch_large(const LoraArgs& a, void* ws, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const PlanBytes p = plan_bytes(a.tokens, a.adapters);
  char* at = static_cast<char*>(ws);
  const LoraPlan plan{reinterpret_cast<int*>(at), reinterpret_cast<int4*>(at + p.perm),
                      reinterpret_cast<int*>(at + p.perm + p.list)};
  // CTAs of the sort, an id or more for each thread (2048 rows: one 27.9 us, two 28.9; 4096 in random order: one
  // 41.5, four 40.2)
  int sorters = 1;
  while (a.tokens > 2 * kPlanThreads && sorters < kMaxCluster && sorters * kPlanThreads < a.tokens) sorters *= 2;
  const int64_t share = ((a.tokens + sorters - 1) / sorters + 31) / 32 * 32;
  const cudaError_t e = launch_grid(lora_plan_kernel, dim3(static_cast<unsigned>(sorters)), kPlanThreads, sorters > 1 ? sorters : 0,
                                    2 * sizeof(int) * static_cast<size_t>(a.adapters + 2), st, a, plan, sorters, share);
  if (e != cudaSuccess) return e;
  const bool vec = row_width<T>(a.x, a.k, a.x_stride) == E && row_width<T>(a.a, a.k, 0) == E &&
                   row_width<T>(a.b, a.rank, 0) == E && output_vectors<T>(a);
  return vec ? launch_tiles<T, true>(a, p, plan, st) : launch_tiles<T, false>(a, p, plan, st);
}

template <typename T>
cudaError_t launch_type(const LoraArgs& a, void* ws, cudaStream_t st) {
  return small_call(a.tokens) ? launch_small<T>(a, st) : launch_large<T>(a, ws, st);
}
}  // namespace

size_t lora_workspace_bytes(int64_t tokens, int64_t adapters) {
  return small_call(tokens) ? 0 : plan_bytes(tokens, adapters).total();
}

cudaError_t lora_launch(const LoraArgs& a, void* ws, cudaStream_t st) {
  if (a.dtype == F16) return launch_type<__half>(a, ws, st);
  if (a.dtype == BF16) return launch_type<__nv_bfloat16>(a, ws, st);
  return launch_type<float>(a, ws, st);
}

}  // namespace tfo
