// cos and sin rows of rotary positions.
//
//   angle[p, i] = 2 pi * position[p] * turns[i],  i < half
//   cos[p, i] = cos[p, half + i] = gain * cos(angle), sin likewise
//
// Positions are integers, so only the fraction of position * turns[i] matters,
// and that is a product of integers modulo 2^64: the turns are given as the
// fraction of a turn in units of 2^-64 (their integer part drops out), the low
// 64 bits of the product are the angle's fraction, and a position of 10^6 loses
// nothing (an fp32 angle would be off by 10^6 * 2^-24 = 0.06 rad there). The
// top 32 bits, as half turns in [-1, 1), go through fp32 sincospi.
//
// Bound by the writes (2 * n * 2 half values). A thread keeps the turns of V
// neighbouring pairs and walks over positions, so every store is a 16-byte
// vector (V values of the output type) and each angle is computed once for
// the two halves of the row. Measured: 131072 positions of 64 pairs, fp32 (134
// MB): 23.3 us, 89 % of the measured copy rate; 64 positions: 2.0 us, a launch.
#include <cmath>

#include "capi_internal.h"
#include "common.cuh"

namespace tfo {

struct TurnsParam {
  uint64_t v[kMaxRopeHalf];  // 2^-64 turns per position
};

__device__ __forceinline__ int64_t table_position(const void* positions, int pos_dtype, int64_t i) {
  if (pos_dtype == POS_I64) return reinterpret_cast<const int64_t*>(positions)[i];
  if (pos_dtype == POS_I32) return reinterpret_cast<const int32_t*>(positions)[i];
  return i;
}

template <typename T, int V>
__global__ void __launch_bounds__(256) rope_tables_kernel(const void* __restrict__ positions, int pos_dtype, int64_t n,
                                                          int half, float gain, T* __restrict__ cosp,
                                                          T* __restrict__ sinp, const __grid_constant__ TurnsParam turns) {
  griddep_launch_dependents();
  // thread -> (slice of V pairs, position), positions strided over the grid
  const int slices = half / V;
  const int per_block = blockDim.x / slices;  // positions of one block step (host: slices <= blockDim.x)
  const int slice = threadIdx.x % slices;
  const int first = threadIdx.x / slices;
  uint64_t t[V];
#pragma unroll
  for (int j = 0; j < V; ++j) t[j] = turns.v[slice * V + j];
  griddep_wait();
  if (first >= per_block) return;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
  int64_t p = static_cast<int64_t>(blockIdx.x) * per_block + first;
  if (p >= n) return;
  int64_t next = table_position(positions, pos_dtype, p);  // loaded one step ahead
  for (; p < n; p += step) {
    const uint64_t pos = static_cast<uint64_t>(next);  // a negative one modulo 2^64
    if (p + step < n) next = table_position(positions, pos_dtype, p + step);
    alignas(16) T c[V], s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float half_turns = static_cast<float>(static_cast<int32_t>((pos * t[j]) >> 32)) * 0x1p-31f;
      float sv, cv;
      sincospif(half_turns, &sv, &cv);
      c[j] = Ty<T>::from_f(cv * gain);
      s[j] = Ty<T>::from_f(sv * gain);
    }
    const int64_t at = p * 2 * half + slice * V;
    if constexpr (V == 1) {
      cosp[at] = cosp[at + half] = c[0];
      sinp[at] = sinp[at + half] = s[0];
    } else {
      *reinterpret_cast<uint4*>(cosp + at) = *reinterpret_cast<const uint4*>(c);
      *reinterpret_cast<uint4*>(cosp + at + half) = *reinterpret_cast<const uint4*>(c);
      *reinterpret_cast<uint4*>(sinp + at) = *reinterpret_cast<const uint4*>(s);
      *reinterpret_cast<uint4*>(sinp + at + half) = *reinterpret_cast<const uint4*>(s);
    }
  }
}

template <typename T>
static cudaError_t launch_tables(const RopeTablesArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  TurnsParam turns;
  for (int i = 0; i < kMaxRopeHalf; ++i) {
    const double t = i < a.half ? a.turns[i] - std::floor(a.turns[i]) : 0.0;  // in [0, 1)
    turns.v[i] = t < 1.0 ? static_cast<uint64_t>(std::ldexp(t, 64)) : 0;
  }
  const bool vec = a.half % V == 0 && reinterpret_cast<uintptr_t>(a.cos) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.sin) % 16 == 0;
  const int slices = vec ? a.half / V : a.half;
  const int per_block = 256 / slices;
  // 131072 positions of 64 pairs, fp32: 27.5 / 24.6 / 23.3 / 36.8 us with 2 / 8 / 16 / 64 CTAs for each SM
  const int64_t blocks = std::min<int64_t>((a.n + per_block - 1) / per_block, static_cast<int64_t>(num_sms()) * 16);
  auto* c = static_cast<T*>(a.cos);
  auto* s = static_cast<T*>(a.sin);
  const float gain = static_cast<float>(a.gain);
  note_launch();
  return vec ? launch_dependent(rope_tables_kernel<T, V>, static_cast<int>(blocks), 256, st, a.positions, a.pos_dtype,
                                a.n, a.half, gain, c, s, turns)
             : launch_dependent(rope_tables_kernel<T, 1>, static_cast<int>(blocks), 256, st, a.positions, a.pos_dtype,
                                a.n, a.half, gain, c, s, turns);
}

cudaError_t rope_tables_launch(const RopeTablesArgs& a, cudaStream_t st) {
  if (a.out_dtype == F16) return launch_tables<__half>(a, st);
  if (a.out_dtype == BF16) return launch_tables<__nv_bfloat16>(a, st);
  return launch_tables<float>(a, st);
}

}  // namespace tfo
