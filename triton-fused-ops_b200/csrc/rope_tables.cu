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
// nearest quarter turn is taken off in integers too, and only what remains, at
// most an eighth of a turn either way, is rounded to fp32: relative to itself, so
// small sines and cosines keep their bits (pairs of a base of 10^7 turn by 10^-7
// rad a position; half turns cut to 32 bits left the sine 4 % off there). sin and
// cos of the remainder are their Taylor series, whose first terms left out are
// below 2^-28.
//
// Bound by the writes (2 * n * 2 half values). A thread keeps the turns of V
// neighbouring pairs and walks over positions, so every store is a 16-byte
// vector (V values of the output type) and each angle is computed once for
// the two halves of the row. Measured: 131072 positions of 64 pairs, fp32 (134
// MB): 23.2 us, 89 % of the measured copy rate; bf16 or fp16 (67 MB): 16.5 us,
// 62 %, by the arithmetic, which does not halve with the bytes; 8192 positions,
// fp32: 4.9 us; 64: 1.9 us, a launch.
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

// sin and cos of 2 pi a 2^-64.
__device__ __forceinline__ void sincos_turns(uint64_t a, float* sine, float* cosine) {
  const uint32_t quarter = static_cast<uint32_t>((a + (1ull << 61)) >> 62);  // the nearest, 4 is 0
  const int64_t rest = static_cast<int64_t>(a - (static_cast<uint64_t>(quarter) << 62));
  // half turns, |x| <= 1/4; in two halves (64-bit conversions run at a quarter of the rate)
  const float x = fmaf(static_cast<float>(static_cast<int32_t>(rest >> 32)), 0x1p-31f,
                       static_cast<float>(static_cast<uint32_t>(rest)) * 0x1p-63f);
  const float x2 = x * x;
  // sin(pi x) = pi x - (pi x)^3 / 3! + ..., pi as the sum of two floats; cos(pi x) = 1 - (pi x)^2 / 2! + ...
  constexpr double pi = 3.14159265358979323846, p2 = pi * pi, p4 = p2 * p2;
  constexpr float pi_hi = static_cast<float>(pi), pi_lo = static_cast<float>(pi - static_cast<double>(pi_hi));
  float u = fmaf(x2, static_cast<float>(pi * p4 * p4 / 362880), static_cast<float>(-pi * p2 * p4 / 5040));
  u = fmaf(x2, u, static_cast<float>(pi * p4 / 120));
  u = fmaf(x2, u, static_cast<float>(-pi * p2 / 6));
  const float s = fmaf(x, pi_hi, x * fmaf(x2, u, pi_lo));
  float v = fmaf(x2, static_cast<float>(-p2 * p4 * p4 / 3628800), static_cast<float>(p4 * p4 / 40320));
  v = fmaf(x2, v, static_cast<float>(-p2 * p4 / 720));
  v = fmaf(x2, v, static_cast<float>(p4 / 24));
  const float c = fmaf(x2, fmaf(x2, v, static_cast<float>(-p2 / 2)), 1.f);
  const bool odd = quarter & 1;
  // a quarter turn on: (c, s) -> (-s, c)
  *sine = __uint_as_float(__float_as_uint(odd ? c : s) ^ ((quarter & 2) << 30));
  *cosine = __uint_as_float(__float_as_uint(odd ? s : c) ^ (((quarter + 1) & 2) << 30));
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
      float sv, cv;
      sincos_turns(pos * t[j], &sv, &cv);
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
    turns.v[i] = t < 1.0 ? static_cast<uint64_t>(std::nearbyint(std::ldexp(t, 64))) : 0;
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
