// Dropout from a counter-based generator (philox.cuh), alone or with a
// residual sum, and its gradient (the same kernel on the output's gradient).
//
//   out[i] = (kept(i) ? x[i] / (1 - p) : 0) [+ residual[i]]
//
// in fp32 with one rounding; a dropped element is zero whatever it was.
//
// Floor: HBM (x and the residual read once, out written once), and next to it
// the generator's 32-bit by 32-bit products, 20 for four elements. A thread
// takes units of 8 neighbouring elements, two at a time: four generator blocks
// side by side, 16-byte accesses. The rounds' keys stay in registers, and the
// counter's upper half is the same for the whole launch (2^34 elements), so that
// what it leads to in the first two rounds is made once for a thread. Measured for
// 8192 x 4096: bf16 35.7 us (57 % of the copy rate; issue slots 61 %, ALU 53 %, the
// multipliers' pipe 45 %: warps wait for busy pipes and for dispatch, hardly for memory),
// with a residual 39.6 (78 %); fp32 43 (95 %), with one 62 (99 %). Off a 16-byte border,
// element by element: bf16 62, fp32 104.
#include "heads.cuh"
#include "philox.cuh"

namespace tfo {

constexpr int kDropThreads = 256;
constexpr int kDropElems = 8;  // of a unit
// Units ahead of the one that a thread works on.
constexpr int kDropAhead = 2;

// Eight elements of T as they lie in memory.
template <typename T> struct Eight {
  static constexpr int kVecs = sizeof(T) / 2;
  uint4 v[kVecs];
  __device__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
  }
  __device__ uint32_t& word(int i) { return reinterpret_cast<uint32_t*>(v)[i]; }
  __device__ void floats(float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        f[2 * j] = __uint_as_float(word(2 * j));
        f[2 * j + 1] = __uint_as_float(word(2 * j + 1));
      } else {
        const float2 p = Pair16<T>::unpack(word(j));
        f[2 * j] = p.x;
        f[2 * j + 1] = p.y;
      }
    }
  }
  __device__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        word(2 * j) = __float_as_uint(f[2 * j]);
        word(2 * j + 1) = __float_as_uint(f[2 * j + 1]);
      } else {
        word(j) = Pair16<T>::pack(f[2 * j], f[2 * j + 1]);
      }
    }
  }
  // The first `left` of them, one by one.
  __device__ void load_some(const T* p, int64_t left) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j < left ? Ty<T>::to_f(p[j]) : 0.f;
    set(f);  // exact: the values are T's
  }
  __device__ void store_some(T* p, int64_t left) {
    float f[8];
    floats(f);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = Ty<T>::from_f(f[j]);
  }
};

// TO: type of the output and, with ADD, of the residual. n <= 2^34 elements from counter `high` * 2^32 on.
// WALK: full CTAs walk on, else each thread has one group of units.
template <typename TX, typename TO, bool ADD, bool VEC, bool WALK>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const TX* __restrict__ x, const TO* __restrict__ residual,
                                                               TO* __restrict__ out, int64_t n, uint32_t high,
                                                               const DropoutArgs d) {
  griddep_launch_dependents();
  griddep_wait();
  const DropKey key(d);
  const uint32_t units = static_cast<uint32_t>((n + kDropElems - 1) / kDropElems);
  constexpr uint32_t NEXT = kDropThreads;                         // from a unit to the thread's next one
  const uint32_t step = gridDim.x * kDropThreads * kDropAhead;
  struct Unit {
    Eight<TX> x;
    Eight<TO> r;
  };
  auto load = [&](uint32_t u, Unit& v) {
    if (u >= units) return;
    const int64_t i = static_cast<int64_t>(u) * kDropElems;
    if (VEC && i + kDropElems <= n) {
      v.x.load(x + i);
      if constexpr (ADD) v.r.load(residual + i);
    } else {
      v.x.load_some(x + i, n - i);
      if constexpr (ADD) v.r.load_some(residual + i, n - i);
    }
  };
  auto finish = [&](uint32_t u, Unit& v) {
    float f[8], r[8];
    v.x.floats(f);
    if constexpr (ADD) v.r.floats(r);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint4 w = key.block(2 * u + k, high);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float& g = f[4 * k + j];
        const bool keep = words[j] >= key.threshold;
        if constexpr (ADD) g = keep ? fmaf(g, d.scale, r[4 * k + j]) : r[4 * k + j];
        else g = keep ? g * d.scale : 0.f;
      }
    }
    if (u >= units) return;
    Eight<TO> o;
    o.set(f);
    const int64_t i = static_cast<int64_t>(u) * kDropElems;
    if (VEC && i + kDropElems <= n) o.store(out + i);
    else o.store_some(out + i, n - i);
  };
  uint32_t u = blockIdx.x * (kDropThreads * kDropAhead) + threadIdx.x;
  Unit v[kDropAhead];
#pragma unroll
  for (int k = 0; k < kDropAhead; ++k) load(u + k * NEXT, v[k]);
  for (; u < units; u += step) {
#pragma unroll
    for (int k = 0; k < kDropAhead; ++k) {
      Unit now = v[k];
      if constexpr (WALK) load(u + step + k * NEXT, v[k]);
      finish(u + k * NEXT, now);
    }
    if constexpr (!WALK) return;
  }
}

// Nothing is dropped, or everything (8192 x 4096 bf16 39 us, or 16).
template <typename TX, typename TO, bool ADD>
__global__ void __launch_bounds__(kDropThreads) dropout_border_kernel(const TX* __restrict__ x, const TO* __restrict__ residual,
                                                                      TO* __restrict__ out, int64_t n, bool all) {
  griddep_launch_dependents();
  griddep_wait();
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kDropThreads) {
    const float f = all ? 0.f : Ty<TX>::to_f(x[i]);
    if constexpr (ADD) out[i] = Ty<TO>::from_f(all ? Ty<TO>::to_f(residual[i]) : f + Ty<TO>::to_f(residual[i]));
    else out[i] = Ty<TO>::from_f(f);
  }
}

namespace {
template <typename TX, typename TO, bool ADD>
cudaError_t launch(const void* x, const void* residual, void* out, int64_t n, const DropoutArgs& d, cudaStream_t st) {
  const auto* xs = static_cast<const TX*>(x);
  const auto* rs = static_cast<const TO*>(residual);
  auto* os = static_cast<TO*>(out);
  // Walking on or done at once, by the bytes that a unit has in flight. Measured for 8192 x 4096 elements, us walking /
  // at once: bf16 36 / 40, with a residual 40 / 51; fp32 54 / 43, with a residual 66 / 62.
  constexpr bool WALK = sizeof(TX) + sizeof(TO) < 8;
  if (d.none || d.all) {
    note_launch();
    auto* kernel = dropout_border_kernel<TX, TO, ADD>;
    const int grid = static_cast<int>(std::min<int64_t>((n + kDropThreads - 1) / kDropThreads, num_sms() * 64ll));
    return launch_dependent(kernel, grid, kDropThreads, st, xs, rs, os, n, d.all);
  }
  const bool vec = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                    reinterpret_cast<uintptr_t>(out)) % 16 == 0;
  auto* kernel = vec ? dropout_kernel<TX, TO, ADD, true, WALK> : dropout_kernel<TX, TO, ADD, false, WALK>;
  constexpr int64_t MOST = 1ll << 34;
  for (int64_t i = 0; i < n; i += MOST) {
    const int64_t m = std::min(MOST, n - i);
    note_launch();
    constexpr int64_t PER_CTA = kDropThreads * kDropElems * kDropAhead;
    int64_t grid = (m + PER_CTA - 1) / PER_CTA;
    if (WALK)
      grid = std::min<int64_t>(grid, static_cast<int64_t>(num_sms()) *
                                         cached_occupancy(reinterpret_cast<const void*>(kernel), kDropThreads, 0));
    const cudaError_t e = launch_dependent(kernel, static_cast<int>(grid), kDropThreads, st, xs + i, ADD ? rs + i : rs, os + i, m,
                                           static_cast<uint32_t>(i / MOST), d);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t launch_same(const void* x, const void* residual, void* out, int64_t n, const DropoutArgs& d, cudaStream_t st) {
  return residual != nullptr ? launch<T, T, true>(x, residual, out, n, d, st) : launch<T, T, false>(x, residual, out, n, d, st);
}

// 16-bit x beside an fp32 residual stream: the sum, or (its gradient) from the stream's type to x's.
template <typename T>
cudaError_t launch_16(const void* x, int x_dtype, const void* residual, void* out, int64_t n, int out_dtype,
                      const DropoutArgs& d, cudaStream_t st) {
  if (x_dtype == out_dtype) return launch_same<T>(x, residual, out, n, d, st);
  return x_dtype == F32 ? launch<float, T, false>(x, nullptr, out, n, d, st)
                        : launch<T, float, true>(x, residual, out, n, d, st);
}
}  // namespace

cudaError_t dropout_launch(const void* x, int x_dtype, const void* residual, void* out, int out_dtype, int64_t n,
                           const DropoutArgs& d, cudaStream_t st) {
  if (x_dtype == F16 || out_dtype == F16) return launch_16<__half>(x, x_dtype, residual, out, n, out_dtype, d, st);
  if (x_dtype == BF16 || out_dtype == BF16)
    return launch_16<__nv_bfloat16>(x, x_dtype, residual, out, n, out_dtype, d, st);
  return launch_same<float>(x, residual, out, n, d, st);
}

}  // namespace tfo
