// Dropout from a counter-based generator (philox.cuh), alone or with a
// residual sum, and its gradient (the same kernel on the output's gradient).
//
//   out[i] = (kept(i) ? x[i] / (1 - p) : 0) [+ residual[i]]
//
// in fp32 with one rounding; a dropped element is zero whatever it was.
//
// Floor: HBM (x and the residual read once, out written once). A thread takes
// 8 neighbouring elements: two generator blocks, and 16-byte accesses.
#include "heads.cuh"
#include "philox.cuh"

namespace tfo {

constexpr int kDropThreads = 256;
constexpr int kDropElems = 8;

// Eight elements of T at a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 v = Pair16<T>::unpack(w[j]);
      f[2 * j] = v.x;
      f[2 * j + 1] = v.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(Pair16<T>::pack(f[0], f[1]), Pair16<T>::pack(f[2], f[3]),
                                              Pair16<T>::pack(f[4], f[5]), Pair16<T>::pack(f[6], f[7]));
  }
}

// TO: type of the output and, with ADD, of the residual.
template <typename TX, typename TO, bool ADD, bool VEC>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const TX* __restrict__ x, const TO* __restrict__ residual,
                                                               TO* __restrict__ out, int64_t n, const DropoutArgs d) {
  griddep_launch_dependents();
  griddep_wait();
  const DropKey key(d);
  const int64_t units = (n + kDropElems - 1) / kDropElems;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; u < units;
       u += static_cast<int64_t>(gridDim.x) * kDropThreads) {
    const int64_t i = u * kDropElems;
    const bool whole = VEC && i + kDropElems <= n;
    float f[8], r[8];
    if (whole) {
      load8(x + i, f);
      if constexpr (ADD) load8(residual + i, r);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = i + j < n ? Ty<TX>::to_f(x[i + j]) : 0.f;
        if constexpr (ADD) r[j] = i + j < n ? Ty<TO>::to_f(residual[i + j]) : 0.f;
      }
    }
    const uint32_t bits = d.none ? 0xffu : d.all ? 0u : key.kept<8>(static_cast<uint64_t>(i));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool keep = bits >> j & 1;
      if constexpr (ADD) f[j] = keep ? fmaf(f[j], d.scale, r[j]) : r[j];
      else f[j] = keep ? f[j] * d.scale : 0.f;
    }
    if (whole) {
      store8(out + i, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < n) out[i + j] = Ty<TO>::from_f(f[j]);
    }
  }
}

namespace {
template <typename TX, typename TO, bool ADD>
cudaError_t launch(const void* x, const void* residual, void* out, int64_t n, const DropoutArgs& d, cudaStream_t st) {
  const bool vec = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                    reinterpret_cast<uintptr_t>(out)) % 16 == 0;
  const int64_t per_cta = static_cast<int64_t>(kDropThreads) * kDropElems;
  const int64_t blocks = std::min<int64_t>((n + per_cta - 1) / per_cta, static_cast<int64_t>(num_sms()) * 64);
  note_launch();
  return launch_dependent(vec ? dropout_kernel<TX, TO, ADD, true> : dropout_kernel<TX, TO, ADD, false>,
                          static_cast<int>(blocks), kDropThreads, st, static_cast<const TX*>(x),
                          static_cast<const TO*>(residual), static_cast<TO*>(out), n, d);
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
