// Counter-based random words for dropout: Philox4x32 with ten rounds (Salmon,
// Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011).
//
// Element i of a call is dropped when word i % 4 of the block of counter
// (i / 4, offset), under the key `seed`, is below p 2^32: what is kept depends
// on the element's index alone, not on the launch, so that the backward pass
// makes the same mask again and nothing is stored.
#pragma once

#include "capi_internal.h"
#include "common.cuh"

namespace tfo {

struct DropKey {
  uint32_t k0[10], k1[10];  // the rounds' keys
  uint32_t off0, off1;      // the call's offset
  uint32_t threshold;
  __device__ explicit DropKey(const DropoutArgs& d) : threshold(d.threshold) {
    const uint64_t seed = d.seed_ptr != nullptr ? static_cast<uint64_t>(*d.seed_ptr) : d.seed;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      k0[i] = static_cast<uint32_t>(seed) + i * 0x9E3779B9u;
      k1[i] = static_cast<uint32_t>(seed >> 32) + i * 0xBB67AE85u;
    }
    off0 = static_cast<uint32_t>(d.offset);
    off1 = static_cast<uint32_t>(d.offset >> 32);
  }
  __device__ uint4 block(uint32_t counter, uint32_t counter_high) const {
    uint32_t a = counter, b = counter_high, c = off0, d = off1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t p = static_cast<uint64_t>(0xD2511F53u) * a, q = static_cast<uint64_t>(0xCD9E8D57u) * c;
      a = static_cast<uint32_t>(q >> 32) ^ b ^ k0[i];
      b = static_cast<uint32_t>(q);
      c = static_cast<uint32_t>(p >> 32) ^ d ^ k1[i];
      d = static_cast<uint32_t>(p);
    }
    return make_uint4(a, b, c, d);
  }
  __device__ uint4 block(uint64_t counter) const {
    return block(static_cast<uint32_t>(counter), static_cast<uint32_t>(counter >> 32));
  }
  // bits * 2 + (whether an element with this word is kept); the threshold is not 0.
  __device__ uint32_t push(uint32_t bits, uint32_t word) const {
    // the carry of word - threshold, shifted in
    asm("{\n\t.reg .u32 t;\n\tadd.cc.u32 t, %1, %2;\n\taddc.u32 %0, %0, %0;\n\t}" : "+r"(bits) : "r"(word), "r"(0u - threshold));
    return bits;
  }
  // Bit j: element first + j is kept. `first` is a multiple of 4 if N is.
  template <int N> __device__ uint32_t kept(uint64_t first) const {
    uint32_t bits = 0;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = N / 4 - 1; i >= 0; --i) {
        const uint4 w = block(first / 4 + i);
        bits = push(push(push(push(bits, w.w), w.z), w.y), w.x);
      }
    } else {
#pragma unroll
      for (int j = N - 1; j >= 0; --j) {
        const uint64_t i = first + j;
        const uint4 w = block(i / 4);
        const uint32_t at = static_cast<uint32_t>(i) & 3u;
        bits = push(bits, at == 0 ? w.x : at == 1 ? w.y : at == 2 ? w.z : w.w);
      }
    }
    return bits;
  }
};

}  // namespace tfo
