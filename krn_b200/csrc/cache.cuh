// What the plan, the append and attention over the paged 8-bit cache share: page sizes, conversions.
#pragma once

#include "host.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace krnb {

constexpr int kErrDeviceIndex = 6;  // mirrors KRN_B200_ERR_DEVICE_INDEX in include/krn_b200.h

// Refuses any page but one of 16, 32, 64, 128 or 256 tokens.
inline int check_page_size(int64_t page_size) {
  if (page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0) return KRN_B200_OK;
  return fail(KRN_B200_ERR_UNSUPPORTED, "page size %lld is not available on sm_100a: pages are 16, 32, 64, 128 or 256 tokens. "
              "Instead: use one of them", (long long)page_size);
}

inline int shift_of(int64_t page_size) {
  int s = 0;
  while ((int64_t(1) << s) < page_size) ++s;
  return s;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// Two e4m3 codes in the low 16 bits, as f16.
__device__ __forceinline__ uint32_t halves_of(uint32_t codes) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(uint16_t(codes)));
  return h2;
}

}  // namespace krnb
