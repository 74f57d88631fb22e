// What the kernels that read a cache share: its codes as numbers.
#pragma once

#include "attn_device.hpp"
#include "cache_index.hpp"

#include <type_traits>

namespace fc {

// The four codes of a word as float32.
template <int kType>
__device__ inline void code_values(uint32_t w, float& x0, float& x1, float& x2, float& x3) {
  if constexpr (kType == FC_CACHE_I8) {
    x0 = (float)(int8_t)(w & 0xff);
    x1 = (float)(int8_t)((w >> 8) & 0xff);
    x2 = (float)(int8_t)((w >> 16) & 0xff);
    x3 = (float)(int8_t)(w >> 24);
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x0 = lo[0], x1 = lo[1], x2 = hi[0], x3 = hi[1];
  }
}

// Checks of a descriptor and its pointers (cache.hip).
fc_status check_cache(const char* who, const fc_cache_desc* d, const fc_cache* c, CacheGeom* g);

}  // namespace fc
