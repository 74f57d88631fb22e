// Attention over a cache, one translation unit per type of cache, FC_CACHE (the
// build compiles this file once for each fc_cache_type).
#include "cached_attn.hpp"

namespace fc {

namespace {

template <int kD, int kR>
hipError_t launch_t(const CachedAttnArgs& a, hipStream_t s) {
  const unsigned slots = (unsigned)((a.items * a.g.Hkv + 7) / 8 * 8);
  const ProfileMark mk = profile_begin(s);
  hipLaunchKernelGGL((cached_attn_kernel<FC_CACHE, kD, kR>), dim3(slots * (unsigned)a.groups), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  profile_end(mk, "cached_attn", s);
  return e;
}

// (a bf16 cache's wide heads take 32 rows at most)
template <int kR>
constexpr int kWide = FC_CACHE == FC_CACHE_BF16 && kR > 2 ? 2 : kR;

template <int kR>
hipError_t launch_r(const CachedAttnArgs& a, hipStream_t s) {
  switch (a.g.D) {
    case 16: return launch_t<16, kR>(a, s);
    case 32: return launch_t<32, kR>(a, s);
    case 48: return launch_t<48, kR>(a, s);
    case 64: return launch_t<64, kR>(a, s);
    case 80: return launch_t<80, kWide<kR>>(a, s);
    case 96: return launch_t<96, kWide<kR>>(a, s);
    case 112: return launch_t<112, kWide<kR>>(a, s);
    case 128: return launch_t<128, kWide<kR>>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

template <>
hipError_t launch_cached_attn<FC_CACHE>(const CachedAttnArgs& a, int row_blocks, hipStream_t s) {
  switch (row_blocks) {
    case 1: return launch_r<1>(a, s);
    case 2: return launch_r<2>(a, s);
    default: return launch_r<4>(a, s);
  }
}

}  // namespace fc
