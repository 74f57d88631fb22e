// Attention over a cache, one translation unit per type of cache, FC_CACHE (the
// build compiles this file once for each fc_cache_type).
#include "cached_attn.hpp"

namespace fc {

namespace {

template <int kD>
hipError_t launch_d(const CachedAttnArgs& a, int row_blocks, int waves, hipStream_t s) {
  const unsigned slots = (unsigned)(((a.shares > 0 ? a.shares : a.g.B) * a.g.Hkv + 7) / 8 * 8);
  const dim3 grid(slots * (unsigned)a.groups);
  const ProfileMark mk = profile_begin(s);
  if (row_blocks == 1 && waves == 4) hipLaunchKernelGGL((cached_attn_kernel<FC_CACHE, kD, 1, 4>), grid, dim3(256), 0, s, a);
  else if (row_blocks == 1) hipLaunchKernelGGL((cached_attn_kernel<FC_CACHE, kD, 1, 8>), grid, dim3(512), 0, s, a);
  else if (waves == 4) hipLaunchKernelGGL((cached_attn_kernel<FC_CACHE, kD, 2, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((cached_attn_kernel<FC_CACHE, kD, 2, 8>), grid, dim3(512), 0, s, a);
  const hipError_t e = hipGetLastError();
  profile_end(mk, "cached_attn", s);
  return e;
}

}  // namespace

template <>
hipError_t launch_cached_attn<FC_CACHE>(const CachedAttnArgs& a, int row_blocks, int waves, hipStream_t s) {
  switch (a.g.D) {
    case 16: return launch_d<16>(a, row_blocks, waves, s);
    case 32: return launch_d<32>(a, row_blocks, waves, s);
    case 48: return launch_d<48>(a, row_blocks, waves, s);
    case 64: return launch_d<64>(a, row_blocks, waves, s);
    case 80: return launch_d<80>(a, row_blocks, waves, s);
    case 96: return launch_d<96>(a, row_blocks, waves, s);
    case 112: return launch_d<112>(a, row_blocks, waves, s);
    case 128: return launch_d<128>(a, row_blocks, waves, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace fc
