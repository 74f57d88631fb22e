// The fast-mode dK/dV kernel above 64 values a head with capped, biased or
// prefix-masked scores,
// one translation unit per kind, FC_SCORE (the build compiles this file once for
// each of attn_score.hpp's sums: 1, 3, 5, 7).
#include "attn_bwd_dkdv_fast.hpp"

namespace fc {

template <>
hipError_t launch_score_dkdv<FC_SCORE>(const Problem& p, const BwdArgs& a, hipStream_t s) {
  switch (p.D) {
    case 80: return launch_dkdv_fast_t<80, FC_SCORE>(p, a, s);
    case 96: return launch_dkdv_fast_t<96, FC_SCORE>(p, a, s);
    case 112: return launch_dkdv_fast_t<112, FC_SCORE>(p, a, s);
    case 128: return launch_dkdv_fast_t<128, FC_SCORE>(p, a, s);
    default: return launch_score_dkdv_vgpr<FC_SCORE>(p, a, s);
  }
}

}  // namespace fc
