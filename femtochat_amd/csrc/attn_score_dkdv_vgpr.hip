// The fast-mode dK/dV kernel up to 64 values a head with capped, biased or
// prefix-masked scores,
// one translation unit per kind, FC_SCORE (the build compiles this file once for
// each of attn_score.hpp's sums: 1, 3, 5, 7), with every MFMA in its vector-register
// form (attn_bwd_dkdv_vgpr.hip).
#include "attn_bwd_dkdv_fast.hpp"

namespace fc {

template <>
hipError_t launch_score_dkdv_vgpr<FC_SCORE>(const Problem& p, const BwdArgs& a, hipStream_t s) {
  switch (p.D) {
    case 16: return launch_dkdv_fast_t<16, FC_SCORE>(p, a, s);
    case 32: return launch_dkdv_fast_t<32, FC_SCORE>(p, a, s);
    case 48: return launch_dkdv_fast_t<48, FC_SCORE>(p, a, s);
    case 64: return launch_dkdv_fast_t<64, FC_SCORE>(p, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace fc
