// The fast-mode forward with capped, biased or prefix-masked scores,
// one translation unit per kind, FC_SCORE (the build compiles this file once for
// each of attn_score.hpp's sums: 1, 3, 5, 7).
#include "attn_fwd_fast.hpp"

namespace fc {

template <>
hipError_t launch_score_fwd<FC_SCORE>(const Problem& p, const FwdArgs& a, hipStream_t s) {
  switch (p.D) {
    case 16: return launch_fwd_fast_t<16, FC_SCORE>(p, a, s);
    case 32: return launch_fwd_fast_t<32, FC_SCORE>(p, a, s);
    case 48: return launch_fwd_fast_t<48, FC_SCORE>(p, a, s);
    case 64: return launch_fwd_fast_t<64, FC_SCORE>(p, a, s);
    case 80: return launch_fwd_fast_t<80, FC_SCORE>(p, a, s);
    case 96: return launch_fwd_fast_t<96, FC_SCORE>(p, a, s);
    case 112: return launch_fwd_fast_t<112, FC_SCORE>(p, a, s);
    case 128: return launch_fwd_fast_t<128, FC_SCORE>(p, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace fc
