// The fast-mode forward (attn_fwd_fast.hpp) on plain scores; attn_score_fwd.hip has
// the capped, biased and prefix-masked ones.
#include "attn_fwd_fast.hpp"

namespace fc {

hipError_t launch_fwd_fast(const Problem& p, const FwdArgs& a, hipStream_t s) {
  switch (p.score) {
    case 0: break;
    case 1: return launch_score_fwd<1>(p, a, s);
    case 3: return launch_score_fwd<3>(p, a, s);
    case 5: return launch_score_fwd<5>(p, a, s);
    case 7: return launch_score_fwd<7>(p, a, s);
    default: return hipErrorInvalidValue;
  }
  switch (p.D) {
    case 16: return launch_fwd_fast_t<16>(p, a, s);
    case 32: return launch_fwd_fast_t<32>(p, a, s);
    case 48: return launch_fwd_fast_t<48>(p, a, s);
    case 64: return launch_fwd_fast_t<64>(p, a, s);
    case 80: return launch_fwd_fast_t<80>(p, a, s);
    case 96: return launch_fwd_fast_t<96>(p, a, s);
    case 112: return launch_fwd_fast_t<112>(p, a, s);
    case 128: return launch_fwd_fast_t<128>(p, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace fc
