// Flash-attention backward, fast mode (bf16 inputs, fp32 accumulation), gfx950.
//
// Semantics as the exact-mode kernels (attn_bwd.hip, which also holds the
// preprocess) and the reference backward (src/kernels.jl:287-379; P and dS
// rounded to bf16 before their second product and dS = 0 for a query with a
// single visible key, ext/FemtoChatCUDAExt.jl:1915-1946).
//
//  * attn_bwd_dkdv_fast: persistent, one workgroup per CU; an item is 128
//    keys of one (batch, KV head), taken heaviest first from a counter per
//    XCD (or in the work order with positions, or row by row for a narrow
//    window).  Each wave keeps its 32 keys' K and V in registers (B operands
//    of S = Q K^T and dP = dO V^T), loops over the GQA group's heads and the
//    query tiles (128 queries) that can see the keys, and accumulates dK and
//    dV in registers.  Q and dO tiles are staged once into swizzled LDS and
//    read both as natural fragments (for S, dP) and through
//    ds_read_b64_tr_b16 (for dV += P^T dO and dK += dS^T Q).
//  * attn_bwd_dq_fast: a workgroup owns 128 queries of one (batch, head);
//    S^T and dP^T are recomputed with the query as the lane index so dS^T is
//    directly the B operand of dQ^T += K^T dS^T; K and V tiles are staged once
//    and K is also read transposed; dQ leaves through LDS in whole rows.
//
// The kernels themselves are in attn_bwd_dkdv_fast.hpp and attn_bwd_dq_fast.hpp;
// this unit instantiates dQ, and dK/dV for D > 64 (attn_bwd_dkdv_vgpr.hip: D <= 64).
#include "attn_bwd_dkdv_fast.hpp"
#include "attn_bwd_dq_fast.hpp"

#include <type_traits>

namespace fc {

hipError_t launch_bwd_dkdv_fast(const Problem& p, const BwdArgs& a, hipStream_t s) {
  switch (p.score) {
    case 0: break;
    case 1: return launch_score_dkdv<1>(p, a, s);
    case 3: return launch_score_dkdv<3>(p, a, s);
    case 5: return launch_score_dkdv<5>(p, a, s);
    case 7: return launch_score_dkdv<7>(p, a, s);
    default: return hipErrorInvalidValue;
  }
  switch (p.D) {
    case 16:
    case 32:
    case 48:
    case 64: return launch_bwd_dkdv_fast_vgpr(p, a, s);
    case 80: return launch_dkdv_fast_t<80>(p, a, s);
    case 96: return launch_dkdv_fast_t<96>(p, a, s);
    case 112: return launch_dkdv_fast_t<112>(p, a, s);
    case 128: return launch_dkdv_fast_t<128>(p, a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_bwd_dq_fast(const Problem& p, const BwdArgs& a, hipStream_t s) {
  switch (p.score) {
    case 0: break;
    case 1: return launch_score_dq<1>(p, a, s);
    case 3: return launch_score_dq<3>(p, a, s);
    case 5: return launch_score_dq<5>(p, a, s);
    case 7: return launch_score_dq<7>(p, a, s);
    default: return hipErrorInvalidValue;
  }
  switch (p.D) {
    case 16: return launch_dq_fast_t<16>(p, a, s);
    case 32: return launch_dq_fast_t<32>(p, a, s);
    case 48: return launch_dq_fast_t<48>(p, a, s);
    case 64: return launch_dq_fast_t<64>(p, a, s);
    case 80: return launch_dq_fast_t<80>(p, a, s);
    case 96: return launch_dq_fast_t<96>(p, a, s);
    case 112: return launch_dq_fast_t<112>(p, a, s);
    case 128: return launch_dq_fast_t<128>(p, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace fc
