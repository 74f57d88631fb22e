// Scores that are more than q.k / sqrt(D): a tanh cap, a bias that falls with the
// distance of query and key, and a prefix that extends the visible keys.  The
// fast-mode kernels take them as a template argument, a sum of
//   kScored  the visible keys may follow a prefix (the other two include it);
//   kCap     s = c tanh(x / c), x = q.k / sqrt(D);
//   kBias    s - slope |q - k|;
// 0 is the plain kernel.
//
// The cap is computed from r = 1 / (exp(2x/c) + 1), one base-2 exponential and one
// reciprocal: tanh(x/c) = 1 - 2r, and its derivative, which the gradients of the
// scores are multiplied by, is 1 - tanh^2 = 4 (r - r^2) (the factor 4 goes into the
// scale at the end).  r is within 2^-22 for any x, infinities included, so a capped
// score is off by at most c 2^-21, far inside the rounding of P to bf16 for any
// cap that caps.
#pragma once

#include "attn_device.hpp"
#include "attn_launch.hpp"

namespace fc {

constexpr int kScored = 1, kCap = 2, kBias = 4;

__device__ inline float cap_part(float x, float cap_in) {
  return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * cap_in) + 1.0f);
}

// A head's slope in base 2, finite whatever the slope is, so that a query's own key (a
// distance of 0) keeps its score.
__device__ inline float base2_slope(float slope) {
  const float s = slope * kLog2e;
  return __builtin_fabsf(s) == INFINITY ? __builtin_copysignf(kFltMax, s) : s;
}

// Whether the dQ kernel sums Delta over the keys (attn_bwd_dq_fast.hpp): windows of up
// to 64 tokens, and query tiles whose keys span at most 256, as those of short sequences
// and of short documents packed into a long row do.
__host__ __device__ inline bool narrow_window(int left, int right) { return left + imax(right, 0) <= 64; }
constexpr int kExactSpan = 256;

// Whether the forward and dQ take a query tile's key tiles in two parts (eight
// waves): grids that leave at most one workgroup on a CU and have tiles that see more
// than ten key tiles, and those of up to 1.75 a CU where that is more than twenty
// (the longest tiles then no longer run alone at the end).  us of the forward and dQ,
// one part -> two: 1 x 4096 tokens, H8 D128 (256 workgroups) 101, 113 -> 83, 98;
// 1 x 6792, H8 D96 (432) 191, 226 -> 146, 177; 3 x 1500, H8 D80 (288) 48, 52 -> 39, 46;
// 4 x 1024, H12 D64 (384, sixteen key tiles) 26, 30 -> 29, 36; 4 x 2048, H8 D128 (512)
// 61, 76 -> 71, 91.
inline bool score_parts(const Problem& p, int cus, unsigned workgroups) {
  if (narrow_window(p.left, p.right)) return false;
  const int64_t span = p.prefix ? p.T : std::min((int64_t)p.T, (int64_t)p.left + p.right + kOrderRows);
  return (workgroups <= (unsigned)cus && span > 10 * kOrderTile) || (4 * (int64_t)workgroups <= 7 * (int64_t)cus && span > 20 * kOrderTile);
}

// The last visible key of query q: the window's, or the end of the prefix of the
// query's document (of the row without positions), -1 past the sequence.
__device__ inline int prefix_ub(int q, int T, int right, int pos_q, bool documents, int prefix_q) {
  if (q >= T) return -1;
  const int start = documents ? min(max(q - pos_q, 0), T) : 0;
  return min(max(q + right, start + min(max(prefix_q, 0), T) - 1), T - 1);
}
// pos and prefix point at the batch row's values (prefix at its one value when it
// is not per token); either may be null.
__device__ inline int score_ub(int q, int T, int right, const int32_t* pos, const int32_t* prefix, bool per_token) {
  if (prefix == nullptr || q >= T) return key_ub(q, T, right);
  return prefix_ub(q, T, right, pos != nullptr ? pos[q] : 0, pos != nullptr, prefix[per_token ? q : 0]);
}

// Scores of a 32-key block of S^T (lane = query): key k0 + acc_row(r, g), d0 = q -
// k0 - 4 g.  Finished base-2 scores, except with a cap alone: then -r, which the
// softmax scales by 2 cap_out and moves by cap_out in the operation that subtracts
// its reference (one multiply-add per score less).
template <int kScore>
__device__ inline void score_block(f32x16& s, int d0, float c2, float cap_in, float cap_out, float slope2) {
  const float d = (float)d0;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    float v = s[r];
    if ((kScore & (kCap | kBias)) == kCap) {
      s[r] = -cap_part(v, cap_in);
      continue;
    }
    if (kScore & kCap) v = __builtin_fmaf(-2.0f * cap_out, cap_part(v, cap_in), cap_out);
    else v *= c2;
    if (kScore & kBias) v = __builtin_fmaf(-slope2, __builtin_fabsf(d - (float)(8 * (r >> 2) + (r & 3))), v);
    s[r] = v;
  }
}

}  // namespace fc
