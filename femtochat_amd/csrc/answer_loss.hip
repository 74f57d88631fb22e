// Losses over the answers of a chat model (gfx950): the clipped policy loss with
// a KL term and the preference loss over pairs of answers, with the gradient of
// the logits.
//
// Both are functions of the answers' log-probabilities: for a token y with the
// vocabulary column x, lp = x[y] - max - log(sum(exp(x - max))), whose gradient
// is d lp / d x = onehot(y) - softmax(x).  What differs is one number per token,
// the derivative w of the loss by lp:
//   policy      r = exp(lp - old), loss = -min(r A, clip(r) A) + kl (exp(d) - d - 1)
//               with d = ref - lp:  w = -A r (unless the clip cuts) + kl (1 - exp(d));
//   preference  h = beta ((lpw - refw) - (lpl - refl)) over the sums lpw, lpl of a
//               pair's chosen and rejected answer, loss = -(1-e) log s(h) - e log s(-h)
//               with s the logistic function:  w = +-beta (e s(h) - (1-e) s(-h)).
//
// All kernels are bound by HBM: the logits are 10^4 times everything else.
//  * answer_fwd_kernel reads the logits once (a workgroup, or a wave, per column,
//    a running maximum and sum per thread) and leaves (max, sum) per token;
//  * answer_grad_kernel is then elementwise over the whole array;
//  * policy_fused_kernel holds a column in the registers of one workgroup and does
//    both, so the logits are read once and the gradient written once.
// The preference loss has no such form: w needs a whole answer's log-probability
// before the first gradient.
// exp is float32, and so are the sums over 16 bytes of logits; the sums over the
// vocabulary, a token's log-probability, its ratio and the sums over an answer are
// float64 (a ratio next to its clip decides a whole column, and an answer's sum is in
// the thousands while h is near 1).
#include "attn_device.hpp"
#include "attn_launch.hpp"

#include "../../include/femtochat_loss.h"

#include <algorithm>
#include <climits>
#include <cstdio>

namespace fc {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// Arguments of every kernel here; each reads what it needs.
struct AnswerArgs {
  const void* logits;   // (V, N) column-major, float32 or bf16
  void* dlogits;        // the same shape and type
  const void* tokens;   // N indices
  const float* old;     // N
  const float* adv;     // one value per adv_per tokens
  const float* ref;     // N (policy, or null) or one value per answer (preference)
  float* losses;        // N (policy) or pairs (preference)
  double* lp;           // N: log-probabilities, 0 where ignored (preference: workspace)
  float* logprobs;      // N or null: the same, float32
  float2* stats;        // N: (max, sum of exp(x - max)), or null
  float* weights;       // d loss / d lp: per token (policy) or per answer (preference), or null
  float* rewards;       // per answer (preference)
  float* reduced;       // null or [1]
  float* count;         // null or [1]
  const float* dy;      // null (1), 1 value, or one per loss (reduction 0)
  int64_t N;
  int64_t ignore_index;
  int64_t keep_from;    // the forward's columns from here on are to stay in the Infinity Cache
  int V;
  int index_base, index_type;
  int reduction;        // 0 none, 1 sum, 2 mean
  int pairs;            // 0: policy
  FastDiv by_T;         // tokens of an answer (weights per answer) or tokens per advantage
  int per_answer;       // the divisor, 1 where every token has its own
  int count_here;       // policy_fused_kernel counts the answers' tokens itself (kCountTokens)
  double clip_lo, clip_hi, kl, beta, smoothing;
};

__device__ inline int64_t index_at(const void* p, int64_t i, int type) {
  return type == 1 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// n / T of a token's index (N < 2^31).
__device__ inline int64_t answer_of(const AnswerArgs& a, int64_t token) {
  return a.per_answer == 1 ? token : (int64_t)divide((uint32_t)token, a.by_T);
}

// The values of a 16-byte chunk of logits.
template <typename E> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int kPer = 4;
  __device__ static inline void unpack(u32x4 u, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  }
  __device__ static inline u32x4 pack(const float* v) {
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  }
};
template <> struct Chunk<bf16> {
  static constexpr int kPer = 8;
  __device__ static inline void unpack(u32x4 u, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  __device__ static inline u32x4 pack(const float* v) {
    u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      u[i] = __builtin_bit_cast(unsigned, bf16x2{static_cast<bf16>(v[2 * i]), static_cast<bf16>(v[2 * i + 1])});
    }
    return u;
  }
};

// exp(x - m) by the hardware's base-2 exponential; -inf gives 0.
__device__ inline float exp_from(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kLog2e); }

// The same for the sums (and for moving them to another maximum): log2(e) in two parts.  The one float32 constant is 1.3e-8
// too small, which moves every log-probability the same way by that much of the
// mean distance to the maximum: 7e-8 at 2^15 Gaussian logits, and 6e-5 of an
// answer of 900 tokens.
constexpr float kLog2eLow = 1.9259629911266175e-8f;
__device__ inline float exp_sum(float x, float m) {
  const float t = x - m;
  return __builtin_amdgcn_exp2f(__builtin_fmaf(t, kLog2e, t * kLog2eLow));
}

// (maximum, sum of exp(x - maximum)) of what a thread, a group or a column has seen;
// s = 0: nothing yet, or only -inf.
// The sums are float64, of float32 sums of a chunk's values: a thread that holds a value
// near the maximum would lose most of its others to a float32 one, up to 1e-7 of the
// column where few values carry it (logits with a standard deviation of 6), always to
// the same side.
struct Column {
  float m;
  double s;
};
__device__ inline double wave_sum(double s) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  return s;
}
__device__ inline double moved(double s, float from, float to) { return s == 0.0 ? 0.0 : s * (double)exp_sum(from, to); }
// A column's threads, waves: each part is moved to the maximum of its group once (a
// tree of pairs would move it by the exponential's rounding, which leans to one side,
// at every level).
__device__ inline Column wave_combine(Column v) {
  float m = v.m;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  return Column{m, wave_sum(moved(v.s, v.m, m))};
}
__device__ inline Column combine4(const Column* c) {
  const float m = fmaxf(fmaxf(c[0].m, c[1].m), fmaxf(c[2].m, c[3].m));
  return Column{m, (moved(c[0].s, c[0].m, m) + moved(c[1].s, c[1].m, m)) + (moved(c[2].s, c[2].m, m) + moved(c[3].s, c[3].m, m))};
}

// One thread's part of a column read once: the values in front of the first
// 16-byte boundary and behind the last one go to the first threads, the chunks
// between them to thread tid, tid + kThreads, ..., kBatch loads in flight; the sum
// moves to a new maximum once per round.
template <typename E, int kThreads, int kBatch, bool kKeep>
__device__ inline Column column_pass(const E* col, int V, int tid) {
  constexpr int kPer = Chunk<E>::kPer;
  const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(col) & 15)) & 15) / (int)sizeof(E), V);
  const int chunks = (V - head) / kPer, tail = V - head - kPer * chunks;
  const E* body = col + head;
  Column acc{-INFINITY, 0.0};
  auto one = [&](float x) {
    const float m = fmaxf(acc.m, x);
    acc = Column{m, moved(acc.s, acc.m, m) + (x == -INFINITY ? 0.0 : (double)exp_sum(x, m))};
  };
  if (tid < head) one(to_f32(col[tid]));
  if (tid < tail) one(to_f32(body[kPer * chunks + tid]));
  for (int base = tid; base < chunks; base += kThreads * kBatch) {
    u32x4 u[kBatch];
    float bm = -INFINITY;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int c = min(base + kThreads * k, chunks - 1);  // a chunk past the end is the last one again, not counted below
      const u32x4* p = reinterpret_cast<const u32x4*>(body + (int64_t)kPer * c);
      u[k] = kKeep ? *p : __builtin_nontemporal_load(p);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      float v[kPer];
      Chunk<E>::unpack(u[k], v);
#pragma unroll
      for (int i = 0; i < kPer; ++i) bm = fmaxf(bm, v[i]);
    }
    const float m = fmaxf(acc.m, bm);
    const float ref = m == -INFINITY ? 0.0f : m;  // only -inf so far: every exponential is 0
    double s = moved(acc.s, acc.m, ref);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      float v[kPer], part = 0.0f;
      Chunk<E>::unpack(u[k], v);
#pragma unroll
      for (int i = 0; i < kPer; ++i) part += exp_sum(v[i], ref);
      s += base + kThreads * k < chunks ? (double)part : 0.0;
    }
    acc = Column{m, s};
  }
  return acc;
}

// lp of a token from its logit and its column's (max, sum).
__device__ inline double log_prob(float x, Column r) { return ((double)x - (double)r.m) - log(r.s); }

struct PolicyToken {
  float loss, weight;
};
// The clip is a comparison of products, so that the unclipped side's gradient
// stays where both are equal; NaN goes through to both results.
__device__ inline PolicyToken policy_token(const AnswerArgs& a, int64_t token, double lp) {
  const double A = (double)a.adv[answer_of(a, token)];
  const double r = exp(lp - (double)a.old[token]);
  const double rA = r * A, cA = (r < 1.0 - a.clip_lo ? 1.0 - a.clip_lo : r > 1.0 + a.clip_hi ? 1.0 + a.clip_hi : r) * A;
  const bool cut = rA > cA;
  double loss = -(cut ? cA : rA), w = cut ? 0.0 : -rA;
  if (a.ref != nullptr) {
    const double d = (double)a.ref[token] - lp, e = expm1(d);
    loss += a.kl * (e - d);
    w -= a.kl * e;
  }
  return PolicyToken{(float)loss, (float)w};
}

// What the column of a token leaves: its statistics, and the policy's loss and
// weight (returned) or the preference's log-probability.
template <typename E>
__device__ inline float finish_token(const AnswerArgs& a, int64_t token, const E* col, Column r) {
  const int64_t y = index_at(a.tokens, token, a.index_type) - a.index_base;
  const double lp = y >= 0 && y < a.V ? log_prob(to_f32(col[y]), r) : __builtin_nan("");
  if (a.stats != nullptr) a.stats[token] = float2{r.m, (float)r.s};
  if (a.logprobs != nullptr) a.logprobs[token] = (float)lp;
  if (a.pairs > 0) {
    a.lp[token] = lp;
    return 0.0f;
  }
  const PolicyToken p = policy_token(a, token, lp);
  if (a.losses != nullptr) a.losses[token] = p.loss;
  if (a.weights != nullptr) a.weights[token] = p.weight;
  return p.weight;
}
// A token outside the answers: no loss, no gradient, its logits are not read.
__device__ inline void skip_token(const AnswerArgs& a, int64_t token) {
  if (a.stats != nullptr) a.stats[token] = float2{0.0f, 1.0f};
  if (a.logprobs != nullptr) a.logprobs[token] = 0.0f;
  if (a.pairs > 0) {
    a.lp[token] = 0.0;
    return;
  }
  if (a.losses != nullptr) a.losses[token] = 0.0f;
  if (a.weights != nullptr) a.weights[token] = 0.0f;
}

template <typename E>
__global__ __launch_bounds__(256) void answer_fwd_kernel(AnswerArgs a) {
  __shared__ Column slots[4];
  const int64_t token = blockIdx.x;
  if (index_at(a.tokens, token, a.index_type) == a.ignore_index) {
    if (threadIdx.x == 0) skip_token(a, token);
    return;
  }
  const E* col = static_cast<const E*>(a.logits) + token * (int64_t)a.V;
  const Column v = wave_combine(token >= a.keep_from ? column_pass<E, 256, 8, true>(col, a.V, threadIdx.x)
                                                     : column_pass<E, 256, 8, false>(col, a.V, threadIdx.x));
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x / 64] = v;
  __syncthreads();
  if (threadIdx.x == 0) finish_token(a, token, col, combine4(slots));
}

// Short columns: a wave each, four to a workgroup, no barrier.
template <typename E>
__global__ __launch_bounds__(256) void answer_fwd_wave_kernel(AnswerArgs a) {
  const int64_t token = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (token >= a.N) return;
  const int lane = threadIdx.x & 63;
  if (index_at(a.tokens, token, a.index_type) == a.ignore_index) {
    if (lane == 0) skip_token(a, token);
    return;
  }
  const E* col = static_cast<const E*>(a.logits) + token * (int64_t)a.V;
  const Column r = wave_combine(token >= a.keep_from ? column_pass<E, 64, 8, true>(col, a.V, lane)
                                                     : column_pass<E, 64, 8, false>(col, a.V, lane));
  if (lane == 0) finish_token(a, token, col, r);
}

// A pair from the sums of its answers' log-probabilities: the loss (returned too),
// the two rewards and the two weights.
__device__ inline float finish_pair(const AnswerArgs& a, int pair, double chosen, double rejected) {
  const double rw = a.beta * (chosen - (double)a.ref[pair]), rl = a.beta * (rejected - (double)a.ref[pair + a.pairs]);
  const double h = rw - rl, e = a.smoothing;
  // softplus(z) = log(1 + exp(z)) and the logistic function without overflow
  const double q = log1p(exp(-fabs(h)));
  const double up = fmax(h, 0.0) + q, down = fmax(-h, 0.0) + q;  // softplus(h), softplus(-h)
  const double sig = 1.0 / (1.0 + exp(-h));                      // exp(inf) gives 0
  const double sig_neg = 1.0 / (1.0 + exp(h));
  const double dh = a.beta * (e * sig - (1.0 - e) * sig_neg);
  // fmax ignores a NaN: h says it.  A side without a share adds nothing, also where h is
  // infinite (an answer whose token has a logit of -inf).
  const float loss = h != h ? __builtin_nanf("") : (float)((e == 1.0 ? 0.0 : (1.0 - e) * down) + (e == 0.0 ? 0.0 : e * up));
  a.losses[pair] = loss;
  if (a.rewards != nullptr) {
    a.rewards[pair] = (float)rw;
    a.rewards[pair + a.pairs] = (float)rl;
  }
  if (a.weights != nullptr) {
    a.weights[pair] = (float)dh;
    a.weights[pair + a.pairs] = (float)-dh;
  }
  return loss;
}

// A workgroup per pair; the sums in a fixed order.
__global__ __launch_bounds__(1024) void preference_pair_kernel(AnswerArgs a) {
  __shared__ double slots[16];
  const int pair = blockIdx.x, T = a.per_answer;
  double sums[2];
  for (int side = 0; side < 2; ++side) {
    const double* lp = a.lp + ((int64_t)pair + (int64_t)side * a.pairs) * T;
    double s = 0.0;
    for (int t = threadIdx.x; t < T; t += 1024) s += lp[t];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x / 64] = s;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += slots[w];
    sums[side] = s;
    __syncthreads();
  }
  if (threadIdx.x == 0) finish_pair(a, pair, sums[0], sums[1]);
}

// Up to kFewPairs pairs of up to kFewTokens tokens in one workgroup, a wave per
// answer, the losses reduced too: a launch less, which is what small steps take.
constexpr int kFewPairs = 8, kFewTokens = 2048;
__global__ __launch_bounds__(128 * kFewPairs) void preference_few_kernel(AnswerArgs a) {
  __shared__ double sums[2 * kFewPairs];
  __shared__ float loss[kFewPairs];
  const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, T = a.per_answer;
  if (wave < 2 * a.pairs) {
    const double* lp = a.lp + (int64_t)wave * T;
    constexpr int kRun = 8;  // loads in flight per lane
    double s = 0.0;
    for (int base = lane; base < T; base += 64 * kRun) {
      double v[kRun];
#pragma unroll
      for (int k = 0; k < kRun; ++k) v[k] = lp[min(base + 64 * k, T - 1)];
#pragma unroll
      for (int k = 0; k < kRun; ++k) s += base + 64 * k < T ? v[k] : 0.0;
    }
    s = wave_sum(s);
    if (lane == 0) sums[wave] = s;
  }
  __syncthreads();
  if ((int)threadIdx.x < a.pairs) loss[threadIdx.x] = finish_pair(a, threadIdx.x, sums[threadIdx.x], sums[threadIdx.x + a.pairs]);
  __syncthreads();
  if (threadIdx.x == 0 && a.reduced != nullptr) {
    double total = 0.0;
    for (int i = 0; i < a.pairs; ++i) total += (double)loss[i];
    a.reduced[0] = (float)(a.reduction == 2 ? total / a.pairs : total);
  }
}

// reduced = the sum of the losses or their mean (over the tokens of answers, or
// the pairs), count = the tokens of answers (also before there are losses); one
// workgroup, float64.
__global__ __launch_bounds__(1024) void answer_reduce_kernel(AnswerArgs a) {
  __shared__ double part[16], cnt[16];
  double s = 0.0, c = 0.0;
  constexpr int kRun = 8;  // loads in flight per thread
  const int64_t n = a.pairs > 0 ? a.pairs : a.N;
  for (int64_t base = threadIdx.x; base < n; base += 1024 * kRun) {
    float loss[kRun];
    bool on[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      const int64_t i = min(base + 1024 * k, n - 1);
      loss[k] = a.losses != nullptr ? a.losses[i] : 0.0f;
      on[k] = a.pairs > 0 || index_at(a.tokens, i, a.index_type) != a.ignore_index;
    }
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      if (base + 1024 * k >= n) continue;
      s += (double)loss[k];
      c += on[k] ? 1.0 : 0.0;
    }
  }
  s = wave_sum(s);
  c = wave_sum(c);
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x / 64] = s;
    cnt[threadIdx.x / 64] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double S = 0.0, C = 0.0;
    for (int w = 0; w < 16; ++w) {
      S += part[w];
      C += cnt[w];
    }
    if (a.reduced != nullptr) a.reduced[0] = (float)(a.reduction == 2 ? S / C : S);
    if (a.count != nullptr) a.count[0] = (float)C;
  }
}

// The mean's divisor, for the mean.
__device__ inline float mean_divisor(const AnswerArgs& a) { return a.pairs > 0 ? (float)a.pairs : a.count[0]; }

// The answers' tokens, counted by one wave.
__device__ inline float count_tokens(const AnswerArgs& a, int lane) {
  constexpr int kRun = 8;  // loads in flight per lane
  const int n = (int)a.N;
  int c = 0;
  for (int base = lane; base < n + lane; base += 64 * kRun) {
    bool on[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) on[k] = index_at(a.tokens, min(base + 64 * k, n - 1), a.index_type) != a.ignore_index;
#pragma unroll
    for (int k = 0; k < kRun; ++k) c += __popcll(__ballot(on[k] && base + 64 * k < n));
  }
  return (float)c;
}

// The factor of a token's column (onehot - softmax): d loss / d lp times dy and
// the mean's divisor.
__device__ inline float grad_factor(const AnswerArgs& a, int64_t token, float weight, float divisor) {
  float w = weight;
  if (a.dy != nullptr) {
    int64_t i = 0;
    if (a.reduction == 0) {
      i = token;
      if (a.pairs > 0) {
        i = answer_of(a, token);
        if (i >= a.pairs) i -= a.pairs;
      }
    }
    w *= a.dy[i];
  }
  if (a.reduction == 2) w /= divisor;
  return w;
}

// The gradient's values of one column, for values j .. j + kPer - 1 in v:
// factor (onehot - exp(x - max) / sum), factor / sum formed once.
template <int kPer>
__device__ inline void grad_values(float* v, float m, float scaled, float factor, int y) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float p = exp_from(v[i], m) * scaled;
    v[i] = (i == y ? factor : 0.0f) - p;
  }
}

// A column's target as an offset from value j, or -1 outside the vocabulary.
__device__ inline int target_from(int64_t y, int V, int64_t j) {
  return y >= 0 && y < V ? (int)max((int64_t)-1, min(y - j, (int64_t)INT_MAX)) : -1;
}

// What the gradient's sweep does with what dlogits holds: adds to it, writes over it,
// or writes over a gradient that has its zeros already (answer_reform_kernel).
constexpr int kAdd = 0, kWrite = 1, kReform = 2;

// The whole (token, vocabulary) array in one sweep, a 16-byte chunk per thread,
// whatever V is; a chunk across two columns goes value by value, and so do the
// values in front of the array's first 16-byte boundary and behind its last one
// (chunk 0 starts at `head` values).  Columns outside the answers are written as
// zeros (kWrite) or left alone, and not read.  `block` is one of `blocks` parts of
// 256 chunks.
template <typename E, int kInto>
__device__ __attribute__((always_inline)) inline void grad_block(const AnswerArgs& a, int head, int64_t block, int64_t blocks) {
  constexpr int kPer = Chunk<E>::kPer;
  const E* x = static_cast<const E*>(a.logits);
  E* out = static_cast<E*>(a.dlogits);
  const int64_t V = a.V, n = a.N * V;
  auto value = [&](int64_t e) {  // one value, anywhere
    const int64_t token = e / V, j = e - token * V;
    const int64_t raw = index_at(a.tokens, token, a.index_type);
    if (raw == a.ignore_index) {
      if (kInto == kWrite) out[e] = from_f32<E>(0.0f);
      return;
    }
    const float2 st = a.stats[token];
    const float f = grad_factor(a, token, a.weights[a.pairs > 0 ? answer_of(a, token) : token], a.reduction == 2 ? mean_divisor(a) : 1.0f);
    float v = to_f32(x[e]);
    grad_values<1>(&v, st.x, f / st.y, f, j == raw - a.index_base ? 0 : -1);
    out[e] = from_f32<E>(kInto == kAdd ? v + to_f32(out[e]) : v);
  };
  // From the array's end: the forward's last reads are still in the Infinity Cache
  // (kKeepBytes).
  const int64_t b0 = head + (blocks - 1 - block) * (256 * kPer);  // the block's first value
  const int64_t e = b0 + (int64_t)threadIdx.x * kPer;
  if (block == 0 && (int)threadIdx.x < head) value(threadIdx.x);
  // A block inside one column has its token and what belongs to it in scalar registers.
  const int64_t t0 = b0 / V, j0 = b0 - t0 * V;
  int64_t token = t0, j = j0 + (int64_t)threadIdx.x * kPer;
  if (j0 + 256 * kPer > V) {
    if (e >= n) return;
    token = e / V;
    j = e - token * V;
    if (j + kPer > V) {
      for (int i = 0; i < kPer; ++i)
        if (e + i < n) value(e + i);
      return;
    }
  }
  const int64_t raw = index_at(a.tokens, token, a.index_type);
  u32x4* o = reinterpret_cast<u32x4*>(out + e);
  if (raw == a.ignore_index) {
    if (kInto == kWrite) __builtin_nontemporal_store(u32x4{0u, 0u, 0u, 0u}, o);
    return;
  }
  const u32x4 u = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x + e));
  u32x4 prior;
  if (kInto == kAdd) prior = __builtin_nontemporal_load(o);
  const float2 st = a.stats[token];
  const float f = grad_factor(a, token, a.weights[a.pairs > 0 ? answer_of(a, token) : token], a.reduction == 2 ? mean_divisor(a) : 1.0f);
  float v[kPer];
  Chunk<E>::unpack(u, v);
  grad_values<kPer>(v, st.x, f / st.y, f, target_from(raw - a.index_base, a.V, j));
  if (kInto == kAdd) {
    float w[kPer];
    Chunk<E>::unpack(prior, w);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] += w[i];
  }
  __builtin_nontemporal_store(Chunk<E>::pack(v), o);
}

template <typename E, int kInto>
__global__ __launch_bounds__(256) void answer_grad_kernel(AnswerArgs a, int head) {
  grad_block<E, kInto>(a, head, blockIdx.x, gridDim.x);
}

// The gradient of a loss that policy_fused_kernel has formed for dy = 1: kept where
// dy[0] is 1 (the loss as the step's last node; the grid reads one value and ends),
// formed again from the logits elsewhere.  That reads and writes what scaling the
// formed one would, less the columns outside the answers, and rounds once.
template <typename E>
__global__ __launch_bounds__(256) void answer_reform_kernel(AnswerArgs a, int head, int64_t blocks) {
  if (a.dy[0] == 1.0f) return;
  for (int64_t i = blockIdx.x; i < blocks; i += gridDim.x) grad_block<E, kReform>(a, head, i, blocks);
}

// ---- the policy loss and its gradient in one pass -------------------------------
// kThreads threads hold a column, up to kChunks 16-byte chunks each: the maximum,
// the sum of exponentials, the loss and the gradient from one read.  The column is
// cut at the array's 16-byte boundaries, so its first and last chunk may be partial
// (value by value), all others are whole.  With kThreads 64 a workgroup has four
// columns and no barrier.
// The packed values again, as far as the compiler knows other ones: it would keep
// the unpacked ones of a pass for the next (twice the registers in bf16).
__device__ inline void forget(u32x4& u) {
  asm volatile("" : "+v"(u));
}

template <typename E, int kThreads, int kChunks, int kWavesPerSimd>
__global__ __launch_bounds__(kThreads == 64 ? 256 : kThreads, kWavesPerSimd) void policy_fused_kernel(AnswerArgs a) {
  constexpr int kPer = Chunk<E>::kPer, kRows = kThreads == 64 ? 4 : 1, kWaves = kThreads / 64;
  __shared__ float smax[kWaves], sw;
  __shared__ double ssum[kWaves];
  const int64_t token = (int64_t)blockIdx.x * kRows + (kRows > 1 ? threadIdx.x / kThreads : 0);
  const int tid = kRows > 1 ? threadIdx.x % kThreads : threadIdx.x;
  if (token >= a.N) return;  // kRows > 1 only: no barrier follows
  const int V = a.V;
  const E* col = static_cast<const E*>(a.logits) + token * (int64_t)V;
  E* out = static_cast<E*>(a.dlogits) + token * (int64_t)V;
  // The gradient's array may lie differently against 16 bytes than the logits:
  // whole stores need the same offset (the launcher checks it).
  const int off = (int)(reinterpret_cast<uintptr_t>(col) & 15) / (int)sizeof(E);
  const int chunks = (off + V + kPer - 1) / kPer;
  const bool on = index_at(a.tokens, token, a.index_type) != a.ignore_index;

  u32x4 u[kChunks];
  float mx = -INFINITY;
  if (on) {
    float divisor = 1.0f;
    if (a.reduction == 2) divisor = a.count_here ? count_tokens(a, tid & 63) : a.count[0];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = tid + kThreads * k, j = kPer * c - off;
      if (j >= 0 && j + kPer <= V) {
        u[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(col + j));
      } else {  // partial or outside: -inf where there is no value
        float v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = j + i >= 0 && j + i < V ? to_f32(col[j + i]) : -INFINITY;
        u[k] = Chunk<E>::pack(v);
      }
    }
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      float v[kPer];
      Chunk<E>::unpack(u[k], v);
#pragma unroll
      for (int i = 0; i < kPer; ++i) mx = fmaxf(mx, v[i]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    if (kWaves > 1) {
      if ((tid & 63) == 0) smax[tid / 64] = mx;
      __syncthreads();
      mx = smax[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, smax[w]);
    }
    const float ref = mx == -INFINITY ? 0.0f : mx;
    double sum = 0.0;  // (as in the forward)
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      float v[kPer], part = 0.0f;
      forget(u[k]);
      Chunk<E>::unpack(u[k], v);
#pragma unroll
      for (int i = 0; i < kPer; ++i) part += exp_sum(v[i], ref);
      sum += (double)part;
    }
    sum = wave_sum(sum);
    if (kWaves > 1) {
      if ((tid & 63) == 0) ssum[tid / 64] = sum;
      __syncthreads();
      sum = ssum[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += ssum[w];
    }
    float w = 0.0f;
    if (tid < 64) w = finish_token(a, token, col, Column{mx, sum});  // every lane of the first wave the same
    if (kWaves > 1) {
      if (tid == 0) sw = w;
      __syncthreads();
      w = sw;
    }
    const float f = grad_factor(a, token, w, divisor), scaled = f / (float)sum;
    const int64_t y = index_at(a.tokens, token, a.index_type) - a.index_base;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = tid + kThreads * k, j = kPer * c - off;
      if (c >= chunks) continue;
      float v[kPer];
      forget(u[k]);
      Chunk<E>::unpack(u[k], v);
      const int64_t at = y >= 0 && y < V ? y - j : -1;
      grad_values<kPer>(v, ref, scaled, f, at >= 0 && at < kPer ? (int)at : -1);
      if (j >= 0 && j + kPer <= V) {
        *reinterpret_cast<u32x4*>(out + j) = Chunk<E>::pack(v);
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (j + i >= 0 && j + i < V) out[j + i] = from_f32<E>(v[i]);
      }
    }
    return;
  }
  if (tid == 0) skip_token(a, token);
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    const int c = tid + kThreads * k, j = kPer * c - off;
    if (c >= chunks) continue;
    if (j >= 0 && j + kPer <= V) {
      *reinterpret_cast<u32x4*>(out + j) = u32x4{0u, 0u, 0u, 0u};
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (j + i >= 0 && j + i < V) out[j + i] = from_f32<E>(0.0f);
    }
  }
}

// x *= dy[0] unless that is 1 (the loss as the step's last node): then the grid
// reads one value and ends.
template <typename E>
__global__ __launch_bounds__(256) void answer_scale_kernel(E* x, int64_t n, const float* dy) {
  const float f = dy[0];
  if (f == 1.0f) return;
  constexpr int kPer = Chunk<E>::kPer;
  const int head = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(E);
  const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
  if (tid < head && tid < n) x[tid] = from_f32<E>(to_f32(x[tid]) * f);
  const int64_t chunks = n > head ? (n - head) / kPer : 0, done = head + chunks * kPer;
  if (done + tid < n) x[done + tid] = from_f32<E>(to_f32(x[done + tid]) * f);  // fewer than kPer values
  for (int64_t c = tid; c < chunks; c += all) {
    u32x4* p = reinterpret_cast<u32x4*>(x + head) + c;
    float v[kPer];
    Chunk<E>::unpack(*p, v);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] *= f;
    *p = Chunk<E>::pack(v);
  }
}

// Columns of up to this many chunks go to a wave.
constexpr int kWaveChunks = 512;
// Up to this many tokens, each wave of the fused kernel counts those of the answers
// instead of a launch of its own before it.  us of a call, launched -> counted here:
// 24 x 259 fp32 10.8 -> 8.3, 1024 x 1000 fp32 13.9 -> 11.3, 1024 x 32768 bf16 39.0 ->
// 37.3, 4096 x 1000 fp32 19.7 -> 23.1, 8192 x 259 20.0 -> 43.6.
constexpr int kCountTokens = 1024;
constexpr int kFusedMost = 16 * 1024;  // chunks of the longest column the fused kernel holds

// Chunks of the longest column: where all columns start on a 16-byte boundary
// they are whole, elsewhere a column may begin and end inside one.
int column_chunks(const AnswerArgs& a, int per) {
  const bool whole = a.V % per == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  return (int)(((int64_t)a.V + (whole ? 0 : per - 1) + per - 1) / per);
}
template <typename E>
int column_chunks(const AnswerArgs& a) { return column_chunks(a, Chunk<E>::kPer); }

// What the forward reads last the gradient, which sweeps from the array's end, reads
// first: the last kKeepBytes are read without the streaming hint, which would keep
// them out of the Infinity Cache (256 MB), everything before them with it, and so is
// everything where no gradient follows (no statistics wanted).  us of the forward and
// the gradient of a preference step together, for 0, 128, 192, 256 MB and everything,
// a quarter of the tokens outside the answers:
//                        the logits just written         the same step again
//   8192 x 32768 bf16    248 236 235 240 263             255 246 249 243 248
//   2262 x 50257 fp32    224 205 202 205 229             209 201 196 192 200
//   4096 x 32768 bf16    127 121 120 126 126             123 122 118 114 115
//   2048 x 32768 bf16     71  60  60  60  59              69  62  62  62  61
// Behind 1 GB of foreign writes the kept columns take the forward 10-45 us more: it
// is the one that waits for those to leave the cache (8192 x 32768: 242 256 263 270 292).
constexpr int64_t kKeepBytes = (int64_t)192 << 20;

template <typename E>
hipError_t launch_fwd(AnswerArgs a, hipStream_t s) {
  a.keep_from = a.stats == nullptr ? a.N : a.N - std::min(a.N, kKeepBytes / ((int64_t)a.V * (int64_t)sizeof(E)));
  const ProfileMark mk = profile_begin(s);
  if (column_chunks<E>(a) <= kWaveChunks)
    hipLaunchKernelGGL((answer_fwd_wave_kernel<E>), dim3((unsigned)((a.N + 3) / 4)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((answer_fwd_kernel<E>), dim3((unsigned)a.N), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  profile_end(mk, "answer_fwd", s);
  return e;
}

hipError_t launch_reduce(const AnswerArgs& a, hipStream_t s) {
  const ProfileMark mk = profile_begin(s);
  hipLaunchKernelGGL(answer_reduce_kernel, dim3(1), dim3(1024), 0, s, a);
  const hipError_t e = hipGetLastError();
  profile_end(mk, "answer_reduce", s);
  return e;
}

// N V <= 2^33 values (answer_args): at most 2^23 + 1 workgroups.
template <typename E>
hipError_t launch_grad(const AnswerArgs& a, int into, hipStream_t s) {
  const int64_t n = a.N * a.V;
  const int head = (int)std::min<int64_t>(n, ((16 - (reinterpret_cast<uintptr_t>(a.logits) & 15)) & 15) / sizeof(E));
  const int64_t blocks = std::max<int64_t>(1, (n - head + 256 * Chunk<E>::kPer - 1) / (256 * Chunk<E>::kPer));
  const ProfileMark mk = profile_begin(s);
  if (into == kReform)  // eight workgroups a CU sweep the array
    hipLaunchKernelGGL((answer_reform_kernel<E>), dim3((unsigned)std::min<int64_t>(2048, blocks)), dim3(256), 0, s, a, head, blocks);
  else if (into == kWrite) hipLaunchKernelGGL((answer_grad_kernel<E, kWrite>), dim3((unsigned)blocks), dim3(256), 0, s, a, head);
  else hipLaunchKernelGGL((answer_grad_kernel<E, kAdd>), dim3((unsigned)blocks), dim3(256), 0, s, a, head);
  const hipError_t e = hipGetLastError();
  profile_end(mk, into == kReform ? "answer_reform" : "answer_grad", s);
  return e;
}

template <typename E, int kThreads, int kChunks, int kWavesPerSimd>
hipError_t launch_fused_t(const AnswerArgs& a, hipStream_t s) {
  constexpr int rows = kThreads == 64 ? 4 : 1;
  const ProfileMark mk = profile_begin(s);
  hipLaunchKernelGGL((policy_fused_kernel<E, kThreads, kChunks, kWavesPerSimd>), dim3((unsigned)((a.N + rows - 1) / rows)),
                     dim3(kThreads == 64 ? 256 : kThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  profile_end(mk, "policy_fused", s);
  return e;
}
// The shape that fits the column with the fewest idle chunks while several
// workgroups share a CU, so that one's loads run under another's reductions and
// stores (us of the shapes tried; the first of each line is taken):
//   8192 x 32768 bf16  512 x 8 192, 256 x 16 208, 256 x 25 220, 1024 x 4 240, 512 x 16 264
//   8192 x 32768 fp32  1024 x 8 376, 512 x 16 380, 256 x 32 388, 1024 x 13 465
//   2000 x 50257 bf16  256 x 25 77, 1024 x 8 84, 512 x 16 86, 1024 x 13 147
//   2000 x 50257 fp32  1024 x 13 173, 512 x 25 173
//   8192 x 8192 bf16   256 x 4 49, 128 x 8 51, 64 x 16 55, 512 x 4 68, 1024 x 4 118
//   4096 x 8192 fp32   256 x 8 46, 128 x 16 49, 512 x 8 50, 1024 x 4 63
//   8192 x 4000 bf16   64 x 8 31, 128 x 8 36, 256 x 4 36, 512 x 4 60
// At 8192 x 32768 that is 5.6 TB/s (bf16) and 5.7 (fp32), where a large copy reaches 4.9.
// Loads carry the streaming hint: without it the same step again takes 202 us of 219
// (8192 x 32768 bf16, every token in an answer), but one behind the logits' writer 238
// of 185, and behind 1 GB of other writes 268 of 198.  Stores do not: with it 207, 190
// and 190 us in these three places, but 2000 x 50257 fp32 behind its writer 173 of 157.
template <typename E>
hipError_t launch_fused(const AnswerArgs& a, hipStream_t s) {
  const int chunks = column_chunks<E>(a);
  if (chunks <= 2 * 64) return launch_fused_t<E, 64, 2, 4>(a, s);
  if (chunks <= 8 * 64) return launch_fused_t<E, 64, 8, 4>(a, s);
  if (chunks <= 4 * 256) return launch_fused_t<E, 256, 4, 8>(a, s);
  if (chunks <= 8 * 256) return launch_fused_t<E, 256, 8, 6>(a, s);
  if (chunks <= 8 * 512) return launch_fused_t<E, 512, 8, 6>(a, s);
  if (chunks <= 25 * 256) return launch_fused_t<E, 256, 25, 4>(a, s);
  if (chunks <= 8 * 1024) return launch_fused_t<E, 1024, 8, 8>(a, s);
  if (chunks <= 13 * 1024) return launch_fused_t<E, 1024, 13, 4>(a, s);
  return launch_fused_t<E, 1024, 16, 4>(a, s);
}

fc_status bad(const char* who, const char* what, fc_status code = FC_ERR_INVALID_ARGUMENT) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  return set_error(code, msg);
}
fc_status done(const char* who, hipError_t e) {
  if (e != hipSuccess) return bad(who, hipGetErrorString(e), FC_ERR_HIP);
  clear_error();
  return FC_OK;
}
bool off4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) != 0; }

// Checks of what every entry point takes; fills the arguments they share.
fc_status answer_args(const char* who, const fc_answer_desc* d, const void* logits, const void* dlogits, bool grad,
                      const void* tokens, AnswerArgs* a, uint32_t flags = FC_FLAG_OVERWRITE) {
  if (d == nullptr) return bad(who, "descriptor is null");
  if (d->V <= 0 || d->answers <= 0 || d->T <= 0) return bad(who, "V, answers and T must be positive");
  const int64_t N = (int64_t)d->answers * d->T;
  // A launch holds fewer than 2^32 threads: 256 per token, or per 1024 values of the gradient.
  if (N >= (int64_t)1 << 22) return bad(who, "at most 2^22 - 1 tokens per call", FC_ERR_UNSUPPORTED);
  if (N * d->V > (int64_t)1 << 33) return bad(who, "more than 2^33 logits", FC_ERR_UNSUPPORTED);
  if (d->index_base != 0 && d->index_base != 1) return bad(who, "index_base must be 0 or 1");
  if (d->index_type != FC_INDEX_I32 && d->index_type != FC_INDEX_I64) return bad(who, "index_type must be FC_INDEX_I32 or FC_INDEX_I64");
  if (d->reduction < FC_REDUCE_NONE || d->reduction > FC_REDUCE_MEAN) return bad(who, "unknown reduction");
  if (d->dtype != FC_F32 && d->dtype != FC_BF16) return bad(who, "dtype must be FC_F32 or FC_BF16");
  if ((d->flags & ~flags) != 0) return bad(who, "unknown flag bits");
  if (logits == nullptr || tokens == nullptr || (grad && dlogits == nullptr)) return bad(who, "a required pointer is null");
  if ((reinterpret_cast<uintptr_t>(tokens) & (d->index_type == FC_INDEX_I64 ? 7 : 3)) != 0)
    return bad(who, "tokens are not aligned to their element size");
  const uintptr_t esz = d->dtype == FC_BF16 ? 2 : 4;
  if ((reinterpret_cast<uintptr_t>(logits) & (esz - 1)) != 0 || (grad && (reinterpret_cast<uintptr_t>(dlogits) & (esz - 1)) != 0))
    return bad(who, "logits and their gradient must be aligned to their element size");
  if (grad && ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15) != 0)
    return bad(who, "logits and their gradient must lie alike against 16 bytes");
  if (grad) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(logits), g = reinterpret_cast<uintptr_t>(dlogits), n = (uintptr_t)N * d->V * esz;
    if (x != g && x < g + n && g < x + n) return bad(who, "the gradient overlaps the logits");
  }
  *a = AnswerArgs{};
  a->logits = logits;
  a->dlogits = const_cast<void*>(dlogits);
  a->tokens = tokens;
  a->N = N;
  a->V = d->V;
  a->ignore_index = d->ignore_index;
  a->index_base = d->index_base;
  a->index_type = d->index_type;
  a->reduction = d->reduction;
  a->per_answer = 1;
  return FC_OK;
}

fc_status policy_args(const char* who, const fc_answer_desc* d, const fc_policy_options* o, const float* old_logprobs,
                      const float* advantages, const float* ref_logprobs, AnswerArgs* a) {
  if (o == nullptr) return bad(who, "options are null");
  if (!(o->clip_low >= 0.0 && o->clip_low <= 1.0) || !(o->clip_high >= 0.0)) return bad(who, "clip_low must be in [0, 1] and clip_high at least 0");
  if (!(o->kl >= 0.0) || o->kl > 1e30) return bad(who, "kl must be finite and at least 0");
  if (old_logprobs == nullptr || advantages == nullptr) return bad(who, "a required pointer is null");
  if (off4(old_logprobs) || off4(advantages) || off4(ref_logprobs)) return bad(who, "float buffers must be 4-byte aligned");
  if (o->kl > 0.0 && ref_logprobs == nullptr) return bad(who, "a KL term needs ref_logprobs");
  a->old = old_logprobs;
  a->adv = advantages;
  a->ref = o->kl > 0.0 ? ref_logprobs : nullptr;
  a->clip_lo = o->clip_low;
  a->clip_hi = o->clip_high;
  a->kl = o->kl;
  if (o->advantage_per_answer != 0) {
    a->per_answer = d->T;
    a->by_T = fast_div((uint32_t)d->T);
  }
  return FC_OK;
}

hipError_t run_fwd(const AnswerArgs& a, bool b16, hipStream_t s) { return b16 ? launch_fwd<bf16>(a, s) : launch_fwd<float>(a, s); }
hipError_t run_grad(const AnswerArgs& a, const fc_answer_desc* d, hipStream_t s) {
  const int into = (d->flags & FC_FLAG_FORMED) != 0 ? kReform : (d->flags & FC_FLAG_OVERWRITE) != 0 ? kWrite : kAdd;
  return d->dtype == FC_BF16 ? launch_grad<bf16>(a, into, s) : launch_grad<float>(a, into, s);
}

}  // namespace

}  // namespace fc

using fc::AnswerArgs;
using fc::bad;
using fc::done;
using fc::off4;

extern "C" {

fc_status fc_policy_loss_fwd(const fc_answer_desc* desc, const fc_policy_options* options, const void* logits,
                             const void* tokens, const float* old_logprobs, const float* advantages,
                             const float* ref_logprobs, float* losses, float* logprobs, float* stats, float* weights,
                             float* reduced, float* count, void* stream) {
  const char* who = "fc_policy_loss_fwd";
  AnswerArgs a;
  fc_status st = fc::answer_args(who, desc, logits, nullptr, false, tokens, &a);
  if (st != FC_OK) return st;
  if ((st = fc::policy_args(who, desc, options, old_logprobs, advantages, ref_logprobs, &a)) != FC_OK) return st;
  if (losses == nullptr) return bad(who, "losses is null");
  if (off4(losses) || off4(logprobs) || off4(weights) || off4(reduced) || off4(count)) return bad(who, "float buffers must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(stats) & 7) != 0) return bad(who, "stats must be 8-byte aligned");
  a.losses = losses;
  a.logprobs = logprobs;
  a.stats = reinterpret_cast<float2*>(stats);
  a.weights = weights;
  a.reduced = reduced;
  a.count = count;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = fc::run_fwd(a, desc->dtype == FC_BF16, s);
  if (e == hipSuccess && (reduced != nullptr || count != nullptr)) e = fc::launch_reduce(a, s);
  return done(who, e);
}

fc_status fc_policy_loss_bwd(const fc_answer_desc* desc, void* dlogits, const void* logits, const void* tokens,
                             const float* stats, const float* weights, const float* dy, const float* count, void* stream) {
  const char* who = "fc_policy_loss_bwd";
  AnswerArgs a;
  const fc_status st = fc::answer_args(who, desc, logits, dlogits, true, tokens, &a, FC_FLAG_OVERWRITE | FC_FLAG_FORMED);
  if (st != FC_OK) return st;
  if ((desc->flags & FC_FLAG_FORMED) != 0 &&
      ((desc->flags & FC_FLAG_OVERWRITE) == 0 || desc->reduction == FC_REDUCE_NONE || dy == nullptr || logits == dlogits))
    return bad(who, "a formed gradient is overwritten, of a sum or a mean, and has a dy and an array of its own");
  if (stats == nullptr || weights == nullptr || (desc->reduction == FC_REDUCE_MEAN && count == nullptr))
    return bad(who, "stats, weights and (for the mean) count are required");
  if (off4(weights) || off4(dy) || off4(count)) return bad(who, "float buffers must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(stats) & 7) != 0) return bad(who, "stats must be 8-byte aligned");
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.weights = const_cast<float*>(weights);
  a.dy = dy;
  a.count = const_cast<float*>(count);
  return done(who, fc::run_grad(a, desc, static_cast<hipStream_t>(stream)));
}

fc_status fc_policy_loss_fused(const fc_answer_desc* desc, const fc_policy_options* options, const void* logits,
                               const void* tokens, const float* old_logprobs, const float* advantages,
                               const float* ref_logprobs, float* losses, float* logprobs, float* stats, float* weights,
                               float* reduced, float* count, void* dlogits, const float* dy, void* stream) {
  const char* who = "fc_policy_loss_fused";
  AnswerArgs a;
  fc_status st = fc::answer_args(who, desc, logits, dlogits, true, tokens, &a);
  if (st != FC_OK) return st;
  if ((st = fc::policy_args(who, desc, options, old_logprobs, advantages, ref_logprobs, &a)) != FC_OK) return st;
  if (losses == nullptr || (desc->reduction == FC_REDUCE_MEAN && count == nullptr))
    return bad(who, "losses and (for the mean) count are required");
  if (off4(losses) || off4(logprobs) || off4(weights) || off4(reduced) || off4(dy) || off4(count)) return bad(who, "float buffers must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(stats) & 7) != 0) return bad(who, "stats must be 8-byte aligned");
  if (logits == dlogits) return bad(who, "the gradient overlaps the logits");
  const bool b16 = desc->dtype == FC_BF16;
  if (fc::column_chunks(a, b16 ? 8 : 4) > fc::kFusedMost)
    return bad(who, "a column of more than 256 KB, with what it may begin inside, is not held at once (use fc_policy_loss_fwd and fc_policy_loss_bwd)", FC_ERR_UNSUPPORTED);
  a.count = count;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  a.count_here = a.N <= fc::kCountTokens;
  if (count != nullptr && !a.count_here) e = fc::launch_reduce(a, s);  // the mean's divisor, before the losses
  if (e != hipSuccess) return done(who, e);
  a.losses = losses;
  a.logprobs = logprobs;
  a.stats = reinterpret_cast<float2*>(stats);
  a.weights = weights;
  a.dy = dy;
  e = b16 ? fc::launch_fused<fc::bf16>(a, s) : fc::launch_fused<float>(a, s);
  a.reduced = reduced;
  if (e == hipSuccess && (reduced != nullptr || (count != nullptr && a.count_here))) e = fc::launch_reduce(a, s);
  return done(who, e);
}

fc_status fc_preference_workspace_bytes(const fc_answer_desc* desc, size_t* bytes) {
  if (desc == nullptr || bytes == nullptr) return bad("fc_preference_workspace_bytes", "a required pointer is null");
  if (desc->answers <= 0 || desc->T <= 0) return bad("fc_preference_workspace_bytes", "answers and T must be positive");
  *bytes = (size_t)desc->answers * (size_t)desc->T * sizeof(double);
  fc::clear_error();
  return FC_OK;
}

fc_status fc_preference_loss_fwd(const fc_answer_desc* desc, const fc_preference_options* options, const void* logits,
                                 const void* tokens, const float* ref_logprobs, float* losses, float* rewards,
                                 float* logprobs, float* stats, float* weights, float* reduced, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  const char* who = "fc_preference_loss_fwd";
  AnswerArgs a;
  const fc_status st = fc::answer_args(who, desc, logits, nullptr, false, tokens, &a);
  if (st != FC_OK) return st;
  if (options == nullptr) return bad(who, "options are null");
  if (desc->answers % 2 != 0) return bad(who, "answers come in pairs: the chosen ones, then the rejected ones");
  if (!(options->beta > 0.0) || options->beta > 1e30) return bad(who, "beta must be finite and above 0");
  if (!(options->label_smoothing >= 0.0 && options->label_smoothing <= 1.0)) return bad(who, "label_smoothing must be in [0, 1]");
  if (ref_logprobs == nullptr || losses == nullptr) return bad(who, "ref_logprobs and losses are required");
  if (off4(ref_logprobs) || off4(losses) || off4(rewards) || off4(logprobs) || off4(weights) || off4(reduced))
    return bad(who, "float buffers must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(stats) & 7) != 0) return bad(who, "stats must be 8-byte aligned");
  size_t need = 0;
  fc_preference_workspace_bytes(desc, &need);
  if (workspace == nullptr || workspace_bytes < need) return bad(who, "the workspace is missing or too small", FC_ERR_WORKSPACE);
  if ((reinterpret_cast<uintptr_t>(workspace) & 7) != 0) return bad(who, "the workspace must be 8-byte aligned", FC_ERR_WORKSPACE);
  a.pairs = desc->answers / 2;
  a.per_answer = desc->T;
  a.by_T = fc::fast_div((uint32_t)desc->T);
  a.ref = ref_logprobs;
  a.lp = static_cast<double*>(workspace);
  a.logprobs = logprobs;
  a.stats = reinterpret_cast<float2*>(stats);
  a.beta = options->beta;
  a.smoothing = options->label_smoothing;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = fc::run_fwd(a, desc->dtype == FC_BF16, s);
  if (e != hipSuccess) return done(who, e);
  a.losses = losses;
  a.rewards = rewards;
  a.weights = weights;
  a.reduced = reduced;
  const bool few = a.pairs <= fc::kFewPairs && desc->T <= fc::kFewTokens;
  const fc::ProfileMark mk = fc::profile_begin(s);
  if (few) hipLaunchKernelGGL(fc::preference_few_kernel, dim3(1), dim3(128 * fc::kFewPairs), 0, s, a);
  else hipLaunchKernelGGL(fc::preference_pair_kernel, dim3((unsigned)a.pairs), dim3(1024), 0, s, a);
  e = hipGetLastError();
  fc::profile_end(mk, "preference_pair", s);
  if (e == hipSuccess && reduced != nullptr && !few) e = fc::launch_reduce(a, s);
  return done(who, e);
}

fc_status fc_preference_loss_bwd(const fc_answer_desc* desc, void* dlogits, const void* logits, const void* tokens,
                                 const float* stats, const float* weights, const float* dy, void* stream) {
  const char* who = "fc_preference_loss_bwd";
  AnswerArgs a;
  const fc_status st = fc::answer_args(who, desc, logits, dlogits, true, tokens, &a);
  if (st != FC_OK) return st;
  if (desc->answers % 2 != 0) return bad(who, "answers come in pairs: the chosen ones, then the rejected ones");
  if (stats == nullptr || weights == nullptr) return bad(who, "stats and weights are required");
  if (off4(weights) || off4(dy)) return bad(who, "float buffers must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(stats) & 7) != 0) return bad(who, "stats must be 8-byte aligned");
  a.pairs = desc->answers / 2;
  a.per_answer = desc->T;
  a.by_T = fc::fast_div((uint32_t)desc->T);
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.weights = const_cast<float*>(weights);
  a.dy = dy;
  return done(who, fc::run_grad(a, desc, static_cast<hipStream_t>(stream)));
}

fc_status fc_scale_gradient(void* x, int32_t dtype, int64_t n, const float* dy, void* stream) {
  const char* who = "fc_scale_gradient";
  if (x == nullptr || dy == nullptr) return bad(who, "a required pointer is null");
  if (n <= 0) return bad(who, "n must be positive");
  if (dtype != FC_F32 && dtype != FC_BF16) return bad(who, "dtype must be FC_F32 or FC_BF16");
  if (off4(dy) || (reinterpret_cast<uintptr_t>(x) & (dtype == FC_BF16 ? 1 : 3)) != 0) return bad(who, "buffers must be aligned to their element size");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t blocks = std::min<int64_t>(2048, (n + 2047) / 2048);  // eight workgroups a CU sweep the array
  const fc::ProfileMark mk = fc::profile_begin(s);
  if (dtype == FC_BF16)
    hipLaunchKernelGGL((fc::answer_scale_kernel<fc::bf16>), dim3((unsigned)blocks), dim3(256), 0, s, static_cast<fc::bf16*>(x), n, dy);
  else
    hipLaunchKernelGGL((fc::answer_scale_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, s, static_cast<float*>(x), n, dy);
  const hipError_t e = hipGetLastError();
  fc::profile_end(mk, "scale_gradient", s);
  return done(who, e);
}

}  // extern "C"
