// Verification of drafted tokens against the target's logits, from given random
// numbers (gfx950).
//
// The next token is the place of u's share among the vocabulary's cumulative weights,
// of which one in V lies next to any u: those are exponentials and sums in float64 (in
// float32 another token would be drawn about once in a hundred rows of 2^15).  An
// acceptance is one comparison of u with a ratio of two probabilities, for which a
// denominator of float32 exponentials is enough, summed by eight in float32 and then in
// float64: within 2^-17 of itself (an exponent's three roundings of 2^-24, times 26 log 2
// where 2^26 values at 2^-26 make up the sum; then v_exp_f32's 2^-22 and the eights' sums).
// float64 operations are what costs here, not the bytes (22 us of them for 704 rows of
// 2^15 bf16 logits that are read in 10), so they are kept for the row where a sequence's
// walk ends.
//
//  * draft_stats_kernel reads every row of logits (target and draft) once: each
//    workgroup leaves a chunk's maximum and the sum of its exponentials.
//  * draft_sums_kernel, a workgroup per sequence and chunk: one wave takes a node per
//    lane, tests all of them at once and follows the accepted ones from the root; the
//    workgroup sums the weights of its chunk of the row where the walk ended.
//  * draft_pick_kernel, a wave per sequence, finds the part that u's share falls into and
//    the token in it.  In small calls the last workgroup of a sequence to leave its sums does
//    that instead (the first kernel zeroed their counter).
//  * With the drafts' distributions a weight is p - q (p where that leaves nothing), whose two sums have to be there
//    first: draft_walk_kernel, before the sums, walks and forms them.
//  * Vocabularies of up to 2048 run whole in draft_small_kernel, a workgroup per sequence.
#include "attn_device.hpp"
#include "attn_launch.hpp"

#include "../../include/femtochat_cache.h"
#include "../../include/femtochat_loss.h"

#include <algorithm>
#include <climits>
#include <cstdio>

namespace fc {

namespace {

constexpr int kDraftThreads = 256;
constexpr int kChunkValues = 8192;
constexpr int kPerThread = kChunkValues / kDraftThreads;

// A chunk's part of a row's softmax, or of its largest value.
struct ChunkStat {
  float most;  // largest logit, NaN where there is one
  int index;   // temperature 0: its first index, -1 where the chunk holds a NaN or +infinity
  double sum;  // of exp((x - most) / temperature)
};
// A row's.
struct RowStat {
  float most;
  double sum;
};
// Where a sequence's walk ended.
struct Walk {
  int last;         // node, -1: nothing is kept
  int residual;     // draws: a draft was refused there, weights max(p - q, 0)
  int next;         // temperature 0
  uint64_t struck;  // candidates: the nodes whose tokens were tried there
  RowStat p, q;
};

struct DraftArgs {
  const void* logits;
  const void* draft;
  const void* tokens;
  const float* u;
  const int32_t *parents, *counts;
  int32_t *path, *kept, *next;
  ChunkStat* stats;  // [B N target rows, B (N - 1) draft rows][chunks]
  Walk* walks;       // [B] (draws)
  double2* both;     // [B][groups][kWaves4]: sums of the two exponentials (draws)
  double* sums;      // [B][groups][kWaves4], of the weights
  int32_t* arrived;  // [B]: workgroups that left their sums
  int B, N, V, chunks;
  int groups;        // workgroups of a sequence in the walk and the pick, a part to each of their waves
  int index64, tree;
  double to_log2;    // log2(e) / temperature
};

template <typename E> constexpr int kPiece = 16 / (int)sizeof(E);
constexpr int kWaves4 = kDraftThreads / 64;

// exp((x - most) / temperature) for x <= most.  2^t = 2^n 2^f, n the nearest whole number
// (its bits come from adding 1.5 2^52) and f in [-1/2, 1/2]: a polynomial of degree 10 through
// the Chebyshev points, within 2^-51 (v_exp_f32 has 2^-22); 20 instructions.  t comes from the
// difference in float64, of which t = 0 at the largest logit whatever its size.
struct Exponent {
  double most, to_log2;  // log2(e) / temperature
  double least;          // of a difference with a weight: 2^-1000
  float most32, cut;     // both in float32: a difference's rounding moves that end by 2^-23 of itself, however large the logits
};
__device__ inline Exponent exponent_of(float most, double to_log2) {
  const double least = -1000.0 / to_log2;
  return Exponent{(double)most, to_log2, least, most, (float)least};
}
__device__ inline float nan_max(float x, float y) { return __builtin_elementwise_maximum(x, y); }
__device__ inline bool weightless(float x, const Exponent& e) { return x - e.most32 <= e.cut; }
// A logit without weight has 2^-1000, which a sum does not notice (weight_of: 0).
__device__ inline double term_of(float x, const Exponent& e) {
  const double d = weightless(x, e) ? e.least : (double)x - e.most;
  const double s = __builtin_fma(d, e.to_log2, 0x1.8p52), f = __builtin_fma(d, e.to_log2, -(s - 0x1.8p52));
  double v = 0x1.e6064532b85cep-28;
  v = __builtin_fma(v, f, 0x1.b675bd731322bp-24);
  v = __builtin_fma(v, f, 0x1.62bfd472702f4p-20);
  v = __builtin_fma(v, f, 0x1.ffcb5405401d9p-17);
  v = __builtin_fma(v, f, 0x1.4309130972597p-13);
  v = __builtin_fma(v, f, 0x1.5d87fe9d7ab38p-10);
  v = __builtin_fma(v, f, 0x1.3b2ab6fba1dcfp-7);
  v = __builtin_fma(v, f, 0x1.c6b08d703ce45p-5);
  v = __builtin_fma(v, f, 0x1.ebfbdff82c598p-3);
  v = __builtin_fma(v, f, 0x1.62e42fefa3a19p-1);
  v = __builtin_fma(v, f, 1.0);
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, s);
  // (a NaN's n is a multiple of 2^29: it stays one)
  return __builtin_bit_cast(double, (uint64_t)((uint32_t)(bits >> 32) + (n << 20)) << 32 | (uint32_t)bits);
}
__device__ inline double weight_of(float x, const Exponent& e) {
  const double v = term_of(x, e);
  return weightless(x, e) ? 0.0 : v;
}

// The values of the row from element e on, as many as 16 bytes hold; -infinity outside
// the row.  `e` counts from the 16-byte boundary at or before the row.
template <typename E>
__device__ inline void load_piece(const E* row, int V, int e, float (&x)[kPiece<E>]) {
  if (e >= 0 && e + kPiece<E> <= V) {
    if constexpr (sizeof(E) == 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(row + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = v[i];
    } else {
      const bf16x8 v = *reinterpret_cast<const bf16x8*>(row + e);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPiece<E>; ++i) x[i] = e + i >= 0 && e + i < V ? static_cast<float>(row[e + i]) : -INFINITY;
  }
}
// How many values of the row's first 16-byte piece lie before the row.
template <typename E>
__device__ inline int row_head(const E* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
}

__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// Sums of the lanes up to each.
__device__ inline double wave_scan(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double s = __shfl_up(v, o);
    if (lane >= o) v += s;
  }
  return v;
}

// One chunk of one row.
template <typename E, bool kGreedy>
__global__ __launch_bounds__(kDraftThreads) void draft_stats_kernel(DraftArgs a) {
  constexpr int P = kPiece<E>, kRounds = kPerThread / P;
  __shared__ float most4[4];
  __shared__ int index4[4];
  __shared__ double sum4[4];
  const int tid = threadIdx.x, wave = tid >> 6;
  if (tid == 0 && blockIdx.x < (unsigned)a.B) a.arrived[blockIdx.x] = 0;
  const int r = blockIdx.x / a.chunks, chunk = blockIdx.x - r * a.chunks;
  const int targets = a.B * a.N;
  const E* row = r < targets ? static_cast<const E*>(a.logits) + (int64_t)r * a.V
                             : static_cast<const E*>(a.draft) + (int64_t)(r - targets) * a.V;
  const int first = chunk * kChunkValues - row_head(row) + tid * P;
  float x[kRounds][P];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) load_piece(row, a.V, first + k * kDraftThreads * P, x[k]);
  float all = -INFINITY;
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) all = nan_max(all, x[k][i]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) all = nan_max(all, __shfl_xor(all, o));
  if ((tid & 63) == 0) most4[wave] = all;
  __syncthreads();
  all = nan_max(nan_max(most4[0], most4[1]), nan_max(most4[2], most4[3]));
  ChunkStat out;
  out.most = all;
  out.index = INT_MAX;
  out.sum = 0.0;
  if (kGreedy) {
    int at = INT_MAX;
#pragma unroll
    for (int k = kRounds - 1; k >= 0; --k)
#pragma unroll
      for (int i = P - 1; i >= 0; --i)
        if (x[k][i] == all && all != -INFINITY) at = first + k * kDraftThreads * P + i;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
    if ((tid & 63) == 0) index4[wave] = at;
    __syncthreads();
    out.index = all != all || all == INFINITY ? -1 : min(min(index4[0], index4[1]), min(index4[2], index4[3]));
  } else if (all != -INFINITY) {
    const float c = (float)a.to_log2;
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      float t = 0.0f;
#pragma unroll
      for (int i = 0; i < P; ++i) t += __builtin_amdgcn_exp2f((x[k][i] - all) * c);
      s += (double)t;
    }
    s = wave_sum(s);
    if ((tid & 63) == 0) sum4[wave] = s;
    __syncthreads();
    out.sum = sum4[0] + sum4[1] + sum4[2] + sum4[3];
  }
  if (tid == 0) a.stats[(int64_t)r * a.chunks + chunk] = out;
}

__device__ inline RowStat row_stat(const DraftArgs& a, int64_t row) {
  const ChunkStat* st = a.stats + row * a.chunks;
  const float to_log2 = (float)a.to_log2;
  RowStat r{-INFINITY, 0.0};
  for (int c0 = 0; c0 < a.chunks; c0 += 8) {
    ChunkStat s[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) s[c] = c0 + c < a.chunks ? st[c0 + c] : ChunkStat{-INFINITY, 0, 0.0};
    const float before = r.most;
#pragma unroll
    for (int c = 0; c < 8; ++c) r.most = nan_max(r.most, s[c].most);
    if (before != -INFINITY) r.sum *= (double)__builtin_amdgcn_exp2f((before - r.most) * to_log2);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (s[c].most != -INFINITY) r.sum += s[c].sum * (double)__builtin_amdgcn_exp2f((s[c].most - r.most) * to_log2);
  }
  return r;
}
// The index of a row's largest logit, -1 where it has none.
__device__ inline int row_best(const DraftArgs& a, int64_t row) {
  const ChunkStat* st = a.stats + row * a.chunks;
  float most = -INFINITY;
  int at = INT_MAX;
  bool bad = false;
  for (int c = 0; c < a.chunks; ++c) {
    const ChunkStat s = st[c];
    bad |= s.index < 0;
    if (s.most > most) most = s.most, at = s.index;
  }
  return bad || at == INT_MAX ? -1 : at;
}

__device__ inline int64_t token_at(const DraftArgs& a, int64_t i) {
  return a.index64 ? static_cast<const int64_t*>(a.tokens)[i] : static_cast<const int32_t*>(a.tokens)[i];
}
__device__ inline double read_lane(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ inline RowStat stat_at(const RowStat& s, int lane) {  // lane: any, of 64
  return RowStat{__shfl(s.most, lane), __shfl(s.sum, lane)};
}

// Sequence b's walk, by one whole wave, a node per lane; the same in every lane.
// kGreedy: best is the index of the largest logit of the lane's row; else p (and with
// draft_logits q) that row's softmax.
template <typename E, bool kGreedy>
__device__ inline Walk walk_nodes(const DraftArgs& a, int b, bool write, int best, const RowStat& row_p, const RowStat& row_q) {
  const int i = threadIdx.x & 63;
  const bool node = i >= 1 && i < a.N;
  const int count = a.counts == nullptr ? a.N : min(max(a.counts[b], 0), a.N);
  const int64_t token = node ? token_at(a, (int64_t)b * a.N + i) : -1;
  int up = i - 1;
  if (a.parents != nullptr && node) up = a.parents[(a.tree == 2 ? (int64_t)b * a.N : 0) + i];
  const double u = !kGreedy && node ? (double)a.u[(int64_t)b * a.N + i] : 1.0;
  const bool known = node && i < count && up >= 0 && up < i && token >= 0 && token < a.V;
  const int64_t row = (int64_t)b * a.N + up;
  bool chosen = false;  // tested by itself: all but candidates, whose test depends on those before them
  double p = 0.0;
  if (kGreedy) {
    chosen = __shfl(best, known ? up : 0) == (int)token && known;
  } else {
    const RowStat st = stat_at(row_p, known ? up : 0), dt = a.draft != nullptr ? stat_at(row_q, known ? up : 0) : st;
    if (known) {
      const float x = static_cast<float>(static_cast<const E*>(a.logits)[row * a.V + token]);
      float d = 0.0f;
      if (a.draft != nullptr) d = static_cast<float>(static_cast<const E*>(a.draft)[((int64_t)b * (a.N - 1) + up) * a.V + token]);
      p = weight_of(x, exponent_of(st.most, a.to_log2)) / st.sum;
      if (a.draft != nullptr) chosen = u * (weight_of(d, exponent_of(dt.most, a.to_log2)) / dt.sum) < p;
    }
  }
  // From the root to the first accepted child, and on.
  const int token32 = (int)token;
  Walk w;
  w.last = count > 0 ? 0 : -1;
  w.struck = 0;
  int kept = count > 0 ? 1 : 0, mine = -1;  // path[lane]
  if (i == 0 && count > 0) mine = 0;
  w.residual = 0;
  while (w.last >= 0) {
    const uint64_t children = __ballot(known && up == w.last);
    uint64_t hit = kGreedy || a.draft != nullptr ? __ballot(chosen) & children : 0;
    if (!kGreedy && a.draft == nullptr) {
      // In order, each against what those before it have left of p; a token that was tried is not taken.
      double left = 1.0;
      uint64_t tried = 0;
      for (uint64_t todo = children; todo != 0; todo &= todo - 1) {
        const int j = __ffsll((long long)todo) - 1;
        if (__ballot((tried >> i & 1) != 0 && token32 == __builtin_amdgcn_readlane(token32, j)) != 0) continue;
        const double pj = read_lane(p, j);
        if (read_lane(u, j) * left < pj) {
          hit = 1ull << j;
          break;
        }
        left -= pj;
        tried |= 1ull << j;
      }
      w.struck = hit == 0 ? children : 0;
    }
    if (hit == 0) {
      w.residual = a.draft != nullptr && children != 0;  // (a token outside the vocabulary was not drawn from q, and is not refused)
      break;
    }
    w.last = __ffsll((long long)hit) - 1;
    if (i == kept) mine = w.last;
    ++kept;
  }
  w.next = -1;
  w.p = w.q = RowStat{-INFINITY, 0.0};
  if (w.last >= 0) {
    if (kGreedy) {
      w.next = __shfl(best, w.last);
    } else {
      w.p = stat_at(row_p, w.last);
      if (w.residual) w.q = stat_at(row_q, w.last);
    }
  }
  if (write) {
    if (i < a.N) a.path[(int64_t)b * a.N + i] = mine;
    if (i == 0) a.kept[b] = kept;
  }
  return w;
}

// What the weights of a row come from.
template <typename E>
struct Weights {
  const E *row, *draft;  // draft: residual, else null
  Exponent p, q;
  double ip, iq;         // residual: 1 / sum
  int V;
  bool alike;            // the two rows lie alike against 16 bytes
};
template <typename E>
__device__ inline Weights<E> weights_of(const DraftArgs& a, const Walk& w, int b) {
  Weights<E> r;
  r.row = static_cast<const E*>(a.logits) + ((int64_t)b * a.N + w.last) * a.V;
  r.draft = w.residual ? static_cast<const E*>(a.draft) + ((int64_t)b * (a.N - 1) + w.last) * a.V : nullptr;
  r.p = exponent_of(w.p.most, a.to_log2);
  r.q = exponent_of(w.q.most, a.to_log2);
  r.ip = r.iq = 1.0;
  r.V = a.V;
  r.alike = row_head(r.row) == row_head(r.draft);
  return r;
}

// The weights of the piece at element e: p (times its sum), less q where the row is a residual's, and 0
// where bits (null: none) strike a value out; bits begin at element `first`.
template <typename E>
__device__ inline void weights(const Weights<E>& w, const uint32_t* bits, int first, int e, double (&out)[kPiece<E>]) {
  constexpr int P = kPiece<E>;
  float x[P], d[P];
  load_piece(w.row, w.V, e, x);
  if (w.draft != nullptr) {
    if (w.alike) {
      load_piece(w.draft, w.V, e, d);
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) d[i] = e + i >= 0 && e + i < w.V ? static_cast<float>(w.draft[e + i]) : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i) out[i] = weight_of(x[i], w.p);
  if (w.draft != nullptr) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const double rest = __builtin_fma(out[i], w.ip, -(weight_of(d[i], w.q) * w.iq));
      out[i] = rest <= 0.0 ? 0.0 : rest;  // (NaN stays)
    }
  } else if (bits != nullptr) {
    const int at = e - first;
    const uint32_t struck = bits[at >> 5] >> (at & 31);
#pragma unroll
    for (int i = 0; i < P; ++i) out[i] = (struck >> i & 1) != 0 ? 0.0 : out[i];
  }
}

// Which of kCount values are struck out: a bit each, from element `first` of the row on
// (pieces begin at multiples of their length, so one word holds a piece's).  All of a
// workgroup's threads call it, or (kThreads 64) one wave for itself.
template <int kCount, int kThreads>
__device__ inline void strike(uint32_t* bits, const DraftArgs& a, int b, uint64_t struck, int first) {
  const int i = threadIdx.x % kThreads;
  const auto sync = [] {
    if (kThreads > 64) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  for (int k = i; k < kCount / 32; k += kThreads) bits[k] = 0;
  sync();
  if (i < 64 && (struck >> i & 1) != 0) {
    const int at = (int)token_at(a, (int64_t)b * a.N + i) - first;
    if (at >= 0 && at < kCount) atomicOr(&bits[at >> 5], 1u << (at & 31));
  }
  sync();
}

// The sum of kPart weights from element `first` on, by a wave, in every lane; bits begin there too.
template <typename E, int kPart>
__device__ inline double part_sum(const Weights<E>& w, const uint32_t* bits, int first) {
  constexpr int P = kPiece<E>;
  const int lane = threadIdx.x & 63;
  double s = 0.0;
#pragma unroll 2
  for (int k = 0; k < kPart / (64 * P); ++k) {
    double v[P];
    weights<E>(w, bits, first, first + (k * 64 + lane) * P, v);
#pragma unroll
    for (int i = 0; i < P; ++i) s += v[i];
  }
  return wave_sum(s);
}

// The stats of the lane's rows, by one whole wave.
template <bool kGreedy>
__device__ inline void node_stats(const DraftArgs& a, int b, int* best, RowStat* p, RowStat* q) {
  const int i = threadIdx.x & 63;
  *best = -1;
  *p = *q = RowStat{-INFINITY, 0.0};
  if (i >= a.N) return;
  if (kGreedy) {
    *best = row_best(a, (int64_t)b * a.N + i);
    return;
  }
  *p = row_stat(a, (int64_t)b * a.N + i);
  if (a.draft != nullptr && i < a.N - 1) *q = row_stat(a, (int64_t)a.B * a.N + (int64_t)b * (a.N - 1) + i);
}

// Draws: the walk, and the sums of the two exponentials where it ended in a refusal.
template <typename E, int kPart>
__global__ __launch_bounds__(kDraftThreads) void draft_walk_kernel(DraftArgs a) {
  constexpr int P = kPiece<E>;
  __shared__ Walk walk;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int b = blockIdx.x / a.groups, group = blockIdx.x - b * a.groups;
  if (tid < 64) {
    int best;
    RowStat p, q;
    node_stats<false>(a, b, &best, &p, &q);
    const Walk w = walk_nodes<E, false>(a, b, group == 0, best, p, q);
    if (tid == 0) {
      walk = w;
      if (group == 0) a.walks[b] = w;
    }
  }
  __syncthreads();
  const Walk w = walk;
  if (w.last < 0 || w.residual == 0) return;
  const Weights<E> ws = weights_of<E>(a, w, b);
  double sp = 0.0, sq = 0.0;
  const auto add = [&](const E* row, const Exponent& e, double& s) {
    const int first = (group * kWaves4 + wave) * kPart - row_head(row);
#pragma unroll 2
    for (int k = 0; k < kPart / (64 * P); ++k) {
      float x[P];
      load_piece(row, a.V, first + (k * 64 + lane) * P, x);
#pragma unroll
      for (int i = 0; i < P; ++i) s += term_of(x[i], e);
    }
  };
  add(ws.row, ws.p, sp);
  add(ws.draft, ws.q, sq);
  sp = wave_sum(sp);
  sq = wave_sum(sq);
  if (lane == 0) a.both[((int64_t)b * a.groups + group) * kWaves4 + wave] = make_double2(sp, sq);
}

// The weights of the row where sequence b's walk ended, as they are after a residual's two sums: false
// where a row has a NaN or +infinity, or only -infinities, and so no sum.
template <typename E, bool kDraws>
__device__ inline bool drawn_row(const DraftArgs& a, int b, const Walk& w, int parts, Weights<E>* ws) {
  const int lane = threadIdx.x & 63;
  double sp = 0.0, sq = 0.0;
  if (kDraws) {  // (they come with the walk, whether it needs them or not)
    for (int i0 = 0; i0 < parts; i0 += 64) {
      const double2 s = i0 + lane < parts ? a.both[(int64_t)b * parts + i0 + lane] : make_double2(0.0, 0.0);
      sp += s.x;
      sq += s.y;
    }
  }
  if (w.last < 0 || !(w.p.sum > 0.0 && w.p.sum < 1e300) || (w.residual != 0 && !(w.q.sum > 0.0 && w.q.sum < 1e300))) return false;
  *ws = weights_of<E>(a, w, b);
  if (kDraws && w.residual != 0) {
    ws->ip = 1.0 / wave_sum(sp);
    ws->iq = 1.0 / wave_sum(sq);
  }
  return true;
}

// Above which a row's weights are something to draw from.  A residual (in units of p) of less than 2^-40
// is the roundings of equal p and q, or rarer than a draft's refusal ever is seen.
__device__ inline double least_left(const Walk& w) { return w.residual != 0 ? 0x1p-40 : 0.0; }

// The part that u's share falls into, and the token in it, by one wave.  part_at(i) is part i's sum; bits:
// kPart / 32 words of LDS.
template <typename E, int kPart, typename Part>
__device__ inline void pick_token(const DraftArgs& a, int b, const Walk& w, Weights<E> ws, int parts, double u, uint32_t* bits, Part part_at) {
  constexpr int P = kPiece<E>;
  constexpr int kMine = kPart / 64, kPieces = kMine / P;  // values of a lane
  constexpr int kHeld = 4;                                // parts of a lane that stay in registers between the sum and the search
  static_assert(kMine % P == 0, "a lane's values are whole pieces");
  const int lane = threadIdx.x & 63;
  const int head = row_head(ws.row);
  uint64_t struck = w.struck;
  double held[kHeld], total = 0.0;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) held[k] = part_at(64 * k + lane);
#pragma unroll
  for (int k = 0; k < kHeld; ++k) total += held[k];
  for (int i0 = 64 * kHeld; i0 < parts; i0 += 64) total += part_at(i0 + lane);
  total = wave_sum(total);
  double before = 0.0, target = u * total;
  int part = parts - 1;
  if (total > least_left(w)) {
    for (int i0 = 0; i0 < parts; i0 += 64) {
      double of_lane = held[0];
#pragma unroll
      for (int k = 1; k < kHeld; ++k) of_lane = i0 == 64 * k ? held[k] : of_lane;
      if (i0 >= 64 * kHeld) of_lane = part_at(i0 + lane);
      const double upto = before + wave_scan(of_lane);
      const uint64_t hit = __ballot(upto > target);
      if (hit != 0) {
        const int at = __ffsll((long long)hit) - 1;
        part = i0 + at;
        before = at > 0 ? __shfl(upto, at - 1) : before;
        break;
      }
      before = __shfl(upto, 63);
    }
  } else {  // nothing is left of p: p itself
    ws.draft = nullptr;
    struck = 0;
    for (int i = 0; i < parts; ++i) total += part_sum<E, kPart>(ws, nullptr, i * kPart - head);
    target = u * total;
    for (part = 0; part < parts - 1; ++part) {
      const double upto = before + part_sum<E, kPart>(ws, nullptr, part * kPart - head);
      if (upto > target) break;
      before = upto;
    }
  }
  target -= before;
  // The token in it.  A lane's values are neighbours here: the order of the sum is theirs.
  const int first = part * kPart - head;
  const uint32_t* strikes = nullptr;
  if (struck != 0) {
    strike<kPart, 64>(bits, a, b, struck, first);
    strikes = bits;
  }
  double v[kPieces][P];
  double mine = 0.0;
  int last_positive = -1;
  const int e0 = first + lane * kMine;
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    weights<E>(ws, strikes, first, e0 + k * P, v[k]);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      mine += v[k][i];
      if (v[k][i] > 0.0) last_positive = e0 + k * P + i;
    }
  }
  const double upto = wave_scan(mine);
  const uint64_t hit = __ballot(upto > target && last_positive >= 0), some = __ballot(last_positive >= 0);
  // (where the two sums' roundings differ, and no value is beyond the target: the last one with any weight)
  const int owner = hit != 0 ? __ffsll((long long)hit) - 1 : some != 0 ? 63 - __clzll((long long)some) : 0;
  if (lane != owner) return;
  double c = upto - mine;
  int at = last_positive;
  bool open = hit != 0;
#pragma unroll
  for (int k = 0; k < kPieces; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) {
      c += v[k][i];
      if (open && v[k][i] > 0.0 && c > target) at = e0 + k * P + i, open = false;
    }
  a.next[b] = at;
}

// u of the next token.
__device__ inline double next_uniform(const DraftArgs& a, int b) {
  return (double)fminf(fmaxf(a.u[(int64_t)b * a.N], 0.0f), 0x1.fffffep-1f);
}

// The sums of the weights, part by part.  kDraws: the walk is done.  kPicks: the last workgroup of a
// sequence to get there picks the token, instead of draft_pick_kernel.
template <typename E, bool kDraws, int kPart, bool kPicks>
__global__ __launch_bounds__(kDraftThreads) void draft_sums_kernel(DraftArgs a) {
  __shared__ Walk walk;
  __shared__ uint32_t bits[kWaves4 * kPart / 32];
  __shared__ int is_last;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int b = blockIdx.x / a.groups, group = blockIdx.x - b * a.groups;
  const int parts = a.groups * kWaves4;
  const double u = kPicks ? next_uniform(a, b) : 0.0;  // (used at the end of a chain of reads: read here)
  if (!kDraws) {
    if (tid < 64) {
      int best;
      RowStat p, q;
      node_stats<false>(a, b, &best, &p, &q);
      const Walk w = walk_nodes<E, false>(a, b, group == 0, best, p, q);
      if (tid == 0) {
        walk = w;
        if (!kPicks && group == 0) a.walks[b] = w;
      }
    }
    __syncthreads();
  }
  const Walk w = kDraws ? a.walks[b] : walk;
  Weights<E> ws;
  if (!drawn_row<E, kDraws>(a, b, w, parts, &ws)) {
    if (kPicks && group == 0 && tid == 0) a.next[b] = -1;
    return;
  }
  const int first = group * kWaves4 * kPart - row_head(ws.row);
  const uint32_t* strikes = nullptr;
  if (w.struck != 0) {
    strike<kWaves4 * kPart, kDraftThreads>(bits, a, b, w.struck, first);
    strikes = bits + wave * (kPart / 32);
  }
  const double s = part_sum<E, kPart>(ws, strikes, first + wave * kPart);
  double* sums = a.sums + (int64_t)b * parts;
  if constexpr (!kPicks) {
    if (lane == 0) sums[group * kWaves4 + wave] = s;
  } else {
    // What the last workgroup reads is written and read at the agent's scope, past the
    // XCDs' own caches; the wave waits for its store before the barrier, and the counter
    // moves behind that.  (A release at that scope would write the whole L2 back: 20 us.)
    if (lane == 0) __hip_atomic_store(&sums[group * kWaves4 + wave], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
      is_last = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.groups - 1;
    __syncthreads();
    if (is_last == 0 || wave != 0) return;
    pick_token<E, kPart>(a, b, w, ws, parts, u, bits, [&](int i) {
      return i < parts ? __hip_atomic_load(&sums[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    });
  }
}

// The next token from the parts' sums: a wave per sequence.
template <typename E, bool kDraws, int kPart>
__global__ __launch_bounds__(64) void draft_pick_kernel(DraftArgs a) {
  __shared__ uint32_t bits[kPart / 32];
  const int b = blockIdx.x, parts = a.groups * kWaves4;
  const double* sums = a.sums + (int64_t)b * parts;
  const double u = next_uniform(a, b);
  const Walk w = a.walks[b];
  Weights<E> ws;
  if (!drawn_row<E, kDraws>(a, b, w, parts, &ws)) {
    if (threadIdx.x == 0) a.next[b] = -1;
    return;
  }
  pick_token<E, kPart>(a, b, w, ws, parts, u, bits, [&](int i) { return i < parts ? sums[i] : 0.0; });
}

template <typename E>
__global__ __launch_bounds__(64) void draft_greedy_kernel(DraftArgs a) {
  const int b = blockIdx.x;
  int best;
  RowStat p, q;
  node_stats<true>(a, b, &best, &p, &q);
  const Walk w = walk_nodes<E, true>(a, b, true, best, p, q);
  if (threadIdx.x == 0) a.next[b] = w.next;
}

// A vocabulary of up to kSmallValues, a workgroup per sequence: its rows one to a wave,
// the walk, and the row where it ended, two values to a thread.
constexpr int kSmallThreads = 1024, kSmallValues = 2048, kSmallWaves = kSmallThreads / 64;

template <typename E, bool kGreedy>
__global__ __launch_bounds__(kSmallThreads) void draft_small_kernel(DraftArgs a) {
  __shared__ RowStat rows[2][64];
  __shared__ int bests[64];
  __shared__ Walk walk;
  __shared__ uint32_t bits[kSmallValues / 32];
  __shared__ double sums[2][kSmallWaves];
  __shared__ int found[kSmallWaves], tops[kSmallWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, b = blockIdx.x;
  const int drafts = a.draft != nullptr ? a.N - 1 : 0;
  for (int r = wave; r < a.N + drafts; r += kSmallWaves) {
    const bool target = r < a.N;
    const E* row = target ? static_cast<const E*>(a.logits) + ((int64_t)b * a.N + r) * a.V
                          : static_cast<const E*>(a.draft) + ((int64_t)b * (a.N - 1) + r - a.N) * a.V;
    float most = -INFINITY;
    int at = INT_MAX;
    for (int i0 = 0; i0 < a.V; i0 += 512) {  // eight loads at a time
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = i0 + k * 64 + lane < a.V ? static_cast<float>(row[i0 + k * 64 + lane]) : -INFINITY;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (kGreedy && x[k] > most) at = i0 + k * 64 + lane;
        most = nan_max(most, x[k]);
      }
    }
    float all = most;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all = nan_max(all, __shfl_xor(all, o));
    if (kGreedy) {
      at = most == all ? at : INT_MAX;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
      if (lane == 0) bests[r] = all != all || all == INFINITY || at == INT_MAX ? -1 : at;
    } else {
      const Exponent e = exponent_of(all, a.to_log2);
      double s = 0.0;
      for (int i0 = 0; i0 < a.V; i0 += 512) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = i0 + k * 64 + lane < a.V ? static_cast<float>(row[i0 + k * 64 + lane]) : -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += weight_of(x[k], e);
      }
      s = wave_sum(s);
      // (a row of -infinities: no sum)
      if (lane == 0) rows[target ? 0 : 1][target ? r : r - a.N] = RowStat{all, all == -INFINITY ? 0.0 : s};
    }
  }
  if (tid < kSmallValues / 32) bits[tid] = 0;
  __syncthreads();
  if (tid < 64) {
    const RowStat none{-INFINITY, 0.0};
    const Walk w = walk_nodes<E, kGreedy>(a, b, true, kGreedy && lane < a.N ? bests[lane] : -1, !kGreedy && lane < a.N ? rows[0][lane] : none,
                                          !kGreedy && lane < drafts ? rows[1][lane] : none);
    if (kGreedy) {
      if (tid == 0) a.next[b] = w.next;
      return;
    }
    if (tid == 0) walk = w;
    if ((w.struck >> lane & 1) != 0) {
      const int at = (int)token_at(a, (int64_t)b * a.N + lane);
      atomicOr(&bits[at >> 5], 1u << (at & 31));
    }
  }
  if (kGreedy) return;
  __syncthreads();
  const Walk w = walk;
  if (w.last < 0 || !(w.p.sum > 0.0 && w.p.sum < 1e300) || (w.residual != 0 && !(w.q.sum > 0.0 && w.q.sum < 1e300))) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const Weights<E> ws = weights_of<E>(a, w, b);
  const double ip = 1.0 / w.p.sum, iq = w.residual != 0 ? 1.0 / w.q.sum : 0.0;
  double p[2], v[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = 2 * tid + k;
    p[k] = v[k] = 0.0;
    if (i < a.V) {
      p[k] = weight_of(static_cast<float>(ws.row[i]), ws.p) * ip;
      v[k] = p[k];
      if (w.residual != 0) v[k] = fmax(p[k] - weight_of(static_cast<float>(ws.draft[i]), ws.q) * iq, 0.0);
      else if ((bits[i >> 5] >> (i & 31) & 1) != 0) v[k] = 0.0;
    }
  }
  double total = 0.0, upto = 0.0;
  for (int round = 0; round < 2; ++round) {  // a second one where nothing is left of p: p itself
    upto = wave_scan(v[0] + v[1]);
    if (lane == 63) sums[round][wave] = upto;
    __syncthreads();
    total = 0.0;
    for (int i = 0; i < kSmallWaves; ++i) {
      if (i == wave) upto += total;
      total += sums[round][i];
    }
    if (total > least_left(w)) break;
    v[0] = p[0], v[1] = p[1];
  }
  const double u = (double)fminf(fmaxf(a.u[(int64_t)b * a.N], 0.0f), 0x1.fffffep-1f), target = u * total;
  const int top = v[1] > 0.0 ? 2 * tid + 1 : v[0] > 0.0 ? 2 * tid : -1;
  const uint64_t hit = __ballot(upto > target && top >= 0), some = __ballot(top >= 0);
  const int wave_top = __shfl(top, some == 0 ? 0 : 63 - __clzll((long long)some));
  if (lane == 0) {
    found[wave] = hit == 0 ? INT_MAX : tid + __ffsll((long long)hit) - 1;
    tops[wave] = wave_top;
  }
  __syncthreads();
  int owner = INT_MAX, last = -1;
  for (int i = 0; i < kSmallWaves; ++i) owner = min(owner, found[i]), last = max(last, tops[i]);
  if (owner == INT_MAX) {  // the two sums' roundings differ: the last one with any weight
    if (tid == 0) a.next[b] = last;
  } else if (tid == owner) {
    a.next[b] = v[0] > 0.0 && (upto - v[1] > target || !(v[1] > 0.0)) ? 2 * tid : 2 * tid + 1;
  }
}

fc_status bad(const char* who, const char* what, fc_status code = FC_ERR_INVALID_ARGUMENT) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  return set_error(code, msg);
}
bool off(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

int chunks_of(const fc_verify_desc* d) {
  const int per = d->dtype == FC_BF16 ? 8 : 4;  // a row may begin inside a piece
  return (int)(((int64_t)d->V + per - 1 + kChunkValues - 1) / kChunkValues);
}
int64_t rows_of(const fc_verify_desc* d) {
  return (int64_t)d->B * d->N + (d->has_draft != 0 && d->temperature > 0.0 ? (int64_t)d->B * (d->N - 1) : 0);
}

fc_status check(const char* who, const fc_verify_desc* d) {
  if (d == nullptr) return bad(who, "descriptor is null");
  if (d->B <= 0 || d->N <= 0 || d->V <= 0) return bad(who, "B, N and V must be positive");
  if (d->N > 64) return bad(who, "at most 64 nodes", FC_ERR_UNSUPPORTED);
  if (d->V > 1 << 26) return bad(who, "at most 2^26 tokens in the vocabulary", FC_ERR_UNSUPPORTED);
  if (d->dtype != FC_F32 && d->dtype != FC_BF16) return bad(who, "dtype must be FC_F32 or FC_BF16");
  if (d->index_type != FC_INDEX_I32 && d->index_type != FC_INDEX_I64) return bad(who, "index_type must be FC_INDEX_I32 or FC_INDEX_I64");
  if (d->tree < 0 || d->tree > 2) return bad(who, "unknown kind of tree");
  if (d->tree != 0 && d->has_draft != 0) return bad(who, "draft_logits go with a run of drafted tokens, not with a tree");
  if (!(d->temperature == 0.0 || (d->temperature >= 0x1p-10 && d->temperature <= 0x1p10)))
    return bad(who, "temperature must be 0 or from 2^-10 to 2^10");
  // A launch holds fewer than 2^32 threads.
  if (d->V <= kSmallValues && (int64_t)d->B * kSmallThreads >= (int64_t)1 << 32)
    return bad(who, "fewer than 2^22 sequences of a small vocabulary", FC_ERR_UNSUPPORTED);
  if (2 * (int64_t)d->B * d->N * chunks_of(d) >= (int64_t)1 << 24) return bad(who, "too many logits: at most 2^23 chunks of 8192", FC_ERR_UNSUPPORTED);
  return FC_OK;
}

// The values of a wave in the walk and the pick: 512 (a workgroup's 2048 take it 4 us of
// float64, at 2048 a wave they take 12) unless that makes more workgroups than the GPU holds
// at once, each of which walks its sequence's nodes again.
constexpr int kShort = 512, kLong = 2048;
int groups_of(const fc_verify_desc* d, int part) {
  const int per = d->dtype == FC_BF16 ? 8 : 4;
  return (int)(((int64_t)d->V + per - 1 + kWaves4 * part - 1) / (kWaves4 * part));
}
int part_of(const fc_verify_desc* d) { return (int64_t)d->B * groups_of(d, kShort) <= 1280 ? kShort : kLong; }

struct Layout {
  size_t stats, walks, both, sums, arrived, total;
};
Layout layout_of(const fc_verify_desc* d) {
  Layout l;
  const size_t chunks = (size_t)chunks_of(d), B = (size_t)d->B, parts = (size_t)groups_of(d, part_of(d)) * kWaves4;
  const bool draws = rows_of(d) > (int64_t)d->B * d->N;
  l.stats = 0;
  l.walks = round256((size_t)rows_of(d) * chunks * sizeof(ChunkStat));
  l.both = l.walks + round256(B * sizeof(Walk));
  l.sums = l.both + (draws ? round256(B * parts * sizeof(double2)) : 0);
  l.arrived = l.sums + round256(B * parts * sizeof(double));
  l.total = d->V <= kSmallValues ? 0 : l.arrived + round256(B * sizeof(int32_t));
  return l;
}

// From this many logits on the pick is a launch of its own: the arrival it saves is 4 us of the GPU's time, the
// launch 2 to 3 of the host's, which is the longer below it (verify_drafts, 5 nodes, candidates and draws:
// 8 x 131072 18.0 and 27.8 us for 20.5 and 29.9, 64 x 8192 17.4 and 21.5 for 14.9 and 20.5).
constexpr int64_t kPickLogits = (int64_t)1 << 22;

template <typename E, int kPart>
hipError_t launch_ends(const DraftArgs& a, hipStream_t s) {
  const dim3 ends((unsigned)(a.B * a.groups));
  if (a.draft != nullptr) {
    const ProfileMark mk = profile_begin(s);
    hipLaunchKernelGGL((draft_walk_kernel<E, kPart>), ends, dim3(kDraftThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    profile_end(mk, "draft_walk", s);
    if (e != hipSuccess) return e;
  }
  const bool draws = a.draft != nullptr, picks = (int64_t)a.B * a.N * a.V < kPickLogits;
  ProfileMark mk = profile_begin(s);
  if (draws && picks) hipLaunchKernelGGL((draft_sums_kernel<E, true, kPart, true>), ends, dim3(kDraftThreads), 0, s, a);
  else if (draws) hipLaunchKernelGGL((draft_sums_kernel<E, true, kPart, false>), ends, dim3(kDraftThreads), 0, s, a);
  else if (picks) hipLaunchKernelGGL((draft_sums_kernel<E, false, kPart, true>), ends, dim3(kDraftThreads), 0, s, a);
  else hipLaunchKernelGGL((draft_sums_kernel<E, false, kPart, false>), ends, dim3(kDraftThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  profile_end(mk, "draft_sums", s);
  if (e != hipSuccess || picks) return e;
  mk = profile_begin(s);
  if (draws) hipLaunchKernelGGL((draft_pick_kernel<E, true, kPart>), dim3((unsigned)a.B), dim3(64), 0, s, a);
  else hipLaunchKernelGGL((draft_pick_kernel<E, false, kPart>), dim3((unsigned)a.B), dim3(64), 0, s, a);
  e = hipGetLastError();
  profile_end(mk, "draft_pick", s);
  return e;
}

template <typename E>
hipError_t launch_verify(const DraftArgs& a, int64_t rows, bool greedy, int part, hipStream_t s) {
  ProfileMark mk = profile_begin(s);
  if (a.V <= kSmallValues) {
    if (greedy) hipLaunchKernelGGL((draft_small_kernel<E, true>), dim3((unsigned)a.B), dim3(kSmallThreads), 0, s, a);
    else hipLaunchKernelGGL((draft_small_kernel<E, false>), dim3((unsigned)a.B), dim3(kSmallThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    profile_end(mk, "draft_small", s);
    return e;
  }
  const dim3 all((unsigned)(rows * a.chunks));
  if (greedy) hipLaunchKernelGGL((draft_stats_kernel<E, true>), all, dim3(kDraftThreads), 0, s, a);
  else hipLaunchKernelGGL((draft_stats_kernel<E, false>), all, dim3(kDraftThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  profile_end(mk, "draft_stats", s);
  if (e != hipSuccess) return e;
  if (!greedy) return part == kShort ? launch_ends<E, kShort>(a, s) : launch_ends<E, kLong>(a, s);
  mk = profile_begin(s);
  hipLaunchKernelGGL((draft_greedy_kernel<E>), dim3((unsigned)a.B), dim3(64), 0, s, a);
  e = hipGetLastError();
  profile_end(mk, "draft_greedy", s);
  return e;
}

}  // namespace

}  // namespace fc

extern "C" {

fc_status fc_verify_workspace_bytes(const fc_verify_desc* desc, size_t* bytes) {
  const char* who = "fc_verify_workspace_bytes";
  const fc_status st = fc::check(who, desc);
  if (st != FC_OK) return st;
  if (bytes == nullptr) return fc::bad(who, "bytes is null");
  *bytes = fc::layout_of(desc).total;
  fc::clear_error();
  return FC_OK;
}

fc_status fc_verify_drafts(const fc_verify_desc* desc, const void* logits, const void* draft_logits, const void* tokens,
                           const float* u, const int32_t* parents, const int32_t* counts, int32_t* path, int32_t* kept,
                           int32_t* next, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "fc_verify_drafts";
  const fc_status st = fc::check(who, desc);
  if (st != FC_OK) return st;
  const bool greedy = desc->temperature == 0.0, draft = desc->has_draft != 0 && desc->N > 1 && !greedy;
  if (logits == nullptr || tokens == nullptr || path == nullptr || kept == nullptr || next == nullptr || (draft && draft_logits == nullptr) ||
      (!greedy && u == nullptr))
    return fc::bad(who, "a required pointer is null");
  if ((desc->tree != 0) != (parents != nullptr)) return fc::bad(who, "parents and the kind of tree do not agree");
  const uintptr_t esz = desc->dtype == FC_BF16 ? 2 : 4;
  if (fc::off(logits, esz) || fc::off(draft_logits, esz)) return fc::bad(who, "logits must be aligned to their element size");
  if (fc::off(tokens, desc->index_type == FC_INDEX_I64 ? 8 : 4) || fc::off(u, 4) || fc::off(parents, 4) || fc::off(counts, 4) ||
      fc::off(path, 4) || fc::off(kept, 4) || fc::off(next, 4))
    return fc::bad(who, "tokens, u and integer buffers must be aligned to their element size");
  const fc::Layout l = fc::layout_of(desc);
  if (l.total > 0 && (workspace == nullptr || workspace_bytes < l.total)) return fc::bad(who, "the workspace is missing or too small", FC_ERR_WORKSPACE);
  if (l.total > 0 && fc::off(workspace, 256)) return fc::bad(who, "the workspace must be 256-byte aligned", FC_ERR_WORKSPACE);
  fc::DraftArgs a{};
  a.logits = logits, a.draft = draft ? draft_logits : nullptr, a.tokens = tokens, a.u = u;
  a.parents = parents, a.counts = counts, a.path = path, a.kept = kept, a.next = next;
  char* ws = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<fc::ChunkStat*>(ws + l.stats);
  a.walks = reinterpret_cast<fc::Walk*>(ws + l.walks);
  a.both = reinterpret_cast<double2*>(ws + l.both);
  a.sums = reinterpret_cast<double*>(ws + l.sums);
  a.arrived = reinterpret_cast<int32_t*>(ws + l.arrived);
  const int part = fc::part_of(desc);
  a.B = desc->B, a.N = desc->N, a.V = desc->V, a.chunks = fc::chunks_of(desc), a.groups = fc::groups_of(desc, part);
  a.index64 = desc->index_type == FC_INDEX_I64, a.tree = desc->tree;
  a.to_log2 = greedy ? 0.0 : 1.4426950408889634074 / desc->temperature;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t rows = (int64_t)a.B * a.N + (draft ? (int64_t)a.B * (a.N - 1) : 0);
  const hipError_t e = desc->dtype == FC_BF16 ? fc::launch_verify<fc::bf16>(a, rows, greedy, part, s)
                                               : fc::launch_verify<float>(a, rows, greedy, part, s);
  if (e != hipSuccess) return fc::bad(who, hipGetErrorString(e), FC_ERR_HIP);
  fc::clear_error();
  return FC_OK;
}

}  // extern "C"
