// Verification of drafted tokens against the target's logits, from given random
// numbers (gfx950).
//
// What is drawn is a comparison of u with ratios of exponentials of the logits, and
// the place of u's share among the vocabulary's cumulative weights, of which one in
// V lies next to any u: so exponentials, sums and weights are float64 (a float32
// sum would draw another token about once in a hundred rows of 2^15), and the
// exponential is a polynomial of 2^f, f in [-1/2, 1/2], within 2^-47 (v_exp_f32 has
// 2^-22).
//
//  * draft_stats_kernel reads every row of logits (target and draft) once: each
//    workgroup leaves a chunk's maximum and the sum of its exponentials.
//  * draft_walk_kernel, a workgroup per sequence and chunk: one wave takes a node per
//    lane, tests all of them at once and follows the accepted ones from the root;
//    then the workgroup sums the weights of its chunk of the row where the walk ended.
//  * draft_pick_kernel finds the chunk that u's share falls into and the token in it.
// The first is bound by HBM, the others are a few microseconds of latency.
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
  float most;  // largest logit
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
  int residual;     // draws: weights max(p - q, 0)
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
  Walk* walks;       // [B]
  double* sums;      // [B][chunks], of the weights
  int B, N, V, chunks;
  int index64, tree;
  double to_log2;    // log2(e) / temperature
};

template <typename E> constexpr int kPiece = 16 / (int)sizeof(E);

// exp of (x - most) / temperature, x <= most: 0 for -infinity, NaN where either is no number.
__device__ inline double weight_of(float x, float most, double to_log2) {
  if (x == -INFINITY) return 0.0;
  double t = ((double)x - (double)most) * to_log2;
  t = t < -1080.0 ? -1080.0 : t;
  const double n = __builtin_rint(t), z = (t - n) * 0.69314718055994530942;
  double e = 1.0 / 39916800.0;  // Taylor's sum up to z^11: |z| <= ln(2) / 2 leaves 2^-47 of the value
  e = __builtin_fma(e, z, 1.0 / 3628800.0);
  e = __builtin_fma(e, z, 1.0 / 362880.0);
  e = __builtin_fma(e, z, 1.0 / 40320.0);
  e = __builtin_fma(e, z, 1.0 / 5040.0);
  e = __builtin_fma(e, z, 1.0 / 720.0);
  e = __builtin_fma(e, z, 1.0 / 120.0);
  e = __builtin_fma(e, z, 1.0 / 24.0);
  e = __builtin_fma(e, z, 1.0 / 6.0);
  e = __builtin_fma(e, z, 0.5);
  e = __builtin_fma(e, z, 1.0);
  e = __builtin_fma(e, z, 1.0);
  return __builtin_ldexp(e, (int)n);
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

// One chunk of one row.
template <typename E, bool kGreedy>
__global__ __launch_bounds__(kDraftThreads) void draft_stats_kernel(DraftArgs a) {
  constexpr int P = kPiece<E>, kRounds = kPerThread / P;
  __shared__ float most4[4];
  __shared__ int index4[4];
  __shared__ double sum4[4];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int r = blockIdx.x / a.chunks, chunk = blockIdx.x - r * a.chunks;
  const int targets = a.B * a.N;
  const E* row = r < targets ? static_cast<const E*>(a.logits) + (int64_t)r * a.V
                             : static_cast<const E*>(a.draft) + (int64_t)(r - targets) * a.V;
  const int first = chunk * kChunkValues - row_head(row) + tid * P;
  float x[kRounds][P];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) load_piece(row, a.V, first + k * kDraftThreads * P, x[k]);
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) m = fmaxf(m, x[k][i]);
  float all = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
  if ((tid & 63) == 0) most4[wave] = all;
  __syncthreads();
  all = fmaxf(fmaxf(most4[0], most4[1]), fmaxf(most4[2], most4[3]));
  ChunkStat out;
  out.most = all;
  out.index = INT_MAX;
  out.sum = 0.0;
  if (kGreedy) {
    int at = INT_MAX;
    bool bad = all == INFINITY;
#pragma unroll
    for (int k = kRounds - 1; k >= 0; --k)
#pragma unroll
      for (int i = P - 1; i >= 0; --i) {
        if (x[k][i] == all && all != -INFINITY) at = first + k * kDraftThreads * P + i;
        bad |= x[k][i] != x[k][i];
      }
    at = bad ? -1 : at;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
    if ((tid & 63) == 0) index4[wave] = at;
    __syncthreads();
    out.index = min(min(index4[0], index4[1]), min(index4[2], index4[3]));
  } else {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kRounds; ++k)
#pragma unroll
      for (int i = 0; i < P; ++i) s += weight_of(x[k][i], all, a.to_log2);
    s = wave_sum(s);
    if ((tid & 63) == 0) sum4[wave] = s;
    __syncthreads();
    out.sum = sum4[0] + sum4[1] + sum4[2] + sum4[3];
  }
  if (tid == 0) a.stats[(int64_t)r * a.chunks + chunk] = out;
}

__device__ inline RowStat row_stat(const DraftArgs& a, int64_t row) {
  const ChunkStat* st = a.stats + row * a.chunks;
  RowStat r;
  r.most = -INFINITY;
  for (int c = 0; c < a.chunks; ++c) r.most = fmaxf(r.most, st[c].most);
  r.sum = 0.0;
  for (int c = 0; c < a.chunks; ++c) {
    const ChunkStat s = st[c];
    // (a chunk of -infinities has the sum 0, or NaN where it holds one)
    r.sum += s.most == -INFINITY ? s.sum : s.sum * weight_of(s.most, r.most, a.to_log2);
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
__device__ inline double shfl64(double v, int from) { return __shfl(v, from); }

// Sequence b's walk, by one whole wave, a node per lane; the same in every lane.
template <typename E, bool kGreedy>
__device__ inline Walk walk_nodes(const DraftArgs& a, int b, bool write) {
  const int i = threadIdx.x & 63;
  const int count = a.counts == nullptr ? a.N : min(max(a.counts[b], 0), a.N);
  const bool there = i >= 1 && i < count;
  int up = i - 1;
  if (a.parents != nullptr && there) up = a.parents[(a.tree == 2 ? (int64_t)b * a.N : 0) + i];
  const bool linked = there && up >= 0 && up < i;
  const int64_t token = there ? token_at(a, (int64_t)b * a.N + i) : -1;
  const bool known = linked && token >= 0 && token < a.V;
  const int64_t row = (int64_t)b * a.N + up;
  bool chosen = false;
  if (kGreedy) {
    chosen = known && row_best(a, row) == (int)token;
  } else {
    double p = 0.0, q = 0.0;
    if (known) {
      const RowStat st = row_stat(a, row);
      p = weight_of(static_cast<float>(static_cast<const E*>(a.logits)[row * a.V + token]), st.most, a.to_log2) / st.sum;
      if (a.draft != nullptr) {
        const int64_t drow = (int64_t)b * (a.N - 1) + up;
        const RowStat dt = row_stat(a, (int64_t)a.B * a.N + drow);
        q = weight_of(static_cast<float>(static_cast<const E*>(a.draft)[drow * a.V + token]), dt.most, a.to_log2) / dt.sum;
      }
    }
    const double u = there ? (double)a.u[(int64_t)b * a.N + i] : 1.0;
    if (a.draft != nullptr) {
      chosen = known && u * q < p;
    } else {
      // Siblings before this node: whether one has its token, and what they have of p.
      bool again = false;
      const int token32 = (int)token;
      for (int j = 1; j < count; ++j) {
        const int uj = __shfl(up, j), tj = __shfl(token32, j), kj = __shfl((int)known, j);
        again |= j < i && kj != 0 && uj == up && tj == token32;
      }
      double left = 1.0;
      for (int j = 1; j < count; ++j) {
        const int uj = __shfl(up, j), fresh = __shfl((int)(known && !again), j);
        const double pj = shfl64(p, j);
        left -= j < i && fresh != 0 && uj == up ? pj : 0.0;
      }
      chosen = known && !again && u * left < p;
    }
  }
  // From the root to the first accepted child, and on.
  Walk w;
  w.last = count > 0 ? 0 : -1;
  w.residual = 0, w.struck = 0;
  w.p = w.q = RowStat{-INFINITY, 0.0};
  int kept = count > 0 ? 1 : 0, mine = -1;  // path[lane]
  if (i == 0 && count > 0) mine = 0;
  while (w.last >= 0) {
    const uint64_t hit = __ballot(chosen && up == w.last);
    if (hit == 0) break;
    w.last = __ffsll((long long)hit) - 1;
    if (i == kept) mine = w.last;
    ++kept;
  }
  w.struck = a.draft == nullptr ? __ballot(known && up == w.last) : 0;
  w.residual = a.draft != nullptr && kept < count;
  if (write) {
    if (i < a.N) a.path[(int64_t)b * a.N + i] = mine;
    if (i == 0) a.kept[b] = kept;
  }
  return w;
}

// Which of a chunk's values are struck out: a bit each, from element `first` of the row on.
__device__ inline void strike(uint32_t* bits, const DraftArgs& a, int b, uint64_t struck, int first) {
  for (int i = threadIdx.x; i < kChunkValues / 32; i += kDraftThreads) bits[i] = 0;
  __syncthreads();
  const int i = threadIdx.x;
  if (i < 64 && (struck >> i & 1) != 0) {
    const int at = (int)token_at(a, (int64_t)b * a.N + i) - first;
    if (at >= 0 && at < kChunkValues) atomicOr(&bits[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
}

// The weights of the piece at element e: p, less q where the row is a residual's, and 0
// where bits (null: none) strike a value out.
template <typename E>
__device__ inline void weights(const DraftArgs& a, const Walk& w, const E* row, const E* drow, const uint32_t* bits, int first,
                               int e, double (&out)[kPiece<E>]) {
  constexpr int P = kPiece<E>;
  float x[P];
  load_piece(row, a.V, e, x);
  const double ip = 1.0 / w.p.sum;
#pragma unroll
  for (int i = 0; i < P; ++i) out[i] = weight_of(x[i], w.p.most, a.to_log2) * ip;
  if (drow != nullptr) {
    const double iq = 1.0 / w.q.sum;
    float d[P];
    if (row_head(drow) == row_head(row)) {
      load_piece(drow, a.V, e, d);
    } else {  // the draft's row lies otherwise against 16 bytes: its values one by one
#pragma unroll
      for (int i = 0; i < P; ++i) d[i] = e + i >= 0 && e + i < a.V ? static_cast<float>(drow[e + i]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const double rest = out[i] - weight_of(d[i], w.q.most, a.to_log2) * iq;
      out[i] = rest > 0.0 ? rest : rest != rest ? rest : 0.0;
    }
  } else if (bits != nullptr) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int at = e + i - first;
      if ((bits[at >> 5] >> (at & 31) & 1) != 0) out[i] = 0.0;
    }
  }
}

// Their sum over a chunk, in every thread.
template <typename E>
__device__ inline double chunk_sum(const DraftArgs& a, const Walk& w, const E* row, const E* drow, const uint32_t* bits, int first,
                                   double* sum4) {
  constexpr int P = kPiece<E>, kRounds = kPerThread / P;
  const int tid = threadIdx.x;
  double s = 0.0;
#pragma unroll 2
  for (int k = 0; k < kRounds; ++k) {
    double v[P];
    weights<E>(a, w, row, drow, bits, first, first + (k * kDraftThreads + tid) * P, v);
#pragma unroll
    for (int i = 0; i < P; ++i) s += v[i];
  }
  s = wave_sum(s);
  __syncthreads();
  if ((tid & 63) == 0) sum4[tid >> 6] = s;
  __syncthreads();
  return sum4[0] + sum4[1] + sum4[2] + sum4[3];
}

template <typename E>
__global__ __launch_bounds__(kDraftThreads) void draft_walk_kernel(DraftArgs a) {
  __shared__ Walk walk;
  __shared__ uint32_t bits[kChunkValues / 32];
  __shared__ double sum4[4];
  const int tid = threadIdx.x, b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  if (tid < 64) {
    Walk w = walk_nodes<E, false>(a, b, chunk == 0);
    if (w.last >= 0) {
      w.p = row_stat(a, (int64_t)b * a.N + w.last);
      if (w.residual) w.q = row_stat(a, (int64_t)a.B * a.N + (int64_t)b * (a.N - 1) + w.last);
    }
    if (tid == 0) {
      walk = w;
      if (chunk == 0) a.walks[b] = w;
    }
  }
  __syncthreads();
  const Walk w = walk;
  if (w.last < 0) return;
  const E* row = static_cast<const E*>(a.logits) + ((int64_t)b * a.N + w.last) * a.V;
  const E* drow = w.residual ? static_cast<const E*>(a.draft) + ((int64_t)b * (a.N - 1) + w.last) * a.V : nullptr;
  const int first = chunk * kChunkValues - row_head(row);
  if (w.struck != 0) strike(bits, a, b, w.struck, first);
  const double s = chunk_sum(a, w, row, drow, w.struck != 0 ? bits : nullptr, first, sum4);
  if (tid == 0) a.sums[(int64_t)b * a.chunks + chunk] = s;
}

template <typename E>
__global__ __launch_bounds__(kDraftThreads) void draft_pick_kernel(DraftArgs a) {
  constexpr int P = kPiece<E>, kPieces = kPerThread / P;
  __shared__ uint32_t bits[kChunkValues / 32];
  __shared__ double sum4[4];
  __shared__ int found4[4], last4[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, b = blockIdx.x;
  const Walk w = a.walks[b];
  if (w.last < 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const double* sums = a.sums + (int64_t)b * a.chunks;
  double total = 0.0;
  for (int c = 0; c < a.chunks; ++c) total += sums[c];
  if (!(total >= 0.0 && total < 1e300)) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const double u = (double)fminf(fmaxf(a.u[(int64_t)b * a.N], 0.0f), 0x1.fffffep-1f);
  const E* row = static_cast<const E*>(a.logits) + ((int64_t)b * a.N + w.last) * a.V;
  const E* drow = w.residual ? static_cast<const E*>(a.draft) + ((int64_t)b * (a.N - 1) + w.last) * a.V : nullptr;
  const uint32_t* strikes = w.struck != 0 ? bits : nullptr;
  const int head = row_head(row);
  int chunk = 0;
  double before = 0.0, target = u * total;
  if (total > 0.0) {
    for (; chunk < a.chunks - 1; ++chunk) {
      const double upto = before + sums[chunk];
      if (upto > target) break;
      before = upto;
    }
  } else {  // nothing is left of p (it was rounded away): p itself, which sums up to 1
    drow = nullptr, strikes = nullptr, target = u;
    for (; chunk < a.chunks - 1; ++chunk) {
      const double upto = before + chunk_sum(a, w, row, drow, strikes, chunk * kChunkValues - head, sum4);
      if (upto > target) break;
      before = upto;
    }
    __syncthreads();
  }
  target -= before;
  const int first = chunk * kChunkValues - head;
  if (strikes != nullptr) strike(bits, a, b, w.struck, first);
  // A thread's values are neighbours here, so that the order of the sum is theirs.
  double v[kPieces][P];
  double mine = 0.0;
  int last_positive = -1;
  const int e0 = first + tid * kPerThread;
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    weights<E>(a, w, row, drow, strikes, first, e0 + k * P, v[k]);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      mine += v[k][i];
      if (v[k][i] > 0.0) last_positive = e0 + k * P + i;
    }
  }
  double upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double s = __shfl_up(upto, o);
    if (lane >= o) upto += s;
  }
  if (lane == 63) sum4[wave] = upto;
  __syncthreads();
  for (int i = 0; i < wave; ++i) upto += sum4[i];
  const uint64_t hit = __ballot(upto > target);
  const uint64_t some = __ballot(last_positive >= 0);
  const int top = __shfl(last_positive, some == 0 ? 0 : 63 - __clzll((long long)some));
  if (lane == 0) {
    found4[wave] = hit == 0 ? INT_MAX : wave * 64 + __ffsll((long long)hit) - 1;
    last4[wave] = top;
  }
  __syncthreads();
  const int owner = min(min(found4[0], found4[1]), min(found4[2], found4[3]));
  if (owner == INT_MAX) {  // the two sums' roundings differ: the last one with any weight
    if (tid == 0) a.next[b] = max(max(last4[0], last4[1]), max(last4[2], last4[3]));
    return;
  }
  if (tid != owner) return;
  double c = upto - mine;
  int at = last_positive;
  bool open = true;
#pragma unroll
  for (int k = 0; k < kPieces; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) {
      c += v[k][i];
      if (open && v[k][i] > 0.0 && c > target) at = e0 + k * P + i, open = false;
    }
  a.next[b] = at;
}

template <typename E>
__global__ __launch_bounds__(64) void draft_greedy_kernel(DraftArgs a) {
  const int b = blockIdx.x;
  const Walk w = walk_nodes<E, true>(a, b, true);
  if (threadIdx.x == 0) a.next[b] = w.last < 0 ? -1 : row_best(a, (int64_t)b * a.N + w.last);
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
  if (2 * (int64_t)d->B * d->N * chunks_of(d) >= (int64_t)1 << 24) return bad(who, "too many logits: at most 2^23 chunks of 8192", FC_ERR_UNSUPPORTED);
  return FC_OK;
}

struct Layout {
  size_t stats, walks, sums, total;
};
Layout layout_of(const fc_verify_desc* d) {
  Layout l;
  const int chunks = chunks_of(d);
  l.stats = 0;
  l.walks = round256((size_t)rows_of(d) * chunks * sizeof(ChunkStat));
  l.sums = l.walks + round256((size_t)d->B * sizeof(Walk));
  l.total = l.sums + round256((size_t)d->B * chunks * sizeof(double));
  return l;
}

template <typename E>
hipError_t launch_verify(const DraftArgs& a, int64_t rows, bool greedy, hipStream_t s) {
  ProfileMark mk = profile_begin(s);
  const dim3 all((unsigned)(rows * a.chunks));
  if (greedy) hipLaunchKernelGGL((draft_stats_kernel<E, true>), all, dim3(kDraftThreads), 0, s, a);
  else hipLaunchKernelGGL((draft_stats_kernel<E, false>), all, dim3(kDraftThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  profile_end(mk, "draft_stats", s);
  if (e != hipSuccess) return e;
  mk = profile_begin(s);
  if (greedy) hipLaunchKernelGGL((draft_greedy_kernel<E>), dim3((unsigned)a.B), dim3(64), 0, s, a);
  else hipLaunchKernelGGL((draft_walk_kernel<E>), dim3((unsigned)(a.B * a.chunks)), dim3(kDraftThreads), 0, s, a);
  e = hipGetLastError();
  profile_end(mk, "draft_walk", s);
  if (e != hipSuccess || greedy) return e;
  mk = profile_begin(s);
  hipLaunchKernelGGL((draft_pick_kernel<E>), dim3((unsigned)a.B), dim3(kDraftThreads), 0, s, a);
  e = hipGetLastError();
  profile_end(mk, "draft_pick", s);
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
  if (workspace == nullptr || workspace_bytes < l.total) return fc::bad(who, "the workspace is missing or too small", FC_ERR_WORKSPACE);
  if (fc::off(workspace, 256)) return fc::bad(who, "the workspace must be 256-byte aligned", FC_ERR_WORKSPACE);
  fc::DraftArgs a{};
  a.logits = logits, a.draft = draft ? draft_logits : nullptr, a.tokens = tokens, a.u = u;
  a.parents = parents, a.counts = counts, a.path = path, a.kept = kept, a.next = next;
  char* ws = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<fc::ChunkStat*>(ws + l.stats);
  a.walks = reinterpret_cast<fc::Walk*>(ws + l.walks);
  a.sums = reinterpret_cast<double*>(ws + l.sums);
  a.B = desc->B, a.N = desc->N, a.V = desc->V, a.chunks = fc::chunks_of(desc);
  a.index64 = desc->index_type == FC_INDEX_I64, a.tree = desc->tree;
  a.to_log2 = greedy ? 0.0 : 1.4426950408889634074 / desc->temperature;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t rows = (int64_t)a.B * a.N + (draft ? (int64_t)a.B * (a.N - 1) : 0);
  const hipError_t e = desc->dtype == FC_BF16 ? fc::launch_verify<fc::bf16>(a, rows, greedy, s) : fc::launch_verify<float>(a, rows, greedy, s);
  if (e != hipSuccess) return fc::bad(who, hipGetErrorString(e), FC_ERR_HIP);
  fc::clear_error();
  return FC_OK;
}

}  // extern "C"
