// Attention of a few new tokens over a cache (gfx950): the kernel.
//
// For the rows of a KV head (its G query heads times N new tokens) and a run of
// its keys,
//   S = K Q^T,  P = exp2(S - m),  O^T += V^T P^T,
// in 16x16x32 MFMA on bf16 operands with float32 accumulation; codes of 8 bits
// are exact in bf16, a key's scale multiplies its scores and a value's scale its
// probabilities, in float32.  P enters the second product as two bf16 values, its
// rounding and the rest: rounded once, it would add as much to O's error as O's own
// rounding does (2.3e-3 of O for 1.7e-3, in the 2-norm).
//
// The work is the reading of the cache, once per KV head, so what a wave needs is
// loads in flight and few instructions per byte:
//  * K's rows are the first product's A operand as they lie: lane (n, g) = (l % 16,
//    l / 16) reads units g ceil(U / 4) + s of row n (8 values each, U = D / 8), and Q's
//    operand holds the same units, as the order of a sum is free.
//  * S^T comes with a query in lane n and keys 4 g + r: that is the second
//    product's B operand where its k order is (block, g, r), so P goes from one
//    product to the next in its registers.
//  * The A operand of the second product holds V's columns, k in that order: lane
//    (n, g) reads C = D / 16 neighbouring values of its eight keys, and its c-th
//    column makes the c-th product's operand (a byte or halfword shuffle of its
//    own registers), whose row n is then column C n + c of O.
//  * Row maxima are not kept from tile to tile: a row's reference moves only
//    where a score exceeds it by 2^8, which a wave asks of its lanes with one vote.
// Each wave reads keys of its own for sixteen or 32 rows, with neither LDS (but for the queries)
// nor barriers in the loop: its operands are used twice at most, and eight waves that shared
// them through LDS in steps of 128 keys waited for each other longer than for the bytes
// (16 sequences of up to 8192 int8 keys, 64 rows, 8 KV heads: 75 us for 61).
//
// The lengths lie on the device, so the launch is the same whatever they are: as many
// workgroups as the GPU holds at once, each of which finds its equal share of all
// sequences' tiles (cache_index.hpp).  A sequence in several shares is joined by a
// second, small kernel.
//
// Measured, codes of 8 bits, heads of 128, a captured call with its join: 64 sequences of up to
// 4096 keys, 5 KV heads, one token each, 45 us (192 MB; the kernel 41, 4.7 TB/s, and a copy reaches
// 5.1); one of 131072 keys, 8 KV heads, 56 us (277 MB; part of it stays in the 256 MB cache between
// calls); 16 of up to 8192 keys, 8 KV heads, 32 nodes of two heads each, 62 us (168 MB, 2.7 TB/s): the two
// waves of a SIMD have an instruction under way for 94% of the time, two thirds of it vector ones, of
// which 190 of 450 a tile turn codes into numbers and 90 make two numbers of each probability.
//
// Rows that do not see a key have P = 0 there, but 0 * infinity is not 0, nor has a P of two numbers one
// sign.  Values that no row sees are taken as zeros.  Where a wave's sums of bf16 values turn out not to be
// finite, it goes through its keys again, with values that are not as zeros, and puts those where they are
// seen at the end.  A NaN of float8 (a caller's own codes) is one to all rows that see it; in tiles that
// some row sees only in part it is taken out and put in likewise, without a second pass.
#pragma once

#include "attn_fast.hpp"
#include "attn_score.hpp"
#include "cache_types.hpp"

namespace fc {

struct CachedAttnArgs {
  CacheGeom g;
  const void *k, *v;
  const float *k_scale, *v_scale;
  const int32_t* table;
  const void* Q;
  void* O;
  const int32_t *lengths, *counts, *parents;
  const float* slopes;
  float* part_o;   // [KV head, row group][2 shares][16 R][D]
  float2* part_s;  // [KV head, row group][2 shares][16 R] (reference, sum)
  int4* parts;     // of a sequence: how many, the first's slot, the second's, its tokens
  int H, N, G, rows;      // rows = G N
  int left;               // INT_MAX / 2: all
  int tree;               // 0 a run, 1 one tree, 2 a tree per sequence
  int groups;             // row groups of 16 R
  int shares;             // workgroups per KV head and row group, each with a share of all tiles; 0: one per sequence
  int least;              // tiles of a share, at least
  float scale_log2, cap_in, cap_out;
};

// ---- which keys a workgroup takes ---------------------------------------------

// The lengths and counts of 64 sequences, one to each lane.
struct Chunk {
  int b0, length, count;
  __device__ inline void load(const CachedAttnArgs& a, int from) {
    b0 = from;
    const int b = from + (int)(threadIdx.x & 63);
    length = b < a.g.B ? a.lengths[b] : 0;
    count = b < a.g.B ? (a.counts != nullptr ? a.counts[b] : a.N) : 0;
  }
  __device__ inline Span mine(const CachedAttnArgs& a) const { return span_of(length, count, a.N, a.left, a.g.capacity); }
  // Of sequence b, which may lie behind the chunk.
  __device__ inline Span of(const CachedAttnArgs& a, int b) {
    if (b - b0 >= 64) load(a, b);
    return span_of(__builtin_amdgcn_readlane(length, b - b0), __builtin_amdgcn_readlane(count, b - b0), a.N, a.left, a.g.capacity);
  }
};

// A place on the line of all sequences' work (cache_index.hpp).
struct Line {
  int64_t share;  // its stretches' length
  int64_t start;  // where a sequence begins
  int b;          // which, B past the end
  Chunk chunk;    // from or around it
};
// The sum of a wave's values up to each lane, in the vector unit (shuffles through LDS take 130 cycles each).
__device__ inline int sum_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, of each sixteen lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15, to the second and fourth
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31, to the last two
  return v;
}
// The first sequence of share x.  Every lane of a wave calls it and gets the same.
__device__ inline Line find_on_line(const CachedAttnArgs& a, int x) {
  const int lane = threadIdx.x & 63;
  const auto length = [&](const Chunk& c) { return c.b0 + lane < a.g.B ? line_length(c.mine(a).tiles) : 0; };
  Line l;
  l.chunk.load(a, 0);
  int n = length(l.chunk), upto = sum_upto(n);  // with the sequences up to this lane's
  int64_t total = __builtin_amdgcn_readlane(upto, 63);
  for (int b0 = 64; b0 < a.g.B; b0 += 64) {
    Chunk c;
    c.load(a, b0);
    total += __builtin_amdgcn_readlane(sum_upto(length(c)), 63);
  }
  l.share = share_of(total, a.shares, a.least);
  l.b = a.g.B;
  l.start = total;
  const int64_t at = x * l.share;
  int64_t before = 0;
  for (int b0 = 0; b0 < a.g.B; b0 += 64) {
    if (b0 > 0) {
      l.chunk.load(a, b0);
      n = length(l.chunk);
      upto = sum_upto(n);
    }
    const uint64_t hit = __ballot(n > 0 && at < before + upto);
    if (hit != 0) {
      const int i = __ffsll((long long)hit) - 1;
      l.b = b0 + i;
      l.start = before + __builtin_amdgcn_readlane(upto - n, i);
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return l;
}

// ---- the nodes --------------------------------------------------------------------

// What a node sees of the nodes, and where it lies in the text.
struct Nodes {
  uint64_t sees[kMaxNodes];  // itself and its ancestors within the window
  int depth[kMaxNodes];      // ancestors; -1 where its parents are not a tree's
};
// Called by one whole wave; lane i, which holds node i's parent, walks from it to the root.
__device__ inline void trace_nodes(Nodes* to, bool tree, int up, int N, int left) {
  const int i = threadIdx.x & 63;
  uint64_t sees = i < N ? 1ull << i : 0;
  int depth = 0, at = i;
  bool good = true;
  if (!tree) {
    depth = i;
    sees = left >= i ? (2ull << i) - 1 : ((2ull << left) - 1) << (i - left);  // (left < i < 64)
  } else {
    while (true) {
      const int next = __shfl(up, at);  // every lane's `at` is below 64
      const bool ok = next >= -1 && next < at;
      const bool go = good && i < N && ok && next >= 0;
      if (i < N && !ok) good = false;
      if (go) {
        at = next;
        ++depth;
        if (depth <= left) sees |= 1ull << at;
      }
      if (__ballot(go) == 0) break;
    }
  }
  if (i < N) {
    to->sees[i] = sees;
    to->depth[i] = good ? depth : -1;
  }
}

// ---- the cache's bytes as operands ------------------------------------------------

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ inline uint32_t pair(float lo, float hi) {
  bf16x2 v;
  v[0] = static_cast<bf16>(lo);
  v[1] = static_cast<bf16>(hi);
  return __builtin_bit_cast(uint32_t, v);
}
// Codes 2 i and 2 i + 1 of a word (exact in bf16).
template <int kType, bool kHigh>
__device__ inline uint32_t code_pair(uint32_t w) {
  if constexpr (kType == FC_CACHE_F8) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHigh));
  } else {
    return kHigh ? pair((float)(int8_t)((w >> 16) & 0xff), (float)(int8_t)(w >> 24))
                 : pair((float)(int8_t)(w & 0xff), (float)(int8_t)((w >> 8) & 0xff));
  }
}
__device__ inline uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ inline uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// kBytes of a row, in words.  They come through buffer descriptors: one without records
// reads as zeros with no branch and no traffic, so a loop's last requests need no
// condition (behind one the compiler would wait for them as if they had been made).
template <int kBytes>
struct Raw {
  uint32_t w[kBytes < 4 ? 1 : kBytes / 4];
  __device__ inline void load(__amdgpu_buffer_rsrc_t r, int offset) {
    if constexpr (kBytes == 1) w[0] = __builtin_amdgcn_raw_buffer_load_b8(r, offset, 0, 0);
    if constexpr (kBytes == 2) w[0] = __builtin_amdgcn_raw_buffer_load_b16(r, offset, 0, 0);
    if constexpr (kBytes == 4) w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, offset, 0, 0);
    if constexpr (kBytes == 8) {
      const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, offset, 0, 0);
      w[0] = v[0], w[1] = v[1];
    }
    if constexpr (kBytes == 16) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0);
      w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
    }
  }
};

template <int kType, int kD>
struct CachedCfg {
  static constexpr int kEsz = kType == FC_CACHE_BF16 ? 2 : 1;
  static constexpr int kU = kD / 8;               // 8-value units of a row
  static constexpr int kSteps = (kU + 3) / 4;     // products of 32 values
  static constexpr int kC = kD <= 16 ? 1 : kD <= 32 ? 2 : kD <= 64 ? 4 : 8;  // columns of V per lane
  static constexpr int kLanes = kD / kC;          // lanes that have columns, of 16
  static constexpr int kRow = kD * kEsz;          // bytes
};

// A row's reference before its first key: no score but -infinity is below it.
constexpr float kNoReference = -0x1.fffffep127f;

// Sums under another reference: by may be 0, which leaves an infinity what it is.
__device__ inline f32x4 scaled(f32x4 v, float by) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_isinf(v[i]) ? v[i] : v[i] * by;
  return r;
}

// What a call needs beside the sequence, the same for every row.
struct CallScores {
  float factor;  // of a product before its key's scale: log2(e) / sqrt(D), or what the cap takes
  float cap_in, cap_out;
  bool slopes;
};

// Reductions over the sixteen lanes of a row of the wave (n), left in all of them.
template <typename Op>
__device__ inline uint32_t reduce16(uint32_t v, Op op) {
  const auto step = [&](auto ctrl) {
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(ctrl)::value, 0xf, 0xf, false));
  };
  step(std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
  step(std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
  step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  step(std::integral_constant<int, 0x140>{});  // row_mirror
  return v;
}

// The rows' queries as operands, for all of a workgroup's waves.
template <int kType, int kD, int kR>
struct Queries {
  using C = CachedCfg<kType, kD>;
  bf16x8 unit[kR][C::kSteps][64];

  // All of kW waves, sixteen threads to a row and kEach rows each: load, then store, which waits for the
  // values.  Returns which there are; the others, of which any may be read, are stored as zeros.
  template <int kW>
  static constexpr int kEach = (16 * kR + 4 * kW - 1) / (4 * kW);
  template <int kW>
  __device__ static inline uint32_t load(bf16x8 (&to)[kEach<kW>], const CachedAttnArgs& a, int b, int h, int first_row, int count) {
    uint32_t there = 0;
#pragma unroll
    for (int i = 0; i < kEach<kW>; ++i) {
      const int of = 4 * kW * i + (int)(threadIdx.x >> 4), row = first_row + of, node = row / a.G, u = threadIdx.x & 15;
      const bool mine = of < 16 * kR && node < count && u < C::kU;
      const bf16* src = static_cast<const bf16*>(a.Q);
      src += mine ? (((int64_t)b * a.N + node) * a.H + h * a.G + row - node * a.G) * kD + 8 * u : 0;
      to[i] = *reinterpret_cast<const bf16x8*>(src);
      there |= mine ? 1u << i : 0;
    }
    return there;
  }
  template <int kW>
  __device__ inline void store(const bf16x8 (&from)[kEach<kW>], uint32_t there) {
    const int u = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < kEach<kW>; ++i) {
      const int of = 4 * kW * i + (int)(threadIdx.x >> 4);
      if (of < 16 * kR && u < 4 * C::kSteps)
        unit[of / 16][u % C::kSteps][of % 16 + 16 * (u / C::kSteps)] = (there >> i & 1) != 0 ? from[i] : Mma<bf16>::zero();
    }
  }
};

// kR blocks of sixteen rows of a KV head, one to each lane n: what they see, their queries
// and their sums.
template <int kType, int kD, int kR>
struct Rows {
  using C = CachedCfg<kType, kD>;
  static constexpr bool k8 = kType != FC_CACHE_BF16;
  uint64_t sees[kR], any_sees;  // nodes that the row, and that any of them all sees
  int low[kR], any_low;         // first key of the sequence, likewise (INT_MAX: none)
  int all_low;                  // behind which every row sees every key of the sequence
  int at[kR];                   // the row's position in the text
  float slope2[kR];
  bool broken[kR];              // NaN
  f32x4 acc[kR][C::kC];         // column C (4 g + r) + c of lane n's row
  float ref[kR], sum[kR];
  uint32_t odd;                 // not 0: a NaN code was taken out

  __device__ inline void begin(const CachedAttnArgs& a, const Nodes& nodes, int b, int h, int first_row, int length, int count) {
    const int n = threadIdx.x & 15;
    any_sees = 0;
    any_low = INT_MAX;
    all_low = 0;
    odd = 0;
#pragma unroll
    for (int rb = 0; rb < kR; ++rb) {
      const int row = first_row + 16 * rb + n, node = row / a.G, head = h * a.G + row - node * a.G;
      const bool there = row < a.rows && node < count;
      const int depth = there ? nodes.depth[node] : 0;
      broken[rb] = there && (depth < 0 || node >= a.g.capacity - length);
      sees[rb] = there && !broken[rb] ? nodes.sees[node] : 0;
      at[rb] = length + depth;
      low[rb] = there && !broken[rb] ? max(at[rb] - a.left, 0) : INT_MAX;
      slope2[rb] = a.slopes != nullptr && there ? base2_slope(a.slopes[head]) : 0.0f;
      any_sees |= sees[rb];
      any_low = min(any_low, low[rb]);
      all_low = max(all_low, there && !broken[rb] ? low[rb] : 0);  // (rows that are not there, or broken, may take whatever comes)
      ref[rb] = kNoReference;
      sum[rb] = 0.0f;
#pragma unroll
      for (int c = 0; c < C::kC; ++c) acc[rb][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const auto either = [](uint32_t x, uint32_t y) { return x | y; };
    any_sees = (uint64_t)reduce16((uint32_t)(any_sees >> 32), either) << 32 | reduce16((uint32_t)any_sees, either);
    any_low = __builtin_amdgcn_readfirstlane((int)reduce16((uint32_t)any_low, [](uint32_t x, uint32_t y) { return min(x, y); }));
    all_low = __builtin_amdgcn_readfirstlane((int)reduce16((uint32_t)all_low, [](uint32_t x, uint32_t y) { return max(x, y); }));
  }

  // Whether all the wave's sums are finite.
  __device__ inline bool all_finite() const {
    float zero = 0.0f;
#pragma unroll
    for (int rb = 0; rb < kR; ++rb)
#pragma unroll
      for (int c = 0; c < C::kC; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) zero = __builtin_fmaf(acc[rb][c][r], 0.0f, zero);
    return __ballot(zero != zero) == 0;
  }

  // Which of a lane's eight keys are set in a mask of 32 from key 4 g on, as halves of
  // the operands' words: keys 2 i and 2 i + 1.
  __device__ static inline u32x4 halves(uint32_t keys) {
    u32x4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bit = 16 * (i >> 1) + 2 * (i & 1);
      m[i] = ((keys >> bit & 1) != 0 ? 0xffffu : 0u) | ((keys >> bit & 2) != 0 ? 0xffff0000u : 0u);
    }
    return m;
  }

  // Keys key0 .. key0 + 31.  Of `keys`: frag(kb, step), scale(kb) of keys 4 g + r, used() once
  // both are; of `values`: frag(c), scale(kb), and for keys of which some row may be blind
  // keep(mask: which of the 32 keys from 4 g on any row sees) and finite() (values that are not
  // become zeros; whether any was).  finite: of bf16 in all tiles.
  template <typename Keys, typename Values>
  __device__ inline void tile(const CallScores& call, bool finite, const Queries<kType, kD, kR>& queries, const Nodes& nodes, int N, int key0, int length, Keys& keys, Values& values) {
    const int g = (threadIdx.x & 63) >> 4;
    // Every row sees every key of a tile before the nodes and behind all rows' first keys.
    const bool masked = finite || key0 < all_low || key0 + kTileKeys > length;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // (the queries would be kept in registers from tile to tile)
    f32x4 s[kR][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) s[rb][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int st = 0; st < C::kSteps; ++st) {
        const bf16x8 f = keys.frag(kb, st);
#pragma unroll
        for (int rb = 0; rb < kR; ++rb) s[rb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, queries.unit[rb][st][lane], s[rb][kb], 0, 0, 0);
      }
    }
    // Scores in base 2.
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const f32x4 f = keys.scale(kb, call.factor);
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) s[rb][kb] *= f;
    }
    keys.used();
    if (call.cap_in > 0.0f) {
#pragma unroll
      for (int rb = 0; rb < kR; ++rb)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[rb][kb][r] = __builtin_fmaf(-2.0f * call.cap_out, cap_part(s[rb][kb][r], 1.0f), call.cap_out);
    }
    int g4 = 4 * g;
    asm volatile("" : "+v"(g4));  // (what follows from it would be kept from tile to tile)
    if (call.slopes) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = key0 + 16 * kb + g4 + r;
          const int pos = masked && key >= length && key < length + N ? length + nodes.depth[key - length] : key;
#pragma unroll
          for (int rb = 0; rb < kR; ++rb) s[rb][kb][r] = __builtin_fmaf(-slope2[rb], (float)(at[rb] - pos), s[rb][kb][r]);
        }
    }
    if (masked) {
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) {
        const uint32_t seen = seen_keys(key0 + g4, low[rb], sees[rb], length);
#pragma unroll
        for (int j = 0; j < 8; ++j)  // P = 0, whatever the reference
          s[rb][j >> 2][j & 3] = (seen >> (16 * (j >> 2) + (j & 3)) & 1) != 0 ? s[rb][j >> 2][j & 3] : -INFINITY;
      }
    }
    // The reference moves where a score is 2^8 beyond it.
    float most[kR];
    bool grows = false;
#pragma unroll
    for (int rb = 0; rb < kR; ++rb) {
      float m = fmaxf(fmaxf(s[rb][0][0], s[rb][0][1]), s[rb][0][2]);
      m = fmaxf(fmaxf(m, s[rb][0][3]), s[rb][1][0]);
      m = fmaxf(fmaxf(m, s[rb][1][1]), s[rb][1][2]);
      most[rb] = fmaxf(m, s[rb][1][3]);
      grows |= most[rb] > ref[rb] + 8.0f;
    }
    if (__ballot(grows) != 0) {
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) {
        float m = fmaxf(most[rb], __shfl_xor(most[rb], 16));
        m = fmaxf(fmaxf(m, __shfl_xor(m, 32)), ref[rb]);
        const float by = __builtin_amdgcn_exp2f(ref[rb] - m);
        ref[rb] = m;
        sum[rb] *= by;
#pragma unroll
        for (int c = 0; c < C::kC; ++c) acc[rb][c] *= by;
      }
    }
    u32x4 ph[kR], pl[kR];
#pragma unroll
    for (int rb = 0; rb < kR; ++rb) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        f32x4 e;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = __builtin_amdgcn_exp2f(s[rb][kb][r] - ref[rb]);
          sum[rb] += e[r];
        }
        if (k8) e *= values.scale(kb);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t hi = pair(e[2 * i], e[2 * i + 1]);
          ph[rb][2 * kb + i] = hi;
          pl[rb][2 * kb + i] = pair(e[2 * i] - __builtin_bit_cast(float, hi << 16), e[2 * i + 1] - __builtin_bit_cast(float, hi & 0xffff0000u));
        }
      }
    }
    if (masked) {
      values.keep(seen_keys(key0 + g4, any_low, any_sees, length));
      if (kType == FC_CACHE_F8) odd |= values.finite();
      if (finite) values.finite();
      if (k8) {  // (an unseen key's scale may be NaN)
#pragma unroll
        for (int rb = 0; rb < kR; ++rb) {
          const u32x4 mine = halves(seen_keys(key0 + g4, low[rb], sees[rb], length));
          ph[rb] &= mine;
          pl[rb] &= mine;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < C::kC; ++c) {
      const bf16x8 f = values.frag(c);
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) acc[rb][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, ph[rb]), acc[rb][c], 0, 0, 0);
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) acc[rb][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, pl[rb]), acc[rb][c], 0, 0, 0);
    }
  }
};
// A word's values that are not finite, all bits of them: halves of bf16, NaN codes of float8.
template <int kType>
__device__ inline uint32_t odd_bits(uint32_t w) {
  if constexpr (kType == FC_CACHE_BF16)
    return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
  const uint32_t top = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // (a code's 7 bits and 1)
  return top | (top - (top >> 7));
}

// The K operand of 8 neighbouring values, and the V operands of eight keys' C columns.
template <int kType>
__device__ inline bf16x8 key_operand(const uint32_t* w) {
  if constexpr (kType == FC_CACHE_BF16) return as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
  else return as_bf16x8(make_uint4(code_pair<kType, false>(w[0]), code_pair<kType, true>(w[0]), code_pair<kType, false>(w[1]), code_pair<kType, true>(w[1])));
}
// Column c of two keys' columns.
template <int kType>
__device__ inline uint32_t two_keys(const uint32_t* x, const uint32_t* y, int c) {
  if constexpr (kType == FC_CACHE_I8) {  // (the rounding to bf16 pairs them)
    return pair((float)(int8_t)(x[c / 4] >> 8 * (c % 4) & 0xff), (float)(int8_t)(y[c / 4] >> 8 * (c % 4) & 0xff));
  } else {
    uint32_t u, v;
    if constexpr (kType == FC_CACHE_BF16) {
      u = x[c / 2], v = y[c / 2];
    } else if (c / 2 % 2 != 0) {
      u = code_pair<kType, true>(x[c / 4]), v = code_pair<kType, true>(y[c / 4]);
    } else {
      u = code_pair<kType, false>(x[c / 4]), v = code_pair<kType, false>(y[c / 4]);
    }
    return c % 2 != 0 ? high_halves(u, v) : low_halves(u, v);
  }
}

// Where a sequence's 16-key blocks lie.  Lane i holds the page of the wave's i-th block
// from here, 64 at a time: a look at the table for each tile would wait for everything
// the wave has on its way (64 x 4096 int8 keys in pages of 64: 64 us for 51).
struct Blocks {
  int page;
  // Blocks at key, key + step, ...
  __device__ inline void fetch(const CachedAttnArgs& a, int b, int key, int step, int end) {
    const int mine = key + step * (int)(threadIdx.x & 63);
    page = mine < end ? (int)cache_page(a.g, a.table, b, mine) : 0;
  }
  // The i-th block, which begins at key: its page's number (-1: none) and its first row.
  __device__ inline int64_t row(const CachedAttnArgs& a, int h, int i, int key, int* number) const {
    const int p = __builtin_amdgcn_readlane(page, i);
    *number = p;
    return ((int64_t)max(p, 0) * a.g.Hkv + h) * a.g.page_size + cache_place(a.g, a.table, key);
  }
};

// The kSteps operands' bytes of a K row, from offset on.
template <int kType, int kSteps>
__device__ inline void load_steps(Raw<kType == FC_CACHE_BF16 ? 16 : 8> (&k)[kSteps], __amdgpu_buffer_rsrc_t r, int offset) {
  if constexpr (kType != FC_CACHE_BF16 && kSteps % 2 == 0) {  // 16 bytes at a time
#pragma unroll
    for (int s = 0; s < kSteps; s += 2) {
      Raw<16> two;
      two.load(r, offset + 8 * s);
      k[s].w[0] = two.w[0], k[s].w[1] = two.w[1], k[s + 1].w[0] = two.w[2], k[s + 1].w[1] = two.w[3];
    }
  } else {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) k[s].load(r, offset + (kType == FC_CACHE_BF16 ? 16 : 8) * s);
  }
}

// A block's sixteen rows, as descriptors without records where it is not there.
template <int kType, int kD>
struct BlockBytes {
  using C = CachedCfg<kType, kD>;
  __amdgpu_buffer_rsrc_t k, v, ks, vs;
  __device__ inline void set(const CachedAttnArgs& a, int64_t row, bool there) {
    const uint32_t rows = there ? 16 : 0;
    k = make_rsrc(static_cast<const char*>(a.k) + row * C::kRow, rows * C::kRow);
    v = make_rsrc(static_cast<const char*>(a.v) + row * C::kRow, rows * C::kRow);
    if constexpr (kType != FC_CACHE_BF16) {
      ks = make_rsrc(a.k_scale + row, 4 * rows);
      vs = make_rsrc(a.v_scale + row, 4 * rows);
    }
  }
};
// Offsets in a block of lane (n, g)'s parts of K (step 0; a unit past the row reads the next
// one's, or zeros, and is left out of the operand) and V (row 4 g).
template <int kType, int kD>
struct LaneOffsets {
  using C = CachedCfg<kType, kD>;
  int k, v;
  __device__ inline LaneOffsets() {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    k = n * C::kRow + 8 * C::kEsz * g * C::kSteps;
    v = 4 * g * C::kRow + C::kC * C::kEsz * (C::kLanes == 16 ? n : min(n, C::kLanes - 1));
  }
};

// The stretches of a workgroup, sequence by sequence: body(b, length, count, first tile, last tile, whole, slot).
// Where `tells`, it leaves for each sequence that begins in it what the join asks.
template <typename Body>
__device__ inline void for_each_stretch(const CachedAttnArgs& a, int x, bool tells, Body body) {
  Line line{0, 0, x, {}};
  if (a.shares > 0)
    line = find_on_line(a, x);
  else
    line.chunk.load(a, x);
  bool again = false;
  for (int b = line.b; b < a.g.B; ++b) {
    const int64_t start = line.start;
    if (a.shares > 0 && start >= (x + 1) * line.share) break;
    const Span span = line.chunk.of(a, b);
    Stretch st{0, span.tiles};
    if (a.shares > 0) {
      line.start += line_length(span.tiles);
      st = stretch_of(start, span.tiles, x, line.share);
      if (st.first >= st.last) continue;
    }
    if (again) __syncthreads();  // the last sequence's LDS is read
    again = true;
    if (a.shares > 0 && st.first == 0 && tells && threadIdx.x == 0) {
      const int64_t last = line_quotient(start + span.tiles + kBegin - 1, line.share);
      a.parts[b] = make_int4((int)(last - x) + 1, (int)part_slot(start, x, line.share), (int)part_slot(start, x + 1, line.share), span.count);
    }
    body(b, span.length, span.count, span.first + st.first, span.first + st.last, st.first == 0 && st.last == span.tiles,
         part_slot(start, x, line.share));
    if (a.shares == 0) break;
  }
}

// Which KV head, row group and share a workgroup has.  Workgroups go to the XCDs in
// turn: the row groups of one share, which read the same keys, are 8 workgroups apart, on
// one XCD and running together.
struct Place {
  int h, group, x;
};
__device__ inline Place place_of(const CachedAttnArgs& a) {
  const int id = blockIdx.x, of8 = id / 8, rest = of8 / a.groups * 8 + id % 8, per_head = a.shares > 0 ? a.shares : a.g.B;
  Place p;
  p.group = of8 % a.groups;
  p.h = rest / per_head;
  p.x = rest - p.h * per_head;
  return p;
}

// The kinds of kC values that are not finite, two bits each: 1 +infinity, 2 -infinity, 3 NaN.
template <int kType, int kC>
__device__ inline uint32_t odd_values(const uint32_t* w) {
  uint32_t kinds = 0;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    if constexpr (kType == FC_CACHE_BF16) {
      const uint32_t v = w[c / 2] >> 16 * (c % 2) & 0xffffu;
      kinds |= (v == 0x7f80u ? 1u : v == 0xff80u ? 2u : (v & 0x7fffu) > 0x7f80u ? 3u : 0u) << 2 * c;
    } else {
      kinds |= (w[c / 4] >> 8 * (c % 4) & 0x7fu) == 0x7fu ? 3u << 2 * c : 0u;
    }
  }
  return kinds;
}
// What marks of the three kinds (bits 1, 2 and 3) add to a sum.
__device__ inline float marked_value(uint32_t marks) {
  return marks == 0 ? 0.0f : marks == 2 ? INFINITY : marks == 4 ? -INFINITY : NAN;
}

// A stretch's end: each of kW waves holds sums of the workgroup's rows over some of its keys.
template <int kType, int kD, int kR, int kW>
struct Exchange {
  using C = CachedCfg<kType, kD>;
  static constexpr int kPad = kD + 4;  // floats of a row: the lanes' stores spread over the banks
  float acc[kR][kW][16 * kPad];        // before that, marks of values that are not finite
  float2 stats[kR][kW][16];

  // A wave's own part; all of its lanes call them.
  __device__ inline void clear(int wave) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
#pragma unroll 1
    for (int rb = 0; rb < kR; ++rb)
#pragma unroll 1
      for (int i = lane; i < 16 * kPad; i += 64) acc[rb][wave][i] = 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // kinds: of the lane's columns of key key0 + 16 kb + 4 g + r.
  __device__ inline void mark(int wave, const Rows<kType, kD, kR>& rows, uint32_t kinds, int key0, int kb, int r, int length) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // (what follows from it would be kept in registers all the time)
    const int n = lane & 15, g = lane >> 4;
    if (n >= C::kLanes) kinds = 0;  // (another lane's columns)
    if (__builtin_expect(__ballot(kinds != 0) == 0, 1)) return;
#pragma unroll
    for (int rb = 0; rb < kR; ++rb)
#pragma unroll 1
      for (int row = 0; row < 16; ++row) {
        const uint64_t sees = (uint64_t)(uint32_t)__shfl((int)(rows.sees[rb] >> 32), row) << 32 | (uint32_t)__shfl((int)rows.sees[rb], row);
        const uint32_t seen = seen_keys(key0 + 4 * g, __shfl(rows.low[rb], row), sees, length);
        if ((seen >> (16 * kb + r) & 1) == 0) continue;
        uint32_t* marks = reinterpret_cast<uint32_t*>(acc[rb][wave]) + row * kPad + C::kC * n;
#pragma unroll 1
        for (uint32_t left = kinds; left != 0;) {
          const int c = (__ffs(left) - 1) / 2;
          atomicOr(&marks[c], 1u << (left >> 2 * c & 3));
          left &= ~(3u << 2 * c);
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
};
template <int kType, int kD, int kR, int kW>
__device__ inline void finish(const CachedAttnArgs& a, const Rows<kType, kD, kR>& rows, Exchange<kType, kD, kR, kW>& x, bool marked, int b, int h,
                              int group, int count, bool whole, int64_t slot) {
  using C = CachedCfg<kType, kD>;
  constexpr int kPad = Exchange<kType, kD, kR, kW>::kPad, kRows = 16 * kR;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int rb = 0; rb < kR; ++rb) {
    float l = rows.sum[rb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) x.stats[rb][wave][n] = make_float2(rows.ref[rb], rows.broken[rb] ? NAN : l);
    float* to = x.acc[rb][wave] + n * kPad;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = C::kC * (4 * g + r);
      if (C::kLanes != 16 && d >= kD) continue;
#pragma unroll
      for (int c = 0; c < C::kC; ++c)
        to[d + c] = marked ? rows.acc[rb][c][r] + marked_value(__float_as_uint(to[d + c])) : rows.acc[rb][c][r];
    }
  }
  __syncthreads();
  // Sixteen threads to a row, four columns each at a time.
  const int64_t out = (((int64_t)h * a.groups + group) * 2 * a.shares + slot) * kRows;
#pragma unroll
  for (int i = 0; i < (kRows + 4 * kW - 1) / (4 * kW); ++i) {
    const int of = 4 * kW * i + (tid >> 4), rb = of / 16, of16 = of % 16;
    const int row = group * kRows + of, node = row / a.G, head = h * a.G + row - node * a.G;
    if (of >= kRows || row >= a.rows) break;
    float by[kW], m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kW; ++w) m = fmaxf(m, x.stats[rb][w][of16].x);
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float2 st = x.stats[rb][w][of16];
      by[w] = __builtin_amdgcn_exp2f(st.x - m);
      sum += st.y * by[w];
    }
    if (!whole && (tid & 15) == 0) a.part_s[out + of] = make_float2(m, sum);
    const float inv = 1.0f / sum;
    bf16* O = static_cast<bf16*>(a.O) + (((int64_t)b * a.N + node) * a.H + head) * kD;
#pragma unroll
    for (int of64 = 0; of64 < (kD + 63) / 64; ++of64) {
      const int d = 64 * of64 + 4 * (tid & 15);
      if (kD % 64 != 0 && d >= kD) break;
      f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        const f32x4 of_wave = *reinterpret_cast<const f32x4*>(x.acc[rb][w] + of16 * kPad + d);
        v += kType == FC_CACHE_BF16 ? scaled(of_wave, by[w]) : of_wave * by[w];
      }
      if (whole) {
        v = node < count ? v * inv : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        *reinterpret_cast<uint2*>(O + d) = make_uint2(pair(v[0], v[1]), pair(v[2], v[3]));
      } else {
        *reinterpret_cast<f32x4*>(a.part_o + (out + of) * kD + d) = v;
      }
    }
  }
}

__device__ inline CallScores scores_of(const CachedAttnArgs& a) {
  return CallScores{a.cap_in > 0.0f ? a.cap_in : a.scale_log2, a.cap_in, a.cap_out, a.slopes != nullptr};
}
__device__ inline const int32_t* parents_of(const CachedAttnArgs& a, int b) {
  return a.parents == nullptr ? nullptr : a.parents + (a.tree == 2 ? (int64_t)b * a.N : 0);
}

// kW waves take every kW-th tile of 32 keys, each straight from memory through its
// registers, for the 16 kR rows of their workgroup: four, or eight where a workgroup has a CU to
// itself.
template <int kType, int kD, int kR, int kW>
__global__ __launch_bounds__(64 * kW, 2) void cached_attn_kernel(CachedAttnArgs a) {
  using C = CachedCfg<kType, kD>;
  constexpr bool k8 = kType != FC_CACHE_BF16;
  __shared__ Nodes nodes;
  __shared__ __attribute__((aligned(16))) Queries<kType, kD, kR> queries;
  __shared__ __attribute__((aligned(16))) Exchange<kType, kD, kR, kW> exchange;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = (threadIdx.x & 63) >> 4;
  const Place at = place_of(a);
  if (at.h >= a.g.Hkv) return;
  const CallScores call = scores_of(a);
  for_each_stretch(a, at.x, at.h == 0 && at.group == 0, [&](int b, int length, int count, int tile0, int tile1, bool whole, int64_t slot) {
    const int end = min(length + count, a.g.capacity), first_row = at.group * 16 * kR;
    if (count == 0) tile1 = tile0;  // (nothing to read)
    Raw<8 * C::kEsz> k[2][C::kSteps];
    Raw<C::kC * C::kEsz> v[8];
    Raw<16> ks[2], vs[2];
    Blocks blocks[2];
    BlockBytes<kType, kD> bytes[2];  // of the tile whose bytes are in k and v or on their way
    int page[2];
    const LaneOffsets<kType, kD> off;
    const auto locate = [&](int i, int key, bool there) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int64_t row = blocks[kb].row(a, at.h, i, key + 16 * kb, &page[kb]);
        bytes[kb].set(a, row, there && key + 16 * kb < end);
      }
    };
    const auto load_k = [&] {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        load_steps<kType>(k[kb], bytes[kb].k, off.k);
        if (k8) ks[kb].load(bytes[kb].ks, 16 * g);
      }
    };
    const auto load_v = [&] {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[4 * kb + r].load(bytes[kb].v, off.v + r * C::kRow);
        if (k8) vs[kb].load(bytes[kb].vs, 16 * g);
      }
    };
    const auto request_k = [&](int i, int key, bool there) {
      locate(i, key, there);
      load_k();
    };
    // What a stretch begins with is requested before any of it is waited for.
    const auto fetch = [&](int key) {
      blocks[0].fetch(a, b, key, kW * kTileKeys, end);
      blocks[1].fetch(a, b, key + 16, kW * kTileKeys, end);
    };
    int tile = tile0 + wave, i = 0;
    fetch(tile * kTileKeys);
    bf16x8 q[Queries<kType, kD, kR>::template kEach<kW>];
    const uint32_t asked = queries.template load<kW>(q, a, b, at.h, first_row, count);
    const int32_t* parents = parents_of(a, b);
    const int up = parents != nullptr && (int)threadIdx.x < a.N ? parents[threadIdx.x] : -1;
    locate(0, tile * kTileKeys, tile < tile1);
    load_k();
    load_v();
    queries.template store<kW>(q, asked);
    if (wave == 0) trace_nodes(&nodes, parents != nullptr, up, a.N, a.left);
    __syncthreads();
    Rows<kType, kD, kR> rows;
    rows.begin(a, nodes, b, at.h, first_row, length, count);
    // Marks what is not finite where it is seen.
    const auto mark = [&] {
      exchange.clear(wave);
      i = 0;
      for (tile = tile0 + wave; tile < tile1; tile += kW) {
        const int key0 = tile * kTileKeys;
        if (i == 0) fetch(key0);
        locate(i, key0, true);
        i = (i + 1) & 63;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll 1
          for (int r = 0; r < 4; ++r) {
            Raw<C::kC * C::kEsz> value;
            value.load(bytes[kb].v, off.v + r * C::kRow);
            exchange.mark(wave, rows, odd_values<kType, C::kC>(value.w), key0, kb, r, length);
          }
      }
    };
    bool again = false;  // (values that are not finite are zeros)
    while (true) {
      for (; tile < tile1; tile += kW) {
        const int key0 = tile * kTileKeys, next = key0 + kW * kTileKeys;
        if (kR == 2 && kW == 4) {
          // Of a CU's two workgroups the one that is behind goes first; the older one would be done at two
          // thirds of the time and leave half the CU idle (16 sequences, 32 nodes: 61 us for 58).
          const int left = 4 * (tile1 - tile), all = tile1 - tile0;
          if (left > 3 * all) __builtin_amdgcn_s_setprio(3);
          else if (left > 2 * all) __builtin_amdgcn_s_setprio(2);
          else if (left > all) __builtin_amdgcn_s_setprio(1);
          else __builtin_amdgcn_s_setprio(0);
        }
        i = (i + 1) & 63;
        if (i == 0) fetch(next);
        // (each operand's next bytes are requested as soon as these have left their registers)
        struct {
          decltype(k)& bytes;
          decltype(ks)& scales;
          const int (&page)[2];
          const int g;
          decltype(request_k)& request;
          const int i, next;
          const bool more;
          __device__ inline bf16x8 frag(int kb, int st) const {
            const bf16x8 f = key_operand<kType>(bytes[kb][st].w);
            return 4 * C::kSteps != C::kU && g * C::kSteps + st >= C::kU ? Mma<bf16>::zero() : f;
          }
          __device__ inline f32x4 scale(int kb, float by) const {
            const float f = page[kb] >= 0 ? by : NAN;  // a page that is none
            return k8 ? __builtin_bit_cast(f32x4, scales[kb]) * f : f32x4{f, f, f, f};
          }
          __device__ inline void used() const { request(i, next, more); }
        } keys{k, ks, page, g, request_k, i, next, tile + kW < tile1};
        struct {
          decltype(v)& bytes;
          decltype(vs)& scales;
          __device__ inline bf16x8 frag(int c) const {
            return as_bf16x8(make_uint4(two_keys<kType>(bytes[0].w, bytes[1].w, c), two_keys<kType>(bytes[2].w, bytes[3].w, c),
                                        two_keys<kType>(bytes[4].w, bytes[5].w, c), two_keys<kType>(bytes[6].w, bytes[7].w, c)));
          }
          __device__ inline f32x4 scale(int kb) const { return __builtin_bit_cast(f32x4, scales[kb]); }
          __device__ inline void keep(uint32_t mask) const {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
              for (uint32_t& w : bytes[j].w) w = (mask >> (16 * (j >> 2) + (j & 3)) & 1) != 0 ? w : 0;
          }
          __device__ inline uint32_t finite() const {
            uint32_t any = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
              for (uint32_t& w : bytes[j].w) {
                const uint32_t odd = odd_bits<kType>(w);
                w &= ~odd;
                any |= odd;
              }
            return any;
          }
        } values{v, vs};
        rows.tile(call, kType == FC_CACHE_BF16 && again, queries, nodes, a.N, key0, length, keys, values);
        load_v();
      }
      if (__builtin_expect(kType != FC_CACHE_BF16 || again || rows.all_finite(), 1)) break;
      again = true;
      mark();
      rows.begin(a, nodes, b, at.h, first_row, length, count);
      tile = tile0 + wave, i = 0;
      fetch(tile * kTileKeys);
      locate(0, tile * kTileKeys, tile < tile1);
      load_k();
      load_v();
    }
    bool marked = again;
    if (kType == FC_CACHE_F8 && __builtin_expect(__ballot(rows.odd != 0) != 0, 0)) {
      marked = true;
      mark();
    }
    finish<kType, kD, kR, kW>(a, rows, exchange, marked, b, at.h, at.group, count, whole, slot);
  });
}

// The parts of a row's sequence, where there are several: kWaves waves to a row, of a workgroup's
// four.  kInfinite: a part may be infinite (bf16).
template <int kD, int kWaves, bool kInfinite>
__global__ __launch_bounds__(256) void cached_attn_join_kernel(CachedAttnArgs a, int rows_per_group) {
  constexpr int kCols = kD / 4;         // threads of a part, four columns each
  constexpr int kAtOnce = 64 / kCols;   // parts of a wave at a time
  __shared__ f32x4 sums[4][kCols];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row_id = blockIdx.x * (4 / kWaves) + wave / kWaves;  // (b, node, head)
  if (kWaves == 1 && row_id >= a.g.B * a.N * a.H) return;
  const int head = row_id % a.H, bn = row_id / a.H, b = bn / a.N, node = bn - b * a.N;
  const int4 of_b = a.parts[b];
  const int parts = of_b.x;
  if (parts < 2) return;
  const int h = head / a.G, row = node * a.G + head - h * a.G, rg = row / rows_per_group, rr = row - rg * rows_per_group;
  const int64_t slots = ((int64_t)h * a.groups + rg) * 2 * a.shares;
  const auto place = [&](int i) { return (slots + (i == 0 ? of_b.y : of_b.z + 2 * (i - 1))) * rows_per_group + rr; };
  float2 st = lane < parts ? a.part_s[place(lane)] : make_float2(-INFINITY, 0.0f);
  float m = st.x, l = st.y;
  for (int i = lane + 64; i < parts; i += 64) {
    st = a.part_s[place(i)];
    const float most = fmaxf(m, st.x);
    l = l * __builtin_amdgcn_exp2f(m - most) + st.y * __builtin_amdgcn_exp2f(st.x - most);
    m = most;
  }
  float all = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
  l *= __builtin_amdgcn_exp2f(m - all);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  const int q = lane / kCols, d = 4 * (lane - q * kCols);
  f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (q < kAtOnce) {
#pragma unroll 4
    for (int i = wave % kWaves * kAtOnce + q; i < parts; i += kWaves * kAtOnce) {
      const int64_t at = place(i);
      const f32x4 part = *reinterpret_cast<const f32x4*>(a.part_o + at * kD + d);
      const float by = __builtin_amdgcn_exp2f(a.part_s[at].x - all);
      v += kInfinite ? scaled(part, by) : part * by;
    }
  }
  f32x4 of_wave = v;
#pragma unroll
  for (int i = 1; i < kAtOnce; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) of_wave[c] += __shfl(v[c], lane + i * kCols);
  if (kWaves > 1) {
    if (lane < kCols) sums[wave][lane] = of_wave;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) of_wave += sums[w][min(lane, kCols - 1)];
  }
  if (lane < kCols) {
    v = node < of_b.w ? of_wave * (1.0f / l) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    bf16* O = static_cast<bf16*>(a.O) + (int64_t)row_id * kD;
    *reinterpret_cast<uint2*>(O + d) = make_uint2(pair(v[0], v[1]), pair(v[2], v[3]));
  }
}

// What a variant of row blocks needs (cached_attn.hip instantiates them by type and head dim).
template <int kType> hipError_t launch_cached_attn(const CachedAttnArgs& a, int row_blocks, int waves, hipStream_t s);
hipError_t launch_cached_attn_join(const CachedAttnArgs& a, int rows_per_group, hipStream_t s);

}  // namespace fc
