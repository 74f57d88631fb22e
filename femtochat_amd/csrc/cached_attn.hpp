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
// loads in flight and few instructions per byte; there is no LDS and no barrier
// in the loop:
//  * A wave takes 32 keys at a time, the next ones' bytes on their way into
//    registers.  Waves, and workgroups, split a sequence's keys among them.
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
//
// Rows that do not see a key have P = 0 there, but 0 * infinity is not 0: in tiles
// that some row sees only in part, values that no row sees are taken as zeros,
// and those that are not finite are left out of the product and put where they are seen.
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
  float* part_o;   // [slot][16 R][D]
  float2* part_s;  // [slot][16 R] (reference, sum)
  int H, N, G, rows;      // rows = G N
  int left;               // INT_MAX / 2: all
  int tree;               // 0 a run, 1 one tree, 2 a tree per sequence
  int groups;             // row groups of 16 R
  int items, share;       // slots per row group, and how many of them share the tiles
  int least;              // tiles of a slot, at least
  float scale_log2, cap_in, cap_out;
};

// ---- which keys a workgroup takes ---------------------------------------------

__device__ inline int wave_sum(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ inline Span span_at(const CachedAttnArgs& a, int b) {
  return span_of(a.lengths[b], a.counts != nullptr ? a.counts[b] : a.N, a.N, a.left, a.g.capacity);
}

struct Slot {
  int b, part, parts, first;  // sequence (-1: none), which of its parts, its first slot
  int tiles;                  // of a part
};
// The sequence of slot x, or (x < 0) the slots of sequence of_b.  Every lane of a
// wave calls it and gets the same.
__device__ inline Slot find_slot(const CachedAttnArgs& a, int x, int of_b) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int b0 = 0; b0 < a.g.B; b0 += 64) total += wave_sum(b0 + lane < a.g.B ? span_at(a, b0 + lane).tiles : 0);
  Slot s;
  s.tiles = slot_tiles(total, a.share, a.least);
  s.b = -1, s.part = 0, s.parts = 0, s.first = 0;
  int before = 0;
  for (int b0 = 0; b0 < a.g.B; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < a.g.B ? (span_at(a, b).tiles + s.tiles - 1) / s.tiles : 0;
    int upto = n;  // slots of the sequences up to this lane's
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      if (lane >= o) upto += v;
    }
    const int mine = before + upto - n;
    const uint64_t hit = __ballot(x >= 0 ? (x >= mine && x < mine + n) : b == of_b);
    if (hit != 0) {
      const int at = __ffsll((long long)hit) - 1;
      s.b = b0 + at;
      s.parts = __shfl(n, at);
      s.first = __shfl(mine, at);
      s.part = x - s.first;
      break;
    }
    before += __shfl(upto, 63);
  }
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  s.part = __builtin_amdgcn_readfirstlane(s.part);
  s.parts = __builtin_amdgcn_readfirstlane(s.parts);
  s.first = __builtin_amdgcn_readfirstlane(s.first);
  s.tiles = __builtin_amdgcn_readfirstlane(s.tiles);
  return s;
}

// ---- the nodes --------------------------------------------------------------------

// What a node sees of the nodes, and where it lies in the text.
struct Nodes {
  uint64_t sees[kMaxNodes];  // itself and its ancestors within the window
  int depth[kMaxNodes];      // ancestors; -1 where its parents are not a tree's
};
// Called by one whole wave; lane i walks from node i to the root.
__device__ inline void trace_nodes(Nodes* to, const int32_t* parents, int N, int left) {
  const int i = threadIdx.x & 63;
  uint64_t sees = i < N ? 1ull << i : 0;
  int depth = 0, at = i;
  bool good = true;
  if (parents == nullptr) {
    depth = i;
    sees = left >= i ? (2ull << i) - 1 : ((2ull << left) - 1) << (i - left);  // (left < i < 64)
  } else {
    const int up = i < N ? parents[i] : -1;
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

template <int kBytes> struct Raw;  // kBytes of a row, in words
template <> struct Raw<1> {
  uint32_t w[1];
  __device__ inline void load(const uint8_t* p) { w[0] = *p; }
};
template <> struct Raw<2> {
  uint32_t w[1];
  __device__ inline void load(const uint8_t* p) { w[0] = *reinterpret_cast<const uint16_t*>(p); }
};
template <> struct Raw<4> {
  uint32_t w[1];
  __device__ inline void load(const uint8_t* p) { w[0] = *reinterpret_cast<const uint32_t*>(p); }
};
template <> struct Raw<8> {
  uint32_t w[2];
  __device__ inline void load(const uint8_t* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
};
template <> struct Raw<16> {
  uint32_t w[4];
  __device__ inline void load(const uint8_t* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
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

// A tile's bytes, as loaded.
template <int kType, int kD>
struct RawTile {
  using C = CachedCfg<kType, kD>;
  Raw<8 * C::kEsz> k[2][C::kSteps];
  Raw<C::kC * C::kEsz> v[8];
  f32x4 ks[2], vs[2];  // 8-bit types
};

template <int kType, int kD, int kR>
__global__ __launch_bounds__(256, kD > 64 && kR * (kType == FC_CACHE_BF16 ? 2 : 1) == 4 ? 1 : 2) void cached_attn_kernel(CachedAttnArgs a) {
  using C = CachedCfg<kType, kD>;
  constexpr bool k8 = kType != FC_CACHE_BF16;
  constexpr int kRows = 16 * kR;
  constexpr int kPad = kD + 4;  // floats of a row of the exchange: its lanes' stores spread over the banks
  __shared__ Nodes nodes;
  __shared__ float exchange[4 * 16 * kPad];
  __shared__ float2 wave_stats[4][kRows];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
  // Workgroups go to the XCDs in turn: the row groups of one slot, which read the
  // same keys, are 8 workgroups apart, on one XCD and running together.
  const int id = blockIdx.x, of8 = id / 8;
  const int rg = of8 % a.groups, rest = of8 / a.groups * 8 + id % 8;
  const int h = rest / a.items, x = rest - h * a.items;
  if (h >= a.g.Hkv) return;
  const Slot slot = find_slot(a, x, -1);
  if (slot.b < 0) return;
  const int b = slot.b;
  const Span span = span_at(a, b);
  const int length = __builtin_amdgcn_readfirstlane(span.length), count = __builtin_amdgcn_readfirstlane(span.count);
  const int tile0 = __builtin_amdgcn_readfirstlane(span.first) + slot.part * slot.tiles;
  const int tile1 = min(tile0 + slot.tiles, __builtin_amdgcn_readfirstlane(span.first + span.tiles));
  const int end = min(length + count, a.g.capacity);

  if (wave == 0) trace_nodes(&nodes, a.parents == nullptr ? nullptr : a.parents + (a.tree == 2 ? (int64_t)b * a.N : 0), a.N, a.left);
  __syncthreads();

  // This lane's row of each block of 16: its node's view, and its slope.
  uint64_t sees[kR];
  int low[kR], at[kR];
  float slope2[kR];
  bool broken[kR];  // NaN
  bf16x8 q[kR][C::kSteps];
  uint64_t any_sees = 0;
  int any_low = INT_MAX, all_low = 0;  // the first key any row sees, and the first that all do
#pragma unroll
  for (int rb = 0; rb < kR; ++rb) {
    const int row = rg * kRows + rb * 16 + n, node = row / a.G, head = h * a.G + row - node * a.G;
    const bool there = row < a.rows && node < count;
    const int depth = there ? nodes.depth[node] : 0;
    broken[rb] = there && (depth < 0 || node >= a.g.capacity - length);
    sees[rb] = there && !broken[rb] ? nodes.sees[node] : 0;
    at[rb] = length + depth;
    low[rb] = there && !broken[rb] ? max(at[rb] - a.left, 0) : INT_MAX;
    slope2[rb] = a.slopes != nullptr && there ? base2_slope(a.slopes[head]) : 0.0f;
    any_sees |= sees[rb];
    any_low = min(any_low, low[rb]);
    // (rows that are not there, or broken, may take whatever comes)
    all_low = max(all_low, there && !broken[rb] ? low[rb] : 0);
    const bf16* src = static_cast<const bf16*>(a.Q) + (((int64_t)b * a.N + node) * a.H + head) * kD;
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s) {
      const int u = g * C::kSteps + s;
      q[rb][s] = there && u < C::kU ? *reinterpret_cast<const bf16x8*>(src + 8 * u) : Mma<bf16>::zero();
    }
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    any_sees |= __shfl_xor(any_sees, o);
    any_low = min(any_low, __shfl_xor(any_low, o));
    all_low = max(all_low, __shfl_xor(all_low, o));
  }
  any_low = __builtin_amdgcn_readfirstlane(any_low);
  all_low = __builtin_amdgcn_readfirstlane(all_low);

  f32x4 acc[kR][C::kC];
  float ref[kR], sum[kR];
#pragma unroll
  for (int rb = 0; rb < kR; ++rb) {
    ref[rb] = -1e30f;
    sum[rb] = 0.0f;
#pragma unroll
    for (int c = 0; c < C::kC; ++c) acc[rb][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // A block of 16 keys lies in one page: its first row, and whether that page is one.
  struct Place {
    int64_t row;
    bool good;
  };
  const auto place = [&](int key) {
    key = key < end ? key : end - 1 - (end - 1) % 16;  // (a tile's second block may begin past the end)
    const int64_t page = cache_page(a.g, a.table, b, key);
    Place p;
    p.good = page >= 0;
    const int64_t row = ((p.good ? page : 0) * a.g.Hkv + h) * a.g.page_size + cache_place(a.g, a.table, key);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)row), hi = __builtin_amdgcn_readfirstlane((uint32_t)(row >> 32));
    p.row = (int64_t)(((uint64_t)hi << 32) | lo);
    return p;
  };
  RawTile<kType, kD> t;
  Place here[2];  // of the tile whose bytes are in t or on their way
  const float factor0 = a.cap_in > 0.0f ? a.cap_in : a.scale_log2;
  const auto load_k = [&](const Place (&p)[2]) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const uint8_t* kr = static_cast<const uint8_t*>(a.k) + p[kb].row * C::kRow;
#pragma unroll
      for (int s = 0; s < C::kSteps; ++s) {
        const int u = g * C::kSteps + s;  // (units past the row: its last one, left out below)
        t.k[kb][s].load(kr + n * C::kRow + 8 * C::kEsz * (4 * C::kSteps == C::kU ? u : min(u, C::kU - 1)));
      }
      if (k8) t.ks[kb] = *reinterpret_cast<const f32x4*>(a.k_scale + p[kb].row + 4 * g);
    }
  };
  const auto load_v = [&](const Place (&p)[2]) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const uint8_t* vr = static_cast<const uint8_t*>(a.v) + p[kb].row * C::kRow;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        t.v[4 * kb + r].load(vr + (4 * g + r) * C::kRow + C::kC * C::kEsz * (C::kLanes == 16 ? n : min(n, C::kLanes - 1)));
      if (k8) t.vs[kb] = *reinterpret_cast<const f32x4*>(a.v_scale + p[kb].row + 4 * g);
    }
  };

  // A tile; the next one's bytes are requested as soon as this one's leave their registers.
  const auto process = [&](bool masked, int key0, bool more) {
    // S^T of the two blocks: lane n's query, keys key0 + 16 kb + 4 g + r.
    f32x4 s[kR][2], factor[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) s[rb][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int st = 0; st < C::kSteps; ++st) {
        uint32_t w[4];
        if constexpr (k8) {
          w[0] = code_pair<kType, false>(t.k[kb][st].w[0]);
          w[1] = code_pair<kType, true>(t.k[kb][st].w[0]);
          w[2] = code_pair<kType, false>(t.k[kb][st].w[1]);
          w[3] = code_pair<kType, true>(t.k[kb][st].w[1]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = t.k[kb][st].w[i];
        }
        if (4 * C::kSteps != C::kU && g * C::kSteps + st >= C::kU) w[0] = w[1] = w[2] = w[3] = 0;
        const bf16x8 kf = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int rb = 0; rb < kR; ++rb) s[rb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[rb][st], s[rb][kb], 0, 0, 0);
      }
      const float c = here[kb].good ? factor0 : NAN;
#pragma unroll
      for (int r = 0; r < 4; ++r) factor[kb][r] = k8 ? c * t.ks[kb][r] : c;
    }
    if (more) {
      const int key = key0 + 4 * kTileKeys;
      here[0] = place(key);
      here[1] = place(key + 16);
      load_k(here);
    }
    // Scores in base 2.
#pragma unroll
    for (int rb = 0; rb < kR; ++rb)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[rb][kb] *= factor[kb];
    if (a.cap_in > 0.0f) {
#pragma unroll
      for (int rb = 0; rb < kR; ++rb)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[rb][kb][r] = __builtin_fmaf(-2.0f * a.cap_out, cap_part(s[rb][kb][r], 1.0f), a.cap_out);
    }
    if (a.slopes != nullptr) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = key0 + 16 * kb + 4 * g + r;
          const int pos = masked && key >= length && key < length + a.N ? length + nodes.depth[key - length] : key;
#pragma unroll
          for (int rb = 0; rb < kR; ++rb) s[rb][kb][r] = __builtin_fmaf(-slope2[rb], (float)(at[rb] - pos), s[rb][kb][r]);
        }
    }
    int g4 = 4 * g;
    if (masked) {
      asm volatile("" : "+v"(g4));  // (what follows from it would be kept from tile to tile)
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) {
        const uint32_t seen = seen_keys(key0 + g4, low[rb], sees[rb], length);
#pragma unroll
        for (int j = 0; j < 8; ++j)  // P = 0: no reference is below -1e30
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
    bf16x8 pf[kR], pl[kR];
#pragma unroll
    for (int rb = 0; rb < kR; ++rb) {
      bf16x8 f, f2;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float e = __builtin_amdgcn_exp2f(s[rb][j >> 2][j & 3] - ref[rb]);
        sum[rb] += e;
        if (k8) e *= t.vs[j >> 2][j & 3];
        f[j] = static_cast<bf16>(e);
        f2[j] = static_cast<bf16>(e - static_cast<float>(f[j]));
      }
      pf[rb] = f;
      pl[rb] = f2;
    }
    // V's columns: word i of key j holds columns 2 i and 2 i + 1.
    constexpr int kW = (C::kC + 1) / 2;
    uint32_t col[8][kW];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < kW; ++i)
        col[j][i] = !k8 ? t.v[j].w[i] : (i & 1) != 0 ? code_pair<kType, true>(t.v[j].w[i / 2]) : code_pair<kType, false>(t.v[j].w[i / 2]);
    // The c-th product's operand.
    const auto column = [&](int c, auto word) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = word(2 * i, c / 2), y = word(2 * i + 1, c / 2);
        w[i] = (c & 1) != 0 ? high_halves(x, y) : low_halves(x, y);
      }
      return as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
    };
    if (masked) {
      if (k8) {  // (a scale may be NaN)
#pragma unroll
        for (int rb = 0; rb < kR; ++rb) {
          const uint32_t seen = seen_keys(key0 + g4, low[rb], sees[rb], length);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool in = (seen >> (16 * (j >> 2) + (j & 3)) & 1) != 0;
            pf[rb][j] = in ? pf[rb][j] : static_cast<bf16>(0.0f);
            pl[rb][j] = in ? pl[rb][j] : static_cast<bf16>(0.0f);
          }
        }
      }
      const uint32_t any_seen = seen_keys(key0 + g4, any_low, any_sees, length);
      bool odd = false;  // a value that is not finite where some row sees it
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = (any_seen >> (16 * (j >> 2) + (j & 3)) & 1) != 0;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          col[j][i] = in ? col[j][i] : 0;
          if (!k8) odd |= (col[j][i] & 0x7f80u) == 0x7f80u || (col[j][i] & 0x7f800000u) == 0x7f800000u;
        }
      }
      if (!k8 && __ballot(odd) != 0) {
        // Rare (and codes of 8 bits are finite).  Which rows see +infinity, -infinity or NaN in which columns: products of
        // ones; such a value is added to those rows alone and is 0 in the others' product.
#pragma unroll 1
        for (int kind = 0; kind < 3; ++kind) {
          const auto is = [&](uint32_t half) {
            return kind == 0 ? half == 0x7f80u : kind == 1 ? half == 0xff80u : (half & 0x7fffu) > 0x7f80u;
          };
          const auto flags = [&](int j, int i) {
            return (is(col[j][i] & 0xffffu) ? 0x3f80u : 0) | (is(col[j][i] >> 16) ? 0x3f800000u : 0);
          };
          const float what = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
#pragma unroll
          for (int c = 0; c < C::kC; ++c) {
            const bf16x8 vf = column(c, flags);
#pragma unroll
            for (int rb = 0; rb < kR; ++rb) {
              const uint32_t seen = seen_keys(key0 + g4, low[rb], sees[rb], length);
              bf16x8 ones;
#pragma unroll
              for (int j = 0; j < 8; ++j) ones[j] = static_cast<bf16>((seen >> (16 * (j >> 2) + (j & 3)) & 1) != 0 ? 1.0f : 0.0f);
              const f32x4 found = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, ones, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[rb][c][r] += found[r] > 0.0f ? what : 0.0f;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < kW; ++i) {
            if ((col[j][i] & 0x7f80u) == 0x7f80u) col[j][i] &= 0xffff0000u;
            if ((col[j][i] & 0x7f800000u) == 0x7f800000u) col[j][i] &= 0xffffu;
          }
      }
    }
#pragma unroll
    for (int c = 0; c < C::kC; ++c) {
      const bf16x8 vf = column(c, [&](int j, int i) { return col[j][i]; });
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) acc[rb][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[rb], acc[rb][c], 0, 0, 0);
#pragma unroll
      for (int rb = 0; rb < kR; ++rb) acc[rb][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[rb], acc[rb][c], 0, 0, 0);
    }
    if (more) load_v(here);
  };

  int tile = tile0 + wave;
  if (tile < tile1 && count > 0) {
    here[0] = place(tile * kTileKeys);
    here[1] = place(tile * kTileKeys + 16);
    load_k(here);
    load_v(here);
    while (true) {
      const int key0 = tile * kTileKeys;
      const bool more = tile + 4 < tile1;
      // Every row sees every key of a tile before the nodes and behind all rows' first keys.
      process(key0 < all_low || key0 + kTileKeys > length, key0, more);
      if (!more) break;
      tile += 4;
    }
  }

  // Join the four waves: each row's largest reference, then the sums.
#pragma unroll
  for (int rb = 0; rb < kR; ++rb) {
    float l = sum[rb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) wave_stats[wave][rb * 16 + n] = make_float2(ref[rb], broken[rb] ? NAN : l);
  }
  __syncthreads();
  const bool whole = slot.parts == 1;
  const int64_t out_slot = ((int64_t)h * a.groups + rg) * a.items + x;
#pragma unroll
  for (int rb = 0; rb < kR; ++rb) {
    const int rr = rb * 16 + n;
    const float2 st0 = wave_stats[0][rr], st1 = wave_stats[1][rr], st2 = wave_stats[2][rr], st3 = wave_stats[3][rr];
    const float m = fmaxf(fmaxf(st0.x, st1.x), fmaxf(st2.x, st3.x));
    const float by = __builtin_amdgcn_exp2f(ref[rb] - m);
    if (rb > 0) __syncthreads();
    float* to = exchange + (wave * 16 + n) * kPad;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < C::kC; ++c) {
        const int d = C::kC * (4 * g + r) + c;
        if (C::kLanes == 16 || d < kD) to[d] = acc[rb][c][r] * by;
      }
    if (wave == 0 && g == 0 && !whole) {
      const float l = st0.y * __builtin_amdgcn_exp2f(st0.x - m) + st1.y * __builtin_amdgcn_exp2f(st1.x - m) +
                      st2.y * __builtin_amdgcn_exp2f(st2.x - m) + st3.y * __builtin_amdgcn_exp2f(st3.x - m);
      a.part_s[out_slot * kRows + rr] = make_float2(m, l);
    }
    __syncthreads();
    // 256 threads: row tid / 16, columns of tid % 16.
    const int orow = tid >> 4, ox = tid & 15;
    const float2 w0 = wave_stats[0][rb * 16 + orow], w1 = wave_stats[1][rb * 16 + orow], w2 = wave_stats[2][rb * 16 + orow],
                 w3 = wave_stats[3][rb * 16 + orow];
    const float om = fmaxf(fmaxf(w0.x, w1.x), fmaxf(w2.x, w3.x));
    const float l = w0.y * __builtin_amdgcn_exp2f(w0.x - om) + w1.y * __builtin_amdgcn_exp2f(w1.x - om) +
                    w2.y * __builtin_amdgcn_exp2f(w2.x - om) + w3.y * __builtin_amdgcn_exp2f(w3.x - om);
    const int row = rg * kRows + rb * 16 + orow, node = row / a.G, head = h * a.G + row - node * a.G;
    const float inv = 1.0f / l;
    if (row < a.rows) {
      bf16* O = static_cast<bf16*>(a.O) + (((int64_t)b * a.N + node) * a.H + head) * kD;
      float* P = a.part_o + (out_slot * kRows + rb * 16 + orow) * kD;
      for (int d = 4 * ox; d < kD; d += 64) {
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(exchange + (w * 16 + orow) * kPad + d);
        if (whole) {
          v = node < count ? v * inv : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          *reinterpret_cast<uint2*>(O + d) = make_uint2(pair(v[0], v[1]), pair(v[2], v[3]));
        } else {
          *reinterpret_cast<f32x4*>(P + d) = v;
        }
      }
    }
  }
}

// The parts of a row's sequence, where there are several: a workgroup per row.
template <int kD>
__global__ __launch_bounds__(256) void cached_attn_join_kernel(CachedAttnArgs a, int rows_per_group) {
  constexpr int kCols = kD / 4;           // threads of a part, four columns each
  constexpr int kAtOnce = 256 / kCols;    // parts at a time
  __shared__ float weight[1024];
  __shared__ float wave_most[4], wave_sums[4];
  __shared__ f32x4 part[kAtOnce * kCols];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row_id = blockIdx.x;  // (b, node, head)
  const int head = row_id % a.H, bn = row_id / a.H, b = bn / a.N, node = bn - b * a.N;
  const Slot slot = find_slot(a, -1, b);
  if (slot.parts <= 1) return;
  const int h = head / a.G, row = node * a.G + head - h * a.G, rg = row / rows_per_group, rr = row - rg * rows_per_group;
  const int64_t first = ((int64_t)h * a.groups + rg) * a.items + slot.first;
  const int parts = min(slot.parts, 1024);
  float m = -1e30f;
  for (int i = tid; i < parts; i += 256) m = fmaxf(m, a.part_s[(first + i) * rows_per_group + rr].x);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) wave_most[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(wave_most[0], wave_most[1]), fmaxf(wave_most[2], wave_most[3]));
  float l = 0.0f;
  for (int i = tid; i < parts; i += 256) {
    const float2 st = a.part_s[(first + i) * rows_per_group + rr];
    const float w = __builtin_amdgcn_exp2f(st.x - m);
    weight[i] = w;
    l += st.y * w;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if ((tid & 63) == 0) wave_sums[wave] = l;
  __syncthreads();
  l = wave_sums[0] + wave_sums[1] + wave_sums[2] + wave_sums[3];
  const int q = tid / kCols, d = 4 * (tid % kCols);
  f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (q < kAtOnce) {
#pragma unroll 4
    for (int i = q; i < parts; i += kAtOnce)
      v += *reinterpret_cast<const f32x4*>(a.part_o + ((first + i) * rows_per_group + rr) * kD + d) * weight[i];
    part[tid] = v;
  }
  __syncthreads();
  if (tid < kCols) {
#pragma unroll 4
    for (int i = 1; i < kAtOnce; ++i) v += part[i * kCols + tid];
    const Span span = span_at(a, b);
    v = node < span.count ? v * (1.0f / l) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    bf16* O = static_cast<bf16*>(a.O) + (int64_t)row_id * kD;
    *reinterpret_cast<uint2*>(O + d) = make_uint2(pair(v[0], v[1]), pair(v[2], v[3]));
  }
}

// What a variant of row blocks needs (cached_attn.hip instantiates them by type and head dim).
template <int kType> hipError_t launch_cached_attn(const CachedAttnArgs& a, int row_blocks, hipStream_t s);
hipError_t launch_cached_attn_join(const CachedAttnArgs& a, int rows_per_group, hipStream_t s);

}  // namespace fc
