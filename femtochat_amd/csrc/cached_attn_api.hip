// Attention over a cache: the entry points, the rules that size a call, and the
// join of a sequence's parts.
#include "cached_attn.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>

namespace fc {

// A wave for each row, or where there are few rows a workgroup: 64 x 10 rows of 4 parts 3 us
// either way, 16 x 32 x 16 rows of 3 parts 6.4 and 18.5 us, 16 rows of 51 parts 6.4 and 3.1 us.
constexpr int kJoinRows = 2048;

namespace {

template <int kD, bool kInfinite>
void launch_join(const CachedAttnArgs& a, int rows_per_group, hipStream_t s) {
  const int rows = a.g.B * a.N * a.H;
  if (rows <= kJoinRows)
    hipLaunchKernelGGL((cached_attn_join_kernel<kD, 4, kInfinite>), dim3(rows), dim3(256), 0, s, a, rows_per_group);
  else
    hipLaunchKernelGGL((cached_attn_join_kernel<kD, 1, kInfinite>), dim3((rows + 3) / 4), dim3(256), 0, s, a, rows_per_group);
}
template <int kD>
void launch_join(const CachedAttnArgs& a, int rows_per_group, hipStream_t s) {
  if (a.g.type == FC_CACHE_BF16) launch_join<kD, true>(a, rows_per_group, s);
  else launch_join<kD, false>(a, rows_per_group, s);
}

}  // namespace

hipError_t launch_cached_attn_join(const CachedAttnArgs& a, int rows_per_group, hipStream_t s) {
  const ProfileMark mk = profile_begin(s);
  switch (a.g.D) {
    case 16: launch_join<16>(a, rows_per_group, s); break;
    case 32: launch_join<32>(a, rows_per_group, s); break;
    case 48: launch_join<48>(a, rows_per_group, s); break;
    case 64: launch_join<64>(a, rows_per_group, s); break;
    case 80: launch_join<80>(a, rows_per_group, s); break;
    case 96: launch_join<96>(a, rows_per_group, s); break;
    case 112: launch_join<112>(a, rows_per_group, s); break;
    default: launch_join<128>(a, rows_per_group, s); break;
  }
  const hipError_t e = hipGetLastError();
  profile_end(mk, "cached_attn_join", s);
  return e;
}

namespace {

fc_status bad(const char* who, const char* what, fc_status code = FC_ERR_INVALID_ARGUMENT) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  return set_error(code, msg);
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
bool off(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

constexpr int kSlots = 512;       // workgroups: two on each of 256 CUs, which their registers allow
constexpr int kLeastTiles = 12;   // of a share: a sequence's beginning and a tile for each wave
// Up to which a sequence is not shared: the join and its launch cost as much as a longer chain (16 int8 sequences,
// 8 KV heads of 128, one token: 32 tiles 13.6 us whole and 15.6 in parts, 40 15.5 and 16.0, 48 17.2 and 16.1;
// 32 tiles of four sequences with two KV heads 12.6 and 14.1, bf16 15.0 and 16.1).  One sequence of one KV head is
// the exception, 12.4 for 11.6 us, bf16 14.8 for 12.0.
constexpr int kWholeTiles = 32;

// The sizes of a call that follow from its descriptor alone (not from the lengths,
// which lie on the device).
struct Plan {
  int row_blocks, groups, shares, waves;
  size_t s_at, parts_at, bytes;  // in the workspace, behind the parts of O
};

Plan plan_of(const CacheGeom& g, int H, int N, int left) {
  Plan p;
  const int rows = H / g.Hkv * N;
  // Two blocks of sixteen rows read the keys once for both: 16 sequences of 4000 int8 keys
  // with 32 rows and 8 KV heads in 32 us for 38.  Where bf16 rows of more than 64 values leave too few registers
  // for that (16 sequences of up to 4000 keys: 42 us for 38) it is worth it from the third block on only (64
  // rows: 49 us for 60).
  const bool spills = g.type == FC_CACHE_BF16 && g.D > 64;
  p.row_blocks = rows > (spills ? 32 : 16) ? 2 : 1;
  p.groups = (rows + 16 * p.row_blocks - 1) / (16 * p.row_blocks);
  // A sequence's tiles, at most.
  const int64_t span = std::min<int64_t>(g.capacity, (int64_t)left + N + kTileKeys);
  const int64_t tiles = (span + kTileKeys - 1) / kTileKeys;
  p.shares = tiles > kWholeTiles ? std::max(1, kSlots / (g.Hkv * p.groups)) : 0;
  // Eight waves where each workgroup has a CU to itself and a tile for more than four: 4 x 13 nodes, 8 heads of 64 with
  // capped and biased scores over 512 keys, 13.0 us with four, 11.8 with eight; 16 x 16 nodes of two heads over 1000 keys 15.2
  // and 13.7; single tokens the same.
  const bool few = (int64_t)g.B * g.Hkv * p.groups <= kSlots / 2;
  p.waves = p.shares == 0 && few && tiles > 4 ? 8 : 4;
  const int64_t rows_kept = (int64_t)g.Hkv * p.groups * 2 * p.shares * 16 * p.row_blocks;
  p.s_at = round256((size_t)rows_kept * g.D * 4);
  p.parts_at = p.s_at + round256((size_t)rows_kept * sizeof(float2));
  p.bytes = p.shares > 0 ? p.parts_at + round256((size_t)g.B * sizeof(int4)) : 0;
  return p;
}

fc_status options_of(const char* who, const CacheGeom& g, const fc_cached_attn_options* o) {
  if (o == nullptr) return bad(who, "options are null");
  if (g.layers != 1) return bad(who, "attention takes one layer's cache");
  if (o->H <= 0 || o->H % g.Hkv != 0) return bad(who, "H must be a multiple of Hkv");
  if (o->H / g.Hkv > 1024) return bad(who, "at most 1024 query heads per KV head", FC_ERR_UNSUPPORTED);
  if (o->N < 1 || o->N > kMaxNodes) return bad(who, "a call takes 1 to 64 new tokens", o->N < 1 ? FC_ERR_INVALID_ARGUMENT : FC_ERR_UNSUPPORTED);
  if (o->left < -1) return bad(who, "left must be -1 (all) or at least 0");
  if (o->tree < 0 || o->tree > 2) return bad(who, "unknown kind of tree");
  if (!(o->softcap == 0.0f || (o->softcap >= 0x1p-10f && o->softcap <= 4096.0f)))
    return bad(who, "softcap must be 0 (none) or from 2^-10 to 4096");
  if (off(o->slopes, 4)) return bad(who, "slopes must be 4-byte aligned");
  if ((int64_t)g.B * o->N * o->H > (int64_t)1 << 24) return bad(who, "at most 2^24 rows (sequences times new tokens times heads)", FC_ERR_UNSUPPORTED);
  return FC_OK;
}
// A launch holds fewer than 2^32 threads (launch_d's grid; eight waves are for few workgroups only).
fc_status launch_fits(const char* who, const CacheGeom& g, const Plan& p) {
  const int64_t slots = ((int64_t)(p.shares > 0 ? p.shares : g.B) * g.Hkv + 7) / 8 * 8;
  return slots * p.groups * 256 < (int64_t)1 << 32 ? FC_OK : bad(who, "fewer than 2^24 workgroups (sequences times KV heads)", FC_ERR_UNSUPPORTED);
}
int left_of(const fc_cached_attn_options* o) { return o->left < 0 ? INT_MAX / 2 : std::min(o->left, INT_MAX / 2); }

}  // namespace

}  // namespace fc

extern "C" {

fc_status fc_cached_attn_workspace_bytes(const fc_cache_desc* desc, const fc_cached_attn_options* options, size_t* bytes) {
  const char* who = "fc_cached_attn_workspace_bytes";
  fc::CacheGeom g;
  char msg[200];
  fc_status st = fc::make_cache(desc, &g, msg, sizeof(msg));
  if (st != FC_OK) return fc::bad(who, msg, st);
  if ((st = fc::options_of(who, g, options)) != FC_OK) return st;
  if (bytes == nullptr) return fc::bad(who, "bytes is null");
  const fc::Plan p = fc::plan_of(g, options->H, options->N, fc::left_of(options));
  if ((st = fc::launch_fits(who, g, p)) != FC_OK) return st;
  *bytes = p.bytes;
  fc::clear_error();
  return FC_OK;
}

fc_status fc_cached_attn(const fc_cache_desc* desc, const fc_cache* cache, const fc_cached_attn_options* options,
                         const void* Q, void* O, const int32_t* lengths, const int32_t* counts, const int32_t* parents,
                         void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "fc_cached_attn";
  fc::CachedAttnArgs a{};
  fc_status st = fc::check_cache(who, desc, cache, &a.g);
  if (st != FC_OK) return st;
  if ((st = fc::options_of(who, a.g, options)) != FC_OK) return st;
  if (Q == nullptr || O == nullptr || lengths == nullptr) return fc::bad(who, "a required pointer is null");
  if ((options->tree != 0) != (parents != nullptr)) return fc::bad(who, "parents and the kind of tree do not agree");
  if (fc::off(Q, 16) || fc::off(O, 16)) return fc::bad(who, "Q and O must be 16-byte aligned");
  if (fc::off(lengths, 4) || fc::off(counts, 4) || fc::off(parents, 4)) return fc::bad(who, "integer buffers must be 4-byte aligned");
  const int left = fc::left_of(options);
  const fc::Plan p = fc::plan_of(a.g, options->H, options->N, left);
  if ((st = fc::launch_fits(who, a.g, p)) != FC_OK) return st;
  const size_t need = p.bytes;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return fc::bad(who, "the workspace is missing or too small", FC_ERR_WORKSPACE);
  if (need > 0 && fc::off(workspace, 256)) return fc::bad(who, "the workspace must be 256-byte aligned", FC_ERR_WORKSPACE);
  a.k = cache->k, a.v = cache->v, a.k_scale = cache->k_scale, a.v_scale = cache->v_scale;
  a.table = desc->max_pages > 0 ? cache->table : nullptr;
  a.Q = Q, a.O = O, a.lengths = lengths, a.counts = counts, a.parents = parents, a.slopes = options->slopes;
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_s = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.s_at);
  a.parts = reinterpret_cast<int4*>(static_cast<char*>(workspace) + p.parts_at);
  a.H = options->H, a.N = options->N, a.G = options->H / desc->Hkv, a.rows = a.G * a.N;
  a.left = left, a.tree = options->tree;
  a.groups = p.groups, a.shares = p.shares, a.least = fc::kLeastTiles;
  const double scale = 1.0 / std::sqrt((double)desc->D);
  a.scale_log2 = (float)(1.4426950408889634 * scale);
  if (options->softcap > 0.0f) {
    a.cap_in = (float)(2.0 * 1.4426950408889634 * scale / (double)options->softcap);
    a.cap_out = (float)(1.4426950408889634 * options->softcap);
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = desc->type == FC_CACHE_BF16 ? fc::launch_cached_attn<FC_CACHE_BF16>(a, p.row_blocks, p.waves, s)
                 : desc->type == FC_CACHE_I8 ? fc::launch_cached_attn<FC_CACHE_I8>(a, p.row_blocks, p.waves, s)
                                             : fc::launch_cached_attn<FC_CACHE_F8>(a, p.row_blocks, p.waves, s);
  if (e == hipSuccess && p.shares > 0) e = fc::launch_cached_attn_join(a, 16 * p.row_blocks, s);
  if (e != hipSuccess) return fc::bad(who, hipGetErrorString(e), FC_ERR_HIP);
  fc::clear_error();
  return FC_OK;
}

}  // extern "C"
