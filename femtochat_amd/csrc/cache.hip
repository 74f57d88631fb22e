// The cache of keys and values (gfx950): tokens are quantised as they are
// written, read back, and moved where a path of drafted tokens is kept.
//
// All three are bound by HBM (or, for a few tokens, by the launch): a thread
// takes 8 values of a key and the same 8 of its value vector, so that one look at
// the table serves both, and D/8 lanes hold a vector, whose largest magnitude is
// a reduction over at most 16 neighbouring lanes (DPP, no LDS).
#include "attn_device.hpp"
#include "attn_launch.hpp"
#include "cache_index.hpp"
#include "cache_types.hpp"

#include <algorithm>
#include <cstdio>

namespace fc {

namespace {

constexpr int kCacheThreads = 256;

struct CacheArgs {
  CacheGeom g;
  void *k, *v;
  float *k_scale, *v_scale;
  const int32_t* table;
  void *K, *V;              // (layers, B, T, Hkv, D)
  const int32_t* from;      // lengths or starts, or null (0)
  const int32_t* counts;    // or null
  const int32_t* path;      // fc_cache_keep
  int T;
  FastDiv by_Hkv;
};

// Lanes that share a vector of U 8-value units.
constexpr int vector_lanes(int U) { return U <= 2 ? 2 : U <= 4 ? 4 : U <= 8 ? 8 : 16; }

// The largest of kLanes neighbouring lanes, in all of them.
template <int kLanes>
__device__ inline uint32_t lanes_max(uint32_t v) {
  const auto step = [&](auto ctrl) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(ctrl)::value, 0xf, 0xf, false));
  };
  step(std::integral_constant<int, 0xB1>{});                      // quad_perm [1, 0, 3, 2]
  if (kLanes > 2) step(std::integral_constant<int, 0x4E>{});      // quad_perm [2, 3, 0, 1]
  if (kLanes > 4) step(std::integral_constant<int, 0x141>{});     // row_half_mirror
  if (kLanes > 8) step(std::integral_constant<int, 0x140>{});     // row_mirror
  return v;
}

__device__ inline void load8(const float* p, float (&x)[8]) {
  const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[i + 4] = b[i];
}
__device__ inline void load8(const bf16* p, float (&x)[8]) {
  const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
}
__device__ inline void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
  reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
}
__device__ inline void store8(bf16* p, const float (&x)[8]) {
  bf16x8 a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = static_cast<bf16>(x[i]);
  *reinterpret_cast<bf16x8*>(p) = a;
}

// One vector's 8 values of this lane into its row; all lanes of the vector call it.
template <int kType, int U>
__device__ inline void write_unit(void* rows, float* scales, int64_t row, int u, const float (&x)[8]) {
  constexpr int D = 8 * U;
  if (kType == FC_CACHE_BF16) {
    if (u < U && row >= 0) store8(static_cast<bf16*>(rows) + row * D + 8 * u, x);
    return;
  }
  // Magnitudes compare as integers, infinities and NaN above all numbers.
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
  most = lanes_max<vector_lanes(U)>(u < U ? most : 0);
  const float top = kType == FC_CACHE_I8 ? 127.0f : 448.0f, a = __uint_as_float(most);
  const bool finite = most < 0x7f800000u, zero = !(a >= 0x1p-100f);
  const float inv = zero ? 0.0f : top / a, scale = !finite ? __uint_as_float(0x7fc00000u) : zero ? 0.0f : a / top;
  if (u >= U || row < 0) return;
  uint32_t w[2] = {0, 0};
  if (finite) {
    if (kType == FC_CACHE_I8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4] |= ((uint32_t)(int)__builtin_rintf(x[i] * inv) & 0xffu) << (8 * (i % 4));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, b, true);
      }
    }
  }
  *reinterpret_cast<uint2*>(static_cast<uint8_t*>(rows) + row * D + 8 * u) = make_uint2(w[0], w[1]);
  if (u == 0) scales[row] = scale;
}

template <int kType, int U>
__device__ inline void read_unit(const void* rows, const float* scales, int64_t row, int u, float (&x)[8]) {
  constexpr int D = 8 * U;
  if (kType == FC_CACHE_BF16) {
    load8(static_cast<const bf16*>(rows) + row * D + 8 * u, x);
    return;
  }
  const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(rows) + row * D + 8 * u);
  const float s = scales[row];
  code_values<kType>(w.x, x[0], x[1], x[2], x[3]);
  code_values<kType>(w.y, x[4], x[5], x[6], x[7]);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= s;
}

// Token t of sequence b and its head of this thread's vector; i lies within the sequence's tokens.
struct Vector {
  int layer, b, t, h, u;
};
template <int U>
__device__ inline Vector vector_of(const CacheArgs& a, int64_t i) {
  constexpr int L = vector_lanes(U);
  const int n = (int)(i / L);
  Vector v;
  v.u = (int)(i % L);
  v.t = (int)divide((uint32_t)n, a.by_Hkv);
  v.h = n - v.t * a.g.Hkv;
  v.b = blockIdx.y;
  v.layer = blockIdx.z;
  return v;
}

// Whole vectors' lanes stay together (a sweep is a multiple of 16 threads).
template <int kType, int U, typename E>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(CacheArgs a) {
  constexpr int D = 8 * U, L = vector_lanes(U);
  const int b = blockIdx.y;
  const int n = a.counts == nullptr ? a.T : min(max(a.counts[b], 0), a.T);
  const int length = a.from == nullptr ? 0 : a.from[b];
  const int64_t last = (int64_t)n * a.g.Hkv * L;
  for (int64_t i = (int64_t)blockIdx.x * kCacheThreads + threadIdx.x; i < last; i += (int64_t)gridDim.x * kCacheThreads) {
    const Vector c = vector_of<U>(a, i);
    const int64_t at = ((((int64_t)c.layer * a.g.B + b) * a.T + c.t) * a.g.Hkv + c.h) * D + 8 * c.u;
    float xk[8] = {}, xv[8] = {};
    if (c.u < U) {
      load8(static_cast<const E*>(a.K) + at, xk);
      load8(static_cast<const E*>(a.V) + at, xv);
    }
    const int64_t row = cache_row(a.g, a.table, c.layer, b, c.h, behind(a.g, length, c.t));
    write_unit<kType, U>(a.k, a.k_scale, row, c.u, xk);
    write_unit<kType, U>(a.v, a.v_scale, row, c.u, xv);
  }
}

template <int kType, int U, typename E>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(CacheArgs a) {
  constexpr int D = 8 * U, L = vector_lanes(U);
  const int b = blockIdx.y;
  const int n = a.counts == nullptr ? a.T : min(max(a.counts[b], 0), a.T);
  const int start = a.from == nullptr ? 0 : a.from[b];
  const int64_t last = (int64_t)a.T * a.g.Hkv * L;
  for (int64_t i = (int64_t)blockIdx.x * kCacheThreads + threadIdx.x; i < last; i += (int64_t)gridDim.x * kCacheThreads) {
    const Vector c = vector_of<U>(a, i);
    if (c.u >= U) continue;
    const int64_t at = ((((int64_t)c.layer * a.g.B + b) * a.T + c.t) * a.g.Hkv + c.h) * D + 8 * c.u;
    float xk[8] = {}, xv[8] = {};
    if (c.t < n) {
      const int64_t row = cache_row(a.g, a.table, c.layer, b, c.h, behind(a.g, start, c.t));
      if (row >= 0) {
        read_unit<kType, U>(a.k, a.k_scale, row, c.u, xk);
        read_unit<kType, U>(a.v, a.v_scale, row, c.u, xv);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) xk[e] = xv[e] = __uint_as_float(0x7fc00000u);
      }
    }
    store8(static_cast<E*>(a.K) + at, xk);
    store8(static_cast<E*>(a.V) + at, xv);
  }
}

// A workgroup moves up to kKeepPieces pieces of every kept token: 16 bytes of a head's k or v, or
// one of its scales.  Its threads take as many tokens at a time as they are, four times over,
// and read them all before they write any: dst j <= path[j] and the path increases, so what
// is written then lies before all that is read later.  The tokens' places are looked up 64
// at a time.  (a thread that moves its piece of one token after another waits for the path, the
// page and the bytes of each four: 20 layers, 32 sequences, 3 tokens on average, 29 us for 5)
constexpr int kKeepPieces = 64, kKeepTokens = 64;
__global__ __launch_bounds__(kCacheThreads) void cache_keep_kernel(CacheArgs a, int pieces, int row_bytes) {
  __shared__ int64_t from_row[kKeepTokens], to_row[kKeepTokens];  // of head 0; -1: nothing to move
  const int b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
  const int per_head = 2 * pieces + (a.k_scale != nullptr ? 2 : 0), first = blockIdx.x * kKeepPieces;
  const int here = min(per_head * a.g.Hkv - first, kKeepPieces), at_once = kCacheThreads / here;
  const int token = tid / here, i = first + tid - token * here;
  const int h = i / per_head, part = i - h * per_head;
  const int n = a.counts == nullptr ? a.T : min(max(a.counts[b], 0), a.T);
  const int length = a.from[b];
  const bool scale = part >= 2 * pieces;
  const int of = scale ? part - 2 * pieces : part / pieces;  // 0: k, 1: v
  char* data = scale ? reinterpret_cast<char*>(of == 0 ? a.k_scale : a.v_scale) : static_cast<char*>(of == 0 ? a.k : a.v);
  const int64_t stride = scale ? 4 : row_bytes;
  data += (int64_t)h * a.g.page_size * stride + (scale ? 0 : 16 * (part % pieces));
  for (int j0 = 0; j0 < n; j0 += kKeepTokens) {
    if (tid < kKeepTokens) {
      const int j = j0 + tid, from = j < n ? a.path[(int64_t)b * a.T + j] : -1;
      const bool moves = from >= 0 && from < a.T && from != j;
      const int64_t src = moves ? cache_row(a.g, a.table, layer, b, 0, behind(a.g, length, from)) : -1;
      const int64_t dst = moves ? cache_row(a.g, a.table, layer, b, 0, behind(a.g, length, j)) : -1;
      from_row[tid] = dst < 0 ? -1 : src;
      to_row[tid] = dst;
    }
    __syncthreads();
    const int m = min(n - j0, kKeepTokens);
    for (int j = 0; j < m; j += 4 * at_once) {
      uint4 x[4];
      int64_t src[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = j + e * at_once + token;
        src[e] = token < at_once && t < m ? from_row[t] : -1;
        x[e] = make_uint4(0, 0, 0, 0);
        if (src[e] < 0) continue;
        if (scale) x[e].x = *reinterpret_cast<const uint32_t*>(data + src[e] * stride);
        else x[e] = *reinterpret_cast<const uint4*>(data + src[e] * stride);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)  // (the bytes are there before the barrier)
        asm volatile("" : "+v"(x[e].x), "+v"(x[e].y), "+v"(x[e].z), "+v"(x[e].w));
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (src[e] < 0) continue;
        char* dst = data + to_row[j + e * at_once + token] * stride;
        if (scale) *reinterpret_cast<uint32_t*>(dst) = x[e].x;
        else *reinterpret_cast<uint4*>(dst) = x[e];
      }
    }
    __syncthreads();
  }
}

template <int kType, int U>
hipError_t launch_tokens(const CacheArgs& a, bool write, bool b16, hipStream_t s) {
  const int64_t threads = (int64_t)a.T * a.g.Hkv * vector_lanes(U);
  // Sweeps where a launch would hold 2^31 threads and more.
  const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 31) / kCacheThreads / ((int64_t)a.g.B * a.g.layers));
  const dim3 grid((unsigned)std::min((threads + kCacheThreads - 1) / kCacheThreads, most), (unsigned)a.g.B, (unsigned)a.g.layers);
  const ProfileMark mk = profile_begin(s);
  if (write) {
    if (b16) hipLaunchKernelGGL((cache_write_kernel<kType, U, bf16>), grid, dim3(kCacheThreads), 0, s, a);
    else hipLaunchKernelGGL((cache_write_kernel<kType, U, float>), grid, dim3(kCacheThreads), 0, s, a);
  } else {
    if (b16) hipLaunchKernelGGL((cache_read_kernel<kType, U, bf16>), grid, dim3(kCacheThreads), 0, s, a);
    else hipLaunchKernelGGL((cache_read_kernel<kType, U, float>), grid, dim3(kCacheThreads), 0, s, a);
  }
  const hipError_t e = hipGetLastError();
  profile_end(mk, write ? "cache_write" : "cache_read", s);
  return e;
}

template <int kType>
hipError_t launch_tokens(const CacheArgs& a, bool write, bool b16, hipStream_t s) {
  switch (a.g.D) {
    case 16: return launch_tokens<kType, 2>(a, write, b16, s);
    case 32: return launch_tokens<kType, 4>(a, write, b16, s);
    case 48: return launch_tokens<kType, 6>(a, write, b16, s);
    case 64: return launch_tokens<kType, 8>(a, write, b16, s);
    case 80: return launch_tokens<kType, 10>(a, write, b16, s);
    case 96: return launch_tokens<kType, 12>(a, write, b16, s);
    case 112: return launch_tokens<kType, 14>(a, write, b16, s);
    case 128: return launch_tokens<kType, 16>(a, write, b16, s);
    default: return hipErrorInvalidValue;
  }
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
bool off(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

fc_status cache_args(const char* who, const fc_cache_desc* d, const fc_cache* c, int32_t T, const int32_t* from,
                     const int32_t* counts, CacheArgs* a) {
  *a = CacheArgs{};
  const fc_status st = check_cache(who, d, c, &a->g);
  if (st != FC_OK) return st;
  if (T <= 0) return bad(who, "T and N must be positive");
  if ((int64_t)T * d->Hkv > (int64_t)1 << 30 || (int64_t)d->B * d->layers > (int64_t)1 << 22)
    return bad(who, "at most 2^30 heads of a sequence's tokens and 2^22 sequences of all layers", FC_ERR_UNSUPPORTED);
  if (off(from, 4) || off(counts, 4)) return bad(who, "integer buffers must be 4-byte aligned");
  a->k = c->k, a->v = c->v, a->k_scale = c->k_scale, a->v_scale = c->v_scale, a->table = c->table;
  if (d->type == FC_CACHE_BF16) a->k_scale = a->v_scale = nullptr;
  if (d->max_pages == 0) a->table = nullptr;
  a->from = from, a->counts = counts, a->T = T;
  a->by_Hkv = fast_div((uint32_t)d->Hkv);
  return FC_OK;
}

fc_status tokens(const char* who, bool write, const fc_cache_desc* d, const fc_cache* c, const void* K, const void* V,
                 int32_t dtype, int32_t T, const int32_t* from, const int32_t* counts, void* stream) {
  CacheArgs a;
  const fc_status st = cache_args(who, d, c, T, from, counts, &a);
  if (st != FC_OK) return st;
  if (dtype != FC_F32 && dtype != FC_BF16) return bad(who, "dtype must be FC_F32 or FC_BF16");
  if (K == nullptr || V == nullptr || (write && from == nullptr)) return bad(who, "a required pointer is null");
  if (off(K, 16) || off(V, 16)) return bad(who, "K and V must be 16-byte aligned");
  a.K = const_cast<void*>(K), a.V = const_cast<void*>(V);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool b16 = dtype == FC_BF16;
  return done(who, d->type == FC_CACHE_BF16 ? launch_tokens<FC_CACHE_BF16>(a, write, b16, s)
                   : d->type == FC_CACHE_I8 ? launch_tokens<FC_CACHE_I8>(a, write, b16, s)
                                            : launch_tokens<FC_CACHE_F8>(a, write, b16, s));
}

}  // namespace

fc_status check_cache(const char* who, const fc_cache_desc* d, const fc_cache* c, CacheGeom* g) {
  char msg[200];
  const fc_status st = make_cache(d, g, msg, sizeof(msg));
  if (st != FC_OK) return bad(who, msg, st);
  if (c == nullptr || c->k == nullptr || c->v == nullptr) return bad(who, "the cache is null");
  if (d->type != FC_CACHE_BF16 && (c->k_scale == nullptr || c->v_scale == nullptr)) return bad(who, "an 8-bit cache has scales");
  if (d->max_pages > 0 && c->table == nullptr) return bad(who, "the table is null");
  if (off(c->k, 16) || off(c->v, 16) || off(c->k_scale, 16) || off(c->v_scale, 16) || off(c->table, 4))
    return bad(who, "the cache must be 16-byte aligned, its table 4-byte");
  return FC_OK;
}

}  // namespace fc

extern "C" {

fc_status fc_cache_write(const fc_cache_desc* desc, const fc_cache* cache, const void* K, const void* V, int32_t in_dtype,
                         int32_t T, const int32_t* lengths, const int32_t* counts, void* stream) {
  return fc::tokens("fc_cache_write", true, desc, cache, K, V, in_dtype, T, lengths, counts, stream);
}

fc_status fc_cache_read(const fc_cache_desc* desc, const fc_cache* cache, void* K, void* V, int32_t out_dtype, int32_t T,
                        const int32_t* starts, const int32_t* counts, void* stream) {
  return fc::tokens("fc_cache_read", false, desc, cache, K, V, out_dtype, T, starts, counts, stream);
}

fc_status fc_cache_keep(const fc_cache_desc* desc, const fc_cache* cache, int32_t N, const int32_t* lengths,
                        const int32_t* path, const int32_t* counts, void* stream) {
  const char* who = "fc_cache_keep";
  fc::CacheArgs a;
  const fc_status st = fc::cache_args(who, desc, cache, N, lengths, counts, &a);
  if (st != FC_OK) return st;
  if (lengths == nullptr || path == nullptr) return fc::bad(who, "a required pointer is null");
  if (fc::off(path, 4)) return fc::bad(who, "integer buffers must be 4-byte aligned");
  a.path = path;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int row_bytes = desc->D * fc::cache_value_bytes(desc->type), pieces = row_bytes / 16;
  const int all = desc->Hkv * (2 * pieces + (a.k_scale != nullptr ? 2 : 0));
  const fc::ProfileMark mk = fc::profile_begin(s);
  hipLaunchKernelGGL(fc::cache_keep_kernel, dim3((unsigned)((all + fc::kKeepPieces - 1) / fc::kKeepPieces), (unsigned)desc->B, (unsigned)desc->layers),
                     dim3(fc::kCacheThreads), 0, s, a, pieces, row_bytes);
  const hipError_t e = hipGetLastError();
  fc::profile_end(mk, "cache_keep", s);
  return fc::done(who, e);
}

}  // extern "C"
