// The sums of a split dK/dV's float32 parts (DkdvSplit), in order, added to the
// caller's gradients or written over them and rounded once.  Bound by HBM or, for the
// small problems that are split, by its launch; four values per thread.
#include "attn_device.hpp"
#include "attn_launch.hpp"

namespace fc {

namespace {

// (gradients may lie off a 16-byte boundary)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <typename V>
__device__ inline void put(V* out, f32x4 s, bool accumulate) {
  if (accumulate) s += __builtin_convertvector(*out, f32x4);
  *out = __builtin_convertvector(s, V);
}

__global__ __launch_bounds__(256) void attn_join_kernel(JoinArgs a) {
  const int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (i >= a.n) return;
  const float* part = (blockIdx.y == 0 ? a.part_k : a.part_v) + i;
  f32x4 s = *reinterpret_cast<const f32x4*>(part);
  for (int k = 1; k < a.parts; ++k) s += *reinterpret_cast<const f32x4*>(part + k * a.n);
  void* const out = blockIdx.y == 0 ? a.dK : a.dV;
  if (a.grad_bf16) put(reinterpret_cast<bf16x4_any*>(static_cast<bf16*>(out) + i), s, a.accumulate != 0);
  else put(reinterpret_cast<f32x4_any*>(static_cast<float*>(out) + i), s, a.accumulate != 0);
}

}  // namespace

hipError_t launch_join(const JoinArgs& a, hipStream_t s) {
  const ProfileMark mk = profile_begin(s);
  hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)((a.n / 4 + 255) / 256), 2), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  profile_end(mk, "attn_join", s);
  return e;
}

}  // namespace fc
