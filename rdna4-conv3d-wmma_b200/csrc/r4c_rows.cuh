// r4c_rows.cuh — rows of logits: addressing and arithmetic shared by the
// log-probability (r4c_logp.cu) and distillation (r4c_distill.cu) kernels.
//
// A row is the class axis at one voxel of an (N, C, D, H, W) map or at one
// token of an (R, C) matrix; r4c_rows_desc gives its place for any strides.
#pragma once

#include <cmath>

#include "r4c_internal.h"

namespace r4c {
namespace rows {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A rest mass 1 - sum(q) below this is the rounding of the teacher's own sum.
constexpr float kRestNoise = 1e-6f;

struct View {
  int64_t inner, so, si, sc;
  __device__ __forceinline__ int64_t base(int64_t r) const { return (r / inner) * so + (r % inner) * si; }
};

inline bool valid_desc(const r4c_rows_desc* d) {
  return d && d->rows >= 0 && d->inner > 0 && d->classes > 0 && std::isfinite(d->temperature) && d->temperature > 0.f;
}
inline bool valid_dtype(int dt) { return dt == R4C_BF16 || dt == R4C_F16 || dt == R4C_F32; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Total order of the finite values and infinities as unsigned integers
// (-0 and +0 equal), ties to the lower class: larger key = ranked first.
__device__ __forceinline__ uint64_t rank_key(float z, int c) {
  const uint32_t b = __float_as_uint(z + 0.f);
  const uint32_t o = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)(0xffffffffu - (uint32_t)c);
}
__device__ __forceinline__ int key_class(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

}  // namespace rows
}  // namespace r4c
