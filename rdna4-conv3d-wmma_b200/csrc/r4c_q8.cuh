// r4c_q8.cuh — an activation in 8 bits: codes with one power of two for every 32 elements in memory order.
//
// Block of 32: a = largest finite magnitude, e = the least integer >= -127 with a <= M 2^e, M = 127 (whole numbers
// with a sign) or 448 (8-bit floating point, 4 exponent and 3 mantissa bits). code = x 2^-e rounded to the nearest,
// ties to even; NaN and infinities get the code of NaN (-128, or 0x7f). The stored byte is e + 127. Powers of two
// keep every product exact, so the codes are the same wherever they are computed, and 8 bits for 32 elements cost
// 3 % where an fp32 scale would cost 12 %. Rounding: half a unit of 2^e, that is at most a / 127 (int8), or 2^-4 of
// the value down to a / 57344 (e4m3).
// Read back: code 2^e in the activation's type, rounded to nearest (only fp16 numbers below 2^-14 can need it), at
// most the type's largest finite number (a code may round up past it).
#pragma once

#include <cuda_fp8.h>

#include "r4c_common.cuh"

namespace r4c {
namespace q8 {

constexpr int kBlock = 32;

// Stored exponent byte of a block whose largest finite magnitude has these fp32 bits. 127 = 1.984375 * 2^6 and
// 448 = 1.75 * 2^8: what is added to the mantissa carries into the exponent when it is above theirs (0x7e0000, 0x600000).
__device__ __forceinline__ int exponent_byte(uint32_t amax_bits, int format) {
  const int b = format == R4C_Q8_INT8 ? (int)((amax_bits + 0x1ffffu) >> 23) - 6 : (int)((amax_bits + 0x1fffffu) >> 23) - 8;
  return b < 0 ? 0 : b;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
__device__ __forceinline__ float scale(int byte) { return __uint_as_float(max((uint32_t)byte << 23, 0x00400000u)); }

// V codes (V = 1, 2, 4 or 8) in the low bytes of the words.
template <int V>
struct Codes {
  uint32_t w[V > 4 ? 2 : 1];
};

template <int V>
__device__ __forceinline__ Codes<V> load_codes(const uint8_t* p) {
  Codes<V> c;
  if constexpr (V == 8) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    c.w[0] = r.x;
    c.w[1] = r.y;
  } else if constexpr (V == 4) {
    c.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (V == 2) {
    c.w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else {
    c.w[0] = *p;
  }
  return c;
}
template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const Codes<V>& c) {
  if constexpr (V == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(c.w[0], c.w[1]);
  else if constexpr (V == 4)
    *reinterpret_cast<uint32_t*>(p) = c.w[0];
  else if constexpr (V == 2)
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)c.w[0];
  else
    *p = (uint8_t)c.w[0];
}

// `finite`: no NaN or infinity among them.
template <int V>
__device__ __forceinline__ Codes<V> encode(const float (&f)[V], int byte, int format, bool finite) {
  static_assert(V % 4 == 0, "whole words of codes");
  Codes<V> c;
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const float2 lo = __fmul2_rn(make_float2(f[4 * i], f[4 * i + 1]), make_float2(inv, inv));
    const float2 hi = __fmul2_rn(make_float2(f[4 * i + 2], f[4 * i + 3]), make_float2(inv, inv));
    if (format == R4C_Q8_INT8) {
      // 1.5 * 2^23 + q rounds q to the nearest whole number, ties to even, and leaves it in the low byte
      const float2 m = make_float2(12582912.f, 12582912.f);
      const float2 a = __fadd2_rn(lo, m), b = __fadd2_rn(hi, m);
      const uint32_t ab = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
      const uint32_t cd = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
      c.w[i] = __byte_perm(ab, cd, 0x5410);
    } else {
      const uint32_t ab = __nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3);
      const uint32_t cd = __nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3);
      c.w[i] = ab | cd << 16;
    }
  }
  if (!finite) {
    const uint32_t nan = format == R4C_Q8_INT8 ? 0x80u : 0x7fu;
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (!(fabsf(f[k]) < INFINITY)) c.w[k / 4] = (c.w[k / 4] & ~(0xffu << (8 * (k % 4)))) | nan << (8 * (k % 4));
  }
  return c;
}

// Bytes below / above which a value may need T's rounding / T's largest number. (fp16's smallest step is 2^-24, a whole
// number's 2^e, an e4m3 code's 2^(e-9). Codes of an fp16 tensor are multiples of its step all the same; others' may not be.)
template <typename T> struct Limits;
template <> struct Limits<__half> {
  static constexpr int low_int8 = 103, low_e4m3 = 112, high_int8 = 136, high_e4m3 = 134;
  static __device__ __forceinline__ float most() { return 65504.f; }
};
template <> struct Limits<__nv_bfloat16> {
  static constexpr int low_int8 = -1, low_e4m3 = -1, high_int8 = 248, high_e4m3 = 246;
  static __device__ __forceinline__ float most() { return __uint_as_float(0x7f7f0000u); }
};
template <> struct Limits<float> {
  static constexpr int low_int8 = -1, low_e4m3 = -1, high_int8 = 248, high_e4m3 = 246;
  static __device__ __forceinline__ float most() { return __uint_as_float(0x7f7fffffu); }
};

// The values of T that the codes stand for.
template <typename T, int V>
__device__ __forceinline__ void decode(const Codes<V>& c, int byte, int format, float (&f)[V]) {
  const float s = scale(byte);
  bool rare = byte < (format == R4C_Q8_INT8 ? Limits<T>::low_int8 : Limits<T>::low_e4m3);   // T's rounding, its largest number, NaN
  if (format == R4C_Q8_INT8) {
    // 0x4b0000uu is 2^23 + u exactly: the signed code is that minus 2^23 + 128 (no integer-to-float conversions,
    // which share a slow pipe). Times 2^e it is exact either way round: one multiply-add a value, while
    // 2^e (2^23 + 128) is a number (e <= 103).
    constexpr int kHigh = Limits<T>::high_int8 < 230 ? Limits<T>::high_int8 : 230;
    uint32_t u[V > 4 ? 2 : 1], zero = 0;
#pragma unroll
    for (int i = 0; i < (V > 4 ? 2 : 1); ++i) {
      u[i] = c.w[i] ^ 0x80808080u;
      zero |= (u[i] - 0x01010101u) & ~u[i];                   // a byte of u is 0: some code is -128
    }
    zero &= V < 4 ? 0x80808080u >> (32 - 8 * (V < 4 ? V : 4)) : 0x80808080u;
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = __uint_as_float(__byte_perm(u[k / 4], 0x4b000000u, 0x7440 + (k & 3)));
    rare |= byte > kHigh || zero != 0;
    if (!rare) {
      const float m = -8388736.f * s;
      if constexpr (V == 1) f[0] = fmaf(f[0], s, m);
#pragma unroll
      for (int k = 0; k + 1 < V; k += 2) {
        const float2 d = __ffma2_rn(make_float2(f[k], f[k + 1]), make_float2(s, s), make_float2(m, m));
        f[k] = d.x;
        f[k + 1] = d.y;
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float q = f[k] - 8388736.f;
      f[k] = q == -128.f ? __uint_as_float(0x7fc00000u) : q * s;
    }
  } else {
    rare |= byte > Limits<T>::high_e4m3;
    if constexpr (V == 1) {
      f[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(c.w[0] & 0xffu), __NV_E4M3))) * s;
    } else {
#pragma unroll
      for (int k = 0; k < V; k += 2) {
        const __nv_fp8x2_storage_t b = (__nv_fp8x2_storage_t)(c.w[k / 4] >> (8 * (k % 4)));
        const float2 d = __fmul2_rn(__half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(b, __NV_E4M3))), make_float2(s, s));
        f[k] = d.x;
        f[k + 1] = d.y;
      }
    }
    if (!rare) return;
  }
  const float most = Limits<T>::most();
#pragma unroll
  for (int k = 0; k < V; ++k) {
    f[k] = f[k] > most ? most : (f[k] < -most ? -most : f[k]);
    f[k] = Elem<T>::to_f(Elem<T>::from_f(f[k]));
  }
}

// The larger magnitudes of two pairs of 16-bit numbers; NaN stays.
template <typename T>
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (__is_same(T, __half)) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Largest finite magnitude (fp32 bits) of a block that lies in neighbouring lanes, each with NW words of T; every lane of
// `mask` takes part. `finite`: this lane's elements all are. 16-bit types are compared two at a time as they lie.
template <typename T, int NW>
__device__ __forceinline__ uint32_t block_amax(const uint32_t (&w)[NW], uint32_t mask, bool* finite) {
  constexpr bool kWide = sizeof(T) == 4;
  constexpr uint32_t kSign = kWide ? 0x7fffffffu : 0x7fff7fffu;
  // infinity's bits: everything from there on is not finite
  constexpr uint32_t kInf = kWide ? 0x7f800000u : (__is_same(T, __half) ? 0x7c00u : 0x7f80u);
  uint32_t m = w[0] & kSign;
#pragma unroll
  for (int k = 1; k < NW; ++k) {
    if constexpr (kWide) m = max(m, w[k] & kSign);
    else m = larger2<T>(m, w[k] & kSign);
  }
  if constexpr (!kWide) m = max(m & 0xffffu, m >> 16);
  const bool bad = m >= kInf;
  *finite = !bad;
  if (__any_sync(mask, bad)) {                  // NaN or infinities somewhere: the finite ones alone
    m = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const uint32_t v = w[k] & kSign;
      if constexpr (kWide) {
        m = max(m, v < kInf ? v : 0u);
      } else {
        m = max(m, (v & 0xffffu) < kInf ? v & 0xffffu : 0u);
        m = max(m, (v >> 16) < kInf ? v >> 16 : 0u);
      }
    }
  }
  constexpr int kLanes = kBlock * (int)sizeof(T) / 4 / NW;
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) m = max(m, __shfl_xor_sync(mask, m, o));
  if constexpr (kWide) return m;
  else if constexpr (__is_same(T, __half)) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
  else return m << 16;
}

}  // namespace q8
}  // namespace r4c
