// r4c_q8.cu — activations into 8 bits and back (r4c_pack8, r4c_unpack8).
//
// Element-wise passes over memory order, bound by HBM: pack reads b bytes and writes 1.03, unpack the reverse
// (b = 2 or 4). A thread holds 8 elements (16 bytes of bf16 / fp16, 32 of fp32), four threads a block of 32, whose
// maximum takes two shuffles; several such pieces a thread keep enough loads in flight.
#include <algorithm>

#include "r4c_internal.h"
#include "r4c_q8.cuh"

namespace r4c {
namespace q8 {

// Measured at 201 M bf16 elements, pack / unpack: five pieces a thread and blocks of 128 threads, ten an SM, 103 / 93 us;
// four and four blocks of 256 118 / 93, two and eight 118 / 97, eight and three 120 / 125.
constexpr int kThreads = 128;
constexpr int kUnroll = 5;

// 8 elements: 16 bytes of 16-bit types, 32 of fp32.
template <typename T>
struct Oct {
  static constexpr int NW = 2 * (int)sizeof(T);
  uint32_t w[NW];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < NW / 4; ++i) {
      const uint4 r = __ldcs(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = r.x, w[4 * i + 1] = r.y, w[4 * i + 2] = r.z, w[4 * i + 3] = r.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < NW / 4; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = 0;
  }
  // element k from memory, for the last, incomplete eight (k is a constant where the loops are unrolled)
  __device__ __forceinline__ void set(int k, T v) {
    if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v);
    else w[k / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(&v) << (16 * (k & 1));
  }
  __device__ __forceinline__ void to_f(float (&f)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (sizeof(T) == 4) {
        f[k] = __uint_as_float(w[k]);
      } else {
        const uint16_t h = (uint16_t)(w[k / 2] >> (16 * (k & 1)));
        f[k] = Elem<T>::to_f(*reinterpret_cast<const T*>(&h));
      }
    }
  }
  __device__ __forceinline__ void from_f(const float (&f)[8]) {
    T* p = reinterpret_cast<T*>(w);
#pragma unroll
    for (int k = 0; k < 8; ++k) p[k] = Elem<T>::from_f(f[k]);
  }
};

// `vec`: x lies on 16 bytes (codes always do). The last, incomplete eight elements go one by one.
template <typename T>
__global__ void __launch_bounds__(kThreads, 10) pack_kernel(const T* __restrict__ x, int64_t count, int vec, int format,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  const int64_t octs = (count + 7) / 8, full = vec ? count / 8 : 0;
  constexpr int step = kThreads;
  // whole warps walk together: the bound is rounded up to a warp's 32 threads
  const int64_t bound = (octs + 31) / 32 * 32, all = (int64_t)gridDim.x * kThreads * kUnroll;
  for (int64_t base = (int64_t)blockIdx.x * kThreads * kUnroll + threadIdx.x; base < bound; base += all) {
    Oct<T> a[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = base + u * step;
      a[u].zero();
      if (i < full) {
        a[u].load(x + i * 8);
      } else if (i < octs) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i * 8 + k < count) a[u].set(k, x[i * 8 + k]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = base + u * step;
      if (i >= bound) break;                       // the same for a whole warp
      float f[8];
      a[u].to_f(f);
      bool finite;
      const int byte = exponent_byte(block_amax<T>(a[u].w, 0xffffffffu, &finite), format);
      const Codes<8> c = encode<8>(f, byte, format, finite);
      if (i >= octs) continue;
      if ((i + 1) * 8 <= count) {
        store_codes<8>(codes + i * 8, c);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i * 8 + k < count) codes[i * 8 + k] = (uint8_t)(c.w[k / 4] >> (8 * (k % 4)));
      }
      if ((i & 3) == 0) exps[i >> 2] = (uint8_t)byte;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 12) unpack_kernel(const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ exps, int64_t count, int vec,
                                                          int format, T* __restrict__ x) {
  const int64_t octs = (count + 7) / 8, full = count / 8;
  constexpr int step = kThreads;
  const int64_t all = (int64_t)gridDim.x * kThreads * kUnroll;
  for (int64_t base = (int64_t)blockIdx.x * kThreads * kUnroll + threadIdx.x; base < octs; base += all) {
    Codes<8> c[kUnroll];
    int byte[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = base + u * step;
      c[u].w[0] = c[u].w[1] = 0;
      byte[u] = 0;
      if (i < full) {
        c[u] = load_codes<8>(codes + i * 8);
      } else if (i < octs) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i * 8 + k < count) c[u].w[k / 4] |= (uint32_t)codes[i * 8 + k] << (8 * (k % 4));
      }
      if (i < octs) byte[u] = exps[i >> 2];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = base + u * step;
      if (i >= octs) break;
      float f[8];
      decode<T, 8>(c[u], byte[u], format, f);
      if (vec && i < full) {
        Oct<T> o;
        o.from_f(f);
        o.store(x + i * 8);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i * 8 + k < count) x[i * 8 + k] = Elem<T>::from_f(f[k]);
      }
    }
  }
}

// A block for every kUnroll * kThreads eights: many short blocks share the memory's time out more evenly than one wave
// of long ones (a copy of 201 MB: 60 against 66 us).
static int64_t grid_for(int64_t count) {
  const int64_t octs = (count + 7) / 8;
  return std::max<int64_t>(1, std::min<int64_t>((octs + kThreads * kUnroll - 1) / (kThreads * kUnroll), 1 << 30));
}

static bool ok_args(const void* x, const void* codes, const void* exps, int64_t count, int dtype, int format) {
  return x && codes && exps && count >= 0 && (dtype == R4C_BF16 || dtype == R4C_F16 || dtype == R4C_F32) &&
         (format == R4C_Q8_INT8 || format == R4C_Q8_E4M3) && (reinterpret_cast<uintptr_t>(codes) & 15) == 0 &&
         (reinterpret_cast<uintptr_t>(x) & (dtype_bytes(dtype) - 1)) == 0;
}

}  // namespace q8
}  // namespace r4c

using namespace r4c::q8;

extern "C" {

int r4c_pack8(const void* x, int64_t count, int dtype, int format, void* codes, void* exponents,
              r4c_stream_t stream) {
  if (count == 0) return R4C_OK;
  if (!ok_args(x, codes, exponents, count, dtype, format)) return R4C_ERR_INVALID;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)grid_for(count);
  const int vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* e = static_cast<uint8_t*>(exponents);
  if (dtype == R4C_BF16)
    pack_kernel<<<grid, kThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(x), count, vec, format, c, e);
  else if (dtype == R4C_F16)
    pack_kernel<<<grid, kThreads, 0, s>>>(static_cast<const __half*>(x), count, vec, format, c, e);
  else
    pack_kernel<<<grid, kThreads, 0, s>>>(static_cast<const float*>(x), count, vec, format, c, e);
  r4c::note_launches(1);
  return cudaGetLastError() == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}

int r4c_unpack8(const void* codes, const void* exponents, int64_t count, int dtype, int format, void* x,
                r4c_stream_t stream) {
  if (count == 0) return R4C_OK;
  if (!ok_args(x, codes, exponents, count, dtype, format)) return R4C_ERR_INVALID;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)grid_for(count);
  const int vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* e = static_cast<const uint8_t*>(exponents);
  if (dtype == R4C_BF16)
    unpack_kernel<<<grid, kThreads, 0, s>>>(c, e, count, vec, format, static_cast<__nv_bfloat16*>(x));
  else if (dtype == R4C_F16)
    unpack_kernel<<<grid, kThreads, 0, s>>>(c, e, count, vec, format, static_cast<__half*>(x));
  else
    unpack_kernel<<<grid, kThreads, 0, s>>>(c, e, count, vec, format, static_cast<float*>(x));
  r4c::note_launches(1);
  return cudaGetLastError() == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}

}  // extern "C"
