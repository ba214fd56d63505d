// r4c_rows.cuh — rows of logits: addressing, arithmetic and the two ways of
// reading them shared by the log-probability (r4c_logp.cu) and distillation
// (r4c_distill.cu) kernels.
//
// A row is the class axis at one voxel of an (N, C, D, H, W) map or at one
// token of an (R, C) matrix; r4c_rows_desc gives its place for any strides.
//
// * Up to kTileClasses classes ("tile"): rows wait in shared memory and G lanes
//   take one into registers, so a kernel reads it once whatever it needs of
//   it, and a backward recomputes the softmax instead of loading saved
//   statistics. Tiles of dense rows are one contiguous piece of memory, copied
//   ahead with 16-byte cp.async whatever the alignment of each row (105
//   classes of 2 bytes start on any even byte); other strides are gathered.
// * Above ("block"): a block, or a cluster of blocks when there are few rows,
//   streams over the row in 16-byte loads and keeps a running maximum and sum.
//
// At 6.5 TB/s an SM has about 11 instructions for each 16-bit logit, and what
// these kernels do for a row as a whole comes on top: most spend their issue
// slots before the memory's time. So the arithmetic is packed (two fp32 a instruction), maxima are taken on
// packed words, and checks are made per vector or per row, not per element.
#pragma once

#include <cmath>

#include "r4c_internal.h"
#include "r4c_sm100.cuh"

namespace r4c {
namespace rows {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A rest mass 1 - sum(q) below this is the rounding of the teacher's own sum
// (of fp32 log-probabilities; r4c_distill.cuh has that of 16-bit ones).
constexpr float kRestNoise = 1e-6f;
constexpr int kTileClasses = 1024;
constexpr int kTileThreads = 256;
constexpr int kSMs = 148;
// Threads to a streamed row: one warp up to 16 KB, else 256. What a row costs
// beyond its elements is paid per warp: 16384 rows of 1500 bf16 classes take
// 125 us forward with 256 threads (119 with an alternative) and 52 us backward
// with 128, 29 (47) and 31 us with 32. More than 32 pairs or alternatives take 256, so that each pair has a
// thread and there are maxima enough to choose from.
// (Where they are many, 128 threads do better for alternatives, whose search
// fewer warps then wait for: 4096 rows of 131072 with one take 201 us, not 231;
// without alternatives 217, not 195. Gradients take 128 as well: 4095 rows of
// 32771 with the entropy's 90 us, not 100.)
constexpr int kWarpRow = 32, kLongRow = 256, kManyRows = 128, kGradRow = 128;
inline int row_threads(int C, int es, int k) { return (int64_t)C * es <= 16 << 10 && k <= kWarpRow ? kWarpRow : kLongRow; }

struct View {
  int64_t inner, so, si, sc;   // inner 0: one stride walks all rows
  __device__ __forceinline__ int64_t base(int64_t r) const {
    return inner == 0 ? r * si : (r / inner) * so + (r % inner) * si;
  }
};

inline bool valid_desc(const r4c_rows_desc* d) {
  return d && d->rows >= 0 && d->inner > 0 && d->classes > 0 && std::isfinite(d->temperature) && d->temperature > 0.f;
}
// The entry's status; a failed launch leaves no error behind for the next call to find.
inline int status(cudaError_t e) {
  if (e == cudaSuccess) return R4C_OK;
  cudaGetLastError();
  return R4C_ERR_CUDA;
}
inline bool valid_dtype(int dt) { return dt == R4C_BF16 || dt == R4C_F16 || dt == R4C_F32; }
inline View make_view(const r4c_rows_desc* d) {
  return {d->inner >= d->rows ? 0 : d->inner, d->outer_stride, d->inner_stride, d->class_stride};
}
inline View make_grad_view(const r4c_rows_desc* d) {
  return {d->inner >= d->rows ? 0 : d->inner, d->grad_outer_stride, d->grad_inner_stride, d->grad_class_stride};
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Of normal positive numbers (0 gives -inf).
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The larger of two, NaN if either is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// Exponents below this give 0 whatever they are; bounding them keeps 0 * -inf out of the entropy.
constexpr float kFloor = -200.f;
// A maximum that may be -inf as the point that differences are taken from.
__device__ __forceinline__ float anchor(float m) { return m == -INFINITY ? 0.f : m; }

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

template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int G>
__device__ __forceinline__ bool group_any(bool p) {
  const unsigned b = __ballot_sync(0xffffffffu, p);
  if (G == 32) return b != 0;
  return ((b >> ((threadIdx.x & 31) & ~(G - 1))) & ((1u << (G & 31)) - 1u)) != 0;
}

// A sum of fp32 numbers that keeps what each addition rounds off.
struct Sum2 {
  float s = 0.f, r = 0.f;
  __device__ __forceinline__ void add(float x) {
    const float y = x - r, t = s + y;
    r = fabsf(t) < INFINITY ? (t - s) - y : 0.f;
    s = t;
  }
  __device__ __forceinline__ double value() const { return (double)s - (double)r; }
};

// ---- 32-bit words of logits, and their largest value without unpacking them all -------------------------------------------------
template <typename T> struct Word;
template <> struct Word<float> {
  static constexpr int kElems = 1;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ void split(uint32_t w, float* v) { v[0] = __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t join(const float* v) { return __float_as_uint(v[0]); }
};
template <> struct Word<__nv_bfloat16> {
  static constexpr int kElems = 2;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void split(uint32_t w, float* v) {
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t join(const float* v) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(v[0], v[1]);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <> struct Word<__half> {
  static constexpr int kElems = 2;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ void split(uint32_t w, float* v) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    v[0] = f.x;
    v[1] = f.y;
  }
  static __device__ __forceinline__ uint32_t join(const float* v) {
    const __half2 p = __floats2half2_rn(v[0], v[1]);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};

// Running maximum and sums of exponentials, t_c = (z_c - m) k with
// k = log2(e) / T: s = sum 2^t, u = sum 2^t t. m = -inf: nothing finite yet.
struct Run {
  float m, s, u;
};

// ---- tile: rows held in registers --------------------------------------------
enum { kGather = 0, kCopy = 1, kCopyPadded = 2 };
struct Tile {
  int64_t nrows, ntiles;
  int C, stride;          // classes; elements between rows in shared memory
  int rows, mode;         // rows of a tile; how they come to shared memory
  int stage_bytes;
  int chunks;             // kCopyPadded: 16-byte chunks of a row
  uint32_t recip;         // ... and 2^32 / chunks, rounded up
};
constexpr int kTileStages = 3;

// One lane's part of a row: E values in units of UB = 16, 8 or 4 bytes (rows
// are that aligned, or UB = 4), taken cyclically by the lanes, so value e is
// class c0 + off(e) and classes ascend with e. With UB = 4 a row of 2-byte
// elements may start in the middle of a word: c0 is then one lower (-1 in
// lane 0: not a class).
template <typename T, int G, int E, int UB>
struct TileRow {
  static constexpr int kG = G, kW = Word<T>::kElems;
  static constexpr int kU = UB / (int)sizeof(T);   // elements of a unit
  static constexpr int kN = E / kU;                // units of a lane
  static constexpr bool VEC = UB > 4, kHalf = UB == 4 && kW == 2;   // kHalf: rows may start in a word's middle
  float v[E];
  int lane, c0, C;
  uint32_t at;   // shared address of the lane's first unit

  static __device__ __forceinline__ constexpr int off(int e) { return e / kU * (G * kU) + e % kU; }
  __device__ __forceinline__ int cls(int e) const { return c0 + off(e); }
  // Units are checked in groups: one test for all lanes and elements of a
  // group, and element by element only in the group where the row ends.
  static constexpr int kGroup = VEC || kN < 4 ? (VEC ? 1 : kN) : 4;
  __device__ __forceinline__ bool whole(int i) const { return kU * G * (i + kGroup) <= C; }
  static __device__ __forceinline__ constexpr int step(int i) { return i * (G * kU * (int)sizeof(T)); }

  __device__ __forceinline__ void load(uint32_t row, int classes) {
    C = classes;
    lane = (threadIdx.x & 31) & (G - 1);
    c0 = kU * lane - (kHalf ? (row >> 1) & 1 : 0);
    at = (kHalf ? row & ~3u : row) + lane * UB;
#pragma unroll
    for (int i0 = 0; i0 < kN; i0 += kGroup) {
      if (VEC) {
        uint32_t w[UB / 4];
#pragma unroll
        for (int h = 0; h < UB / 4; ++h) w[h] = Word<T>::kNegInf;
        if (cls(i0 * kU) < C) {
          if constexpr (UB == 16)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at + step(i0)) : "memory");
          else if constexpr (UB == 8)
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at + step(i0)) : "memory");
        }
#pragma unroll
        for (int h = 0; h < UB / 4; ++h) Word<T>::split(w[h], v + i0 * kU + h * kW);
      } else {
        uint32_t w[kGroup];
        if (whole(i0)) {
#pragma unroll
          for (int j = 0; j < kGroup; ++j)
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[j]) : "r"(at + step(i0 + j)) : "memory");
        } else {
#pragma unroll
          for (int j = 0; j < kGroup; ++j) {
            const int c = cls((i0 + j) * kU);
            w[j] = Word<T>::kNegInf;
            if (c < C) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[j]) : "r"(at + step(i0 + j)) : "memory");
            if (kHalf && c + 1 >= C) w[j] = (w[j] & 0xffffu) | (Word<T>::kNegInf & 0xffff0000u);
          }
        }
#pragma unroll
        for (int j = 0; j < kGroup; ++j) Word<T>::split(w[j], v + (i0 + j) * kU);
      }
    }
    if (kHalf && c0 < 0) v[0] = -INFINITY;
  }
  // Writes g over the row in shared memory.
  __device__ __forceinline__ void store(const float* g) const {
#pragma unroll
    for (int i0 = 0; i0 < kN; i0 += kGroup) {
      if (VEC) {
        uint32_t w[UB / 4];
#pragma unroll
        for (int h = 0; h < UB / 4; ++h) w[h] = Word<T>::join(g + i0 * kU + h * kW);
        if (cls(i0 * kU) < C) {
          if constexpr (UB == 16)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + step(i0)), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3]) : "memory");
          else if constexpr (UB == 8)
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + step(i0)), "r"(w[0]), "r"(w[1]) : "memory");
        }
        continue;
      }
      const bool all = whole(i0);
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        const uint32_t a = at + step(i0 + j), w = Word<T>::join(g + (i0 + j) * kU);
        const int c = cls((i0 + j) * kU);
        const bool lo = !(kHalf && i0 + j == 0) || c0 >= 0;   // else the half word is another row's
        if (lo && (all || c + kU <= C)) asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(w) : "memory");
        else if (!lo) asm volatile("st.shared.b16 [%0], %1;" ::"r"(a + 2), "h"((uint16_t)(w >> 16)) : "memory");
        else if (kHalf && c < C) asm volatile("st.shared.b16 [%0], %1;" ::"r"(a), "h"((uint16_t)w) : "memory");
      }
    }
  }
  // Values are worked on eight at a time, as far as the row reaches in any lane.
  static constexpr int kPart = E < 8 ? E : 8;
  __device__ __forceinline__ bool reaches(int e0) const { return e0 == 0 || off(e0) < C; }
  __device__ __forceinline__ float max() const {
    float m = v[0];
#pragma unroll
    for (int e0 = 0; e0 < E; e0 += kPart) {
      if (!reaches(e0)) break;
#pragma unroll
      for (int e = e0; e < e0 + kPart; ++e) m = fmaxf(m, v[e]);
    }
    return group_max<G>(m);
  }
  // v = f(v), two at a time.
  template <typename F>
  __device__ __forceinline__ void each2(F&& f) {
#pragma unroll
    for (int e0 = 0; e0 < E; e0 += kPart) {
      if (!reaches(e0)) break;
#pragma unroll
      for (int e = e0; e < e0 + kPart; e += 2) {
        const float2 g = f(make_float2(v[e], v[e + 1]));
        v[e] = g.x;
        v[e + 1] = g.y;
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ float sh_get(uint32_t a) {
  if (sizeof(T) == 4) {
    float x;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
    return x;
  }
  uint16_t h;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(h) : "r"(a) : "memory");
  return Elem<T>::to_f(*reinterpret_cast<const T*>(&h));
}
template <typename T>
__device__ __forceinline__ void sh_put(uint32_t a, float x) {
  if (sizeof(T) == 4) asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(x) : "memory");
  else {
    const T t = Elem<T>::from_f(x);
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(a), "h"(*reinterpret_cast<const uint16_t*>(&t)) : "memory");
  }
}

// Starts the copy of a tile of dense rows (the last chunk of the last tile in part).
__device__ __forceinline__ void tile_fetch(const Tile& t, const void* z, int64_t tile, int es, uint32_t dst) {
  const int64_t r0 = tile * t.rows;
  if (tile < t.ntiles) {
    const int nr = (int)(t.nrows - r0 < t.rows ? t.nrows - r0 : t.rows);
    const int bytes = nr * t.C * es;
    const uint8_t* src = static_cast<const uint8_t*>(z) + r0 * t.C * es;
    const int pad = t.stride * es - t.chunks * 16;
    for (int b = threadIdx.x; b * 16 < bytes; b += kTileThreads) {
      const uint32_t d = dst + b * 16 + (t.mode == kCopyPadded ? (int)__umulhi(b, t.recip) * pad : 0);
      sm100::cp_async_16(d, src + (int64_t)b * 16, bytes - b * 16 < 16 ? bytes - b * 16 : 16);
    }
  }
  sm100::cp_async_commit();
}
// Gathers a tile of rows that lie anyhow.
template <typename T>
__device__ __forceinline__ void tile_gather(const Tile& t, const View& v, const void* z, int64_t tile, T* stage) {
  const int64_t r0 = tile * t.rows;
  const int nr = (int)(t.nrows - r0 < t.rows ? t.nrows - r0 : t.rows);
  const T* src = static_cast<const T*>(z);
  if (v.sc == 1 && t.C >= 16) {   // lanes along the classes
    for (int q = threadIdx.x / 32; q < nr; q += kTileThreads / 32) {
      const int64_t at = v.base(r0 + q);
      for (int c = threadIdx.x & 31; c < t.C; c += 32) stage[q * t.stride + c] = src[at + c];
    }
  } else {                        // lanes along the rows
    for (int q = threadIdx.x; q < nr; q += kTileThreads) {
      const int64_t at = v.base(r0 + q);
#pragma unroll 8
      for (int c = 0; c < t.C; ++c) stage[q * t.stride + c] = src[at + c * v.sc];
    }
  }
}
// Writes a stage back to the rows of dz (the block has synchronized). dz lies as the stage was filled.
template <typename T>
__device__ __forceinline__ void tile_flush(const Tile& t, const View& v, void* dz, int64_t tile, const T* stage) {
  const int64_t r0 = tile * t.rows;
  const int nr = (int)(t.nrows - r0 < t.rows ? t.nrows - r0 : t.rows);
  if (t.mode != kGather) {
    const int bytes = nr * t.C * (int)sizeof(T);
    const uint8_t* src = reinterpret_cast<const uint8_t*>(stage);
    uint8_t* dst = static_cast<uint8_t*>(dz) + r0 * t.C * sizeof(T);
    const int pad = t.stride * (int)sizeof(T) - t.chunks * 16;
    for (int b = threadIdx.x; b * 16 < bytes; b += kTileThreads) {
      const int s = b * 16 + (t.mode == kCopyPadded ? (int)__umulhi(b, t.recip) * pad : 0);
      if (bytes - b * 16 >= 16) *reinterpret_cast<uint4*>(dst + (int64_t)b * 16) = *reinterpret_cast<const uint4*>(src + s);
      else
        for (int i = 0; i < bytes - b * 16; i += (int)sizeof(T))
          *reinterpret_cast<T*>(dst + (int64_t)b * 16 + i) = *reinterpret_cast<const T*>(src + s + i);
    }
  } else if (v.sc == 1 && t.C >= 16) {
    T* dst = static_cast<T*>(dz);
    for (int q = threadIdx.x / 32; q < nr; q += kTileThreads / 32) {
      const int64_t at = v.base(r0 + q);
      for (int c = threadIdx.x & 31; c < t.C; c += 32) dst[at + c] = stage[q * t.stride + c];
    }
  } else {
    T* dst = static_cast<T*>(dz);
    for (int q = threadIdx.x; q < nr; q += kTileThreads) {
      const int64_t at = v.base(r0 + q);
#pragma unroll 4
      for (int c = 0; c < t.C; ++c) dst[at + c * v.sc] = stage[q * t.stride + c];
    }
  }
}

// Walks the tiles of a persistent block: body(first row of the tile, row
// within it, shared address of the row, in range) for each group of G lanes
// and row (in two parts: the first is the same for the block, so addresses
// need no 64-bit arithmetic per row). All lanes of a warp call body together;
// a group without a row of its own repeats the last one and writes nothing.
template <typename T, int G, bool WRITES, typename Body>
__device__ __forceinline__ void tile_walk(const Tile& t, const View& v, const void* z, const View& dv, void* dz,
                                          Body&& body) {
  extern __shared__ __align__(16) uint8_t stages[];
  constexpr int R = kTileThreads / G;
  const int sub = threadIdx.x / G;
  const uint32_t base = sm100::smem_u32(stages);
  if (t.mode != kGather)
    for (int s = 0; s < kTileStages - 1; ++s)
      tile_fetch(t, z, blockIdx.x + (int64_t)s * gridDim.x, sizeof(T), base + s * t.stage_bytes);
  int st = 0;
  for (int64_t tile = blockIdx.x; tile < t.ntiles; tile += gridDim.x) {
    if (t.mode != kGather) {
      sm100::cp_async_wait<kTileStages - 2>();
      __syncthreads();   // this tile has landed for everyone, the last one is done with
      const int nx = st == 0 ? kTileStages - 1 : st - 1;
      tile_fetch(t, z, tile + (int64_t)(kTileStages - 1) * gridDim.x, sizeof(T), base + nx * t.stage_bytes);
    } else {
      __syncthreads();
      tile_gather<T>(t, v, z, tile, reinterpret_cast<T*>(stages));
      __syncthreads();
    }
    const int64_t r0 = tile * t.rows;
    const int nr = (int)(t.nrows - r0 < t.rows ? t.nrows - r0 : t.rows);
    for (int i = 0; i < nr; i += R) {
      const int q = i + sub, at = q < nr ? q : nr - 1;
      body(r0, at, base + st * t.stage_bytes + at * (t.stride * (int)sizeof(T)), q < nr);
    }
    if (WRITES) {
      __syncthreads();
      tile_flush<T>(t, dv, dz, tile, reinterpret_cast<T*>(stages + st * t.stage_bytes));
    }
    if (t.mode != kGather) st = st == kTileStages - 1 ? 0 : st + 1;
  }
}

inline bool dense_rows(const View& v, int64_t rows, int classes, const void* p) {
  return v.inner == 0 && (v.sc == 1 || classes == 1) && (v.si == classes || rows == 1) && ((uintptr_t)p & 15) == 0;
}
// Lanes per row and values per lane by the number of classes: as few lanes as
// 32 registers of values allow, since what a row costs beyond its elements is
// paid once per group of lanes.
struct TileKind {
  int g, e, ub;
};
inline int row_unit(int C, int es) { return C * es % 16 == 0 ? 16 : C * es % 8 == 0 ? 8 : 4; }
inline TileKind tile_kind(int C, int es) {
  const int ub = row_unit(C, es);
  if (C <= 32) return {1, C <= 4 ? 4 : C <= 8 ? 8 : C <= 16 ? 16 : 32, ub};
  int g = 2;
  while (C > g * 32) g *= 2;
  return {g, 32, ub == 16 ? 16 : 4};
}
// Calls f(G, E, UB as constants) for a kind; a unit needs as many values as it holds.
template <int G_, int E_, int UB_>
struct TileConst {
  static constexpr int G = G_, E = E_, UB = UB_;
};
template <typename T, typename F>
inline cudaError_t for_tile_kind(const TileKind& k, F&& f) {
#define R4C_TILE(G, E)                                            \
  if (k.g == G && k.e == E) {                                     \
    if constexpr (E * sizeof(T) >= 16)                            \
      if (k.ub == 16) return f(TileConst<G, E, 16>{});            \
    if constexpr (G == 1)                                         \
      if (k.ub == 8) return f(TileConst<G, E, 8>{});              \
    return f(TileConst<G, E, 4>{});                               \
  }
  R4C_TILE(1, 4) R4C_TILE(1, 8) R4C_TILE(1, 16) R4C_TILE(1, 32) R4C_TILE(2, 32) R4C_TILE(4, 32) R4C_TILE(8, 32)
  R4C_TILE(16, 32) R4C_TILE(32, 32)
#undef R4C_TILE
  return cudaErrorInvalidValue;
}
// Tiles of up to 16 KB, 8 KB for the shortest rows (at least one row for each
// group of lanes): three of them in flight in each of the blocks of an SM keep the memory busy.
inline Tile make_tile(int64_t nrows, int C, int es, int g, bool dense) {
  Tile t{};
  t.nrows = nrows;
  t.C = C;
  t.mode = !dense ? kGather : C * es % 16 ? kCopy : kCopyPadded;
  // rows that lie an even number of units apart would meet in the same banks
  const int unit = row_unit(C, es);
  t.stride = t.mode == kCopy ? C : ((C * es + unit - 1) / unit | 1) * unit / es;
  t.chunks = C * es / 16;
  t.recip = t.chunks ? (uint32_t)(((1ull << 32) + t.chunks - 1) / t.chunks) : 0;
  const int r = kTileThreads / g;
  int reps = (g == 1 ? 8 << 10 : 16 << 10) / (r * t.stride * es);
  reps = reps < 1 ? 1 : reps > 16 ? 16 : reps;
  // few rows: smaller tiles, so that every SM gets some
  while (reps > 1 && nrows < (int64_t)r * reps * 2 * kSMs) reps /= 2;
  t.rows = r * reps;
  t.ntiles = (nrows + t.rows - 1) / t.rows;
  t.stage_bytes = (t.rows * t.stride * es + 31) / 16 * 16;
  return t;
}
inline size_t tile_smem(const Tile& t) { return (size_t)(t.mode == kGather ? 1 : kTileStages) * t.stage_bytes; }

// Blocks of a kernel that an SM holds, remembered per host thread (asking
// takes longer than a launch): a persistent grid of more would leave some of
// them to run alone after the others. Also allows the kernel its shared
// memory where that is above the default (44 KB, with the kernels' static
// shared memory).
constexpr int kMostShared = 200 << 10;
template <typename K>
inline int blocks_per_sm(K* kernel, int threads, size_t smem) {
  struct Known {
    const void* kernel;
    size_t smem;
    int dev, blocks;
  };
  static thread_local Known known[256];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const void* f = reinterpret_cast<const void*>(kernel);
  Known& k = known[((reinterpret_cast<uintptr_t>(f) >> 4) * 2654435761u + smem / 16 * 40503u + dev) % 256];
  if (k.kernel == f && k.smem == smem && k.dev == dev) return k.blocks;
  // the allowance is the kernel's for good, so it is one for all sizes: a later, smaller one would take it back
  if (smem > kMostShared) return 0;
  if (smem > 44 << 10 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess)
    return 0;
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) return 0;
  k = {f, smem, dev, n};
  return n;
}
// *blocks: the size of the grid.
template <typename K, typename A>
inline cudaError_t launch_tile(K* kernel, const Tile& t, int* blocks, cudaStream_t st, const A& a) {
  const size_t smem = tile_smem(t);
  const int per_sm = blocks_per_sm(kernel, kTileThreads, smem);
  if (per_sm < 1) return cudaErrorInvalidConfiguration;
  *blocks = (int)(t.ntiles < kSMs * per_sm ? t.ntiles : kSMs * per_sm);
  kernel<<<*blocks, kTileThreads, smem, st>>>(a);
  return cudaGetLastError();
}

// ---- block: rows streamed ------------------------------------------------------
template <typename T> struct Vec {
  static constexpr int kElems = 16 / (int)sizeof(T);
  static __device__ __forceinline__ void split(const uint4& x, float* v) {
    constexpr int w = Word<T>::kElems;
    Word<T>::split(x.x, v);
    Word<T>::split(x.y, v + w);
    Word<T>::split(x.z, v + 2 * w);
    Word<T>::split(x.w, v + 3 * w);
  }
  static __device__ __forceinline__ float top(const uint4& x) {
    return Word<T>::top(Word<T>::max(Word<T>::max(x.x, x.y), Word<T>::max(x.z, x.w)));
  }
  static __device__ __forceinline__ uint4 join(const float* v) {
    constexpr int w = Word<T>::kElems;
    return make_uint4(Word<T>::join(v), Word<T>::join(v + w), Word<T>::join(v + 2 * w), Word<T>::join(v + 3 * w));
  }
};

// A row as 16-byte vectors of the aligned memory around it: vector v holds
// the classes [v * kElems - off, ...); the first and last may be partly outside.
template <typename T>
struct VecRow {
  const uint4* p;
  const T* row;
  int off, nv, C;
  __device__ __forceinline__ VecRow(const T* z, int classes) : row(z), C(classes) {
    off = (int)(((uintptr_t)z & 15) / sizeof(T));
    p = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(z) & ~(uintptr_t)15);
    nv = (off + C + Vec<T>::kElems - 1) / Vec<T>::kElems;
  }
  __device__ __forceinline__ int first_full() const { return off ? 1 : 0; }
  __device__ __forceinline__ int end_full() const { return (off + C) / Vec<T>::kElems; }
  __device__ __forceinline__ int cls(int v) const { return v * Vec<T>::kElems - off; }
};

__device__ __forceinline__ Run run_empty() { return {-INFINITY, 0.f, 0.f}; }
__device__ __forceinline__ Run run_merge(const Run& a, const Run& b, float k) {
  const float m = fmaxf(a.m, b.m), mm = anchor(m);
  const float ta = max_nan((a.m - mm) * k, kFloor), tb = max_nan((b.m - mm) * k, kFloor);
  const float fa = ex2(ta), fb = ex2(tb);
  return {m, a.s * fa + b.s * fb, fa * (a.u + ta * a.s) + fb * (b.u + tb * b.s)};
}
// A thread's part, in two interleaved chains (packed fp32 arithmetic).
struct Run2 {
  float m;
  float2 s, u;
  __device__ __forceinline__ Run join() const { return {m, s.x + s.y, u.x + u.y}; }
};
__device__ __forceinline__ Run2 run2_empty() { return {-INFINITY, {0.f, 0.f}, {0.f, 0.f}}; }
template <bool ENT>
__device__ __forceinline__ void run2_raise(Run2& r, float m, float k) {
  if (m > r.m) {
    const float t = max_nan((r.m - m) * k, kFloor), f = ex2(t);
    const float2 f2 = {f, f}, t2 = {t, t};
    if (ENT) r.u = __fmul2_rn(f2, __ffma2_rn(t2, r.s, r.u));
    r.s = __fmul2_rn(f2, r.s);
    r.m = m;
  }
}
// x[0..N) with r.m at least their maximum; N even.
template <int N, bool ENT>
__device__ __forceinline__ void run2_add(Run2& r, const float* x, float k) {
  const float mm = -anchor(r.m);
  const float2 m2 = {mm, mm}, k2 = {k, k};
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float2 t = __fmul2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), m2), k2);
    if (ENT) t = make_float2(max_nan(t.x, kFloor), max_nan(t.y, kFloor));
    const float2 e = {ex2(t.x), ex2(t.y)};
    r.s = __fadd2_rn(r.s, e);
    if (ENT) r.u = __ffma2_rn(e, t, r.u);
  }
}
// A row in registers: v becomes the exponents t, and the group's run over it
// comes back (places outside the row hold -inf and add nothing).
template <typename Row>
__device__ __forceinline__ Run tile_run(Row& x, float k) {
  const float m = x.max(), mm = -anchor(m);
  const float2 m2 = {mm, mm}, k2 = {k, k};
  float2 s = {0.f, 0.f}, u = {0.f, 0.f};
  x.each2([&](float2 z) {
    float2 t = __fmul2_rn(__fadd2_rn(z, m2), k2);
    t = make_float2(max_nan(t.x, kFloor), max_nan(t.y, kFloor));
    const float2 e = {ex2(t.x), ex2(t.y)};
    s = __fadd2_rn(s, e);
    u = __ffma2_rn(e, t, u);
    return t;
  });
  return {m, group_sum<Row::kG>(s.x + s.y), group_sum<Row::kG>(u.x + u.y)};
}
// The same without the entropy's sum: v becomes the exponentials themselves.
template <typename Row>
__device__ __forceinline__ Run tile_exp(Row& x, float k) {
  const float m = x.max(), mm = -anchor(m);
  const float2 m2 = {mm, mm}, k2 = {k, k};
  float2 s = {0.f, 0.f};
  x.each2([&](float2 z) {
    const float2 t = __fmul2_rn(__fadd2_rn(z, m2), k2);
    const float2 e = {ex2(t.x), ex2(t.y)};
    s = __fadd2_rn(s, e);
    return e;
  });
  return {m, group_sum<Row::kG>(s.x + s.y), 0.f};
}

// As run2_add<N, true>, with the exponents bounded only in a batch that turns
// u into NaN: 0 * -inf, from a masked class (the sum s then needs no repair).
template <int N, int U, typename Split>
__device__ __forceinline__ void run2_batch(Run2& r, float k, Split&& split) {
  const float mm = -anchor(r.m);
  const float2 m2 = {mm, mm}, k2 = {k, k};
  float2 u = r.u;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float x[N];
    split(i, x);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 t = __fmul2_rn(__fadd2_rn(make_float2(x[j], x[j + 1]), m2), k2);
      const float2 e = {ex2(t.x), ex2(t.y)};
      r.s = __fadd2_rn(r.s, e);
      u = __ffma2_rn(e, t, u);
    }
  }
  if (isnan(u.x + u.y)) {
    u = r.u;
#pragma unroll 1
    for (int i = 0; i < U; ++i) {
      float x[N];
      split(i, x);
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float2 t = __fmul2_rn(__fadd2_rn(make_float2(x[j], x[j + 1]), m2), k2);
        t = make_float2(max_nan(t.x, kFloor), max_nan(t.y, kFloor));
        u = __ffma2_rn(make_float2(ex2(t.x), ex2(t.y)), t, u);
      }
    }
  }
  r.u = u;
}
template <bool ENT>
__device__ __forceinline__ void run2_one(Run2& r, float x, float k) {
  run2_raise<ENT>(r, x, k);
  const float y[2] = {x, -INFINITY};
  run2_add<2, ENT>(r, y, k);
}
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
// Joins the threads' runs of a block; every thread gets the result. The
// maximum goes first, so that each thread rescales its sums once.
template <int NT>
struct RunShared {
  float m[NT / 32];
  float2 su[NT / 32];
};
template <int NT>
__device__ __forceinline__ Run run_block(Run r, float k, RunShared<NT>& sh) {
  constexpr int W = NT / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float wm = warp_max(r.m);
  if (lane == 0) sh.m[warp] = wm;
  __syncthreads();
  float m = sh.m[0];
#pragma unroll
  for (int i = 1; i < W; ++i) m = fmaxf(m, sh.m[i]);
  const float t = max_nan((r.m - anchor(m)) * k, kFloor), f = ex2(t);
  const float s = group_sum<32>(f * r.s), u = group_sum<32>(f * (r.u + t * r.s));
  if (lane == 0) sh.su[warp] = make_float2(s, u);
  __syncthreads();
  Run out{m, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < W; ++i) {
    out.s += sh.su[i].x;
    out.u += sh.su[i].y;
  }
  return out;
}

// A thread's own ring of 16-byte vectors in shared memory: batches of U
// vectors (a block's stride apart) are copied ahead with cp.async and read
// back by the thread that asked for them, so the copies in flight cost
// neither registers nor barriers.
template <int NT, int U, int S>
struct VecRing {
  static constexpr int kBytes = NT * U * S * 16;
  uint32_t base;
  int in, out;
  __device__ __forceinline__ explicit VecRing(void* smem)
      : base(sm100::smem_u32(smem) + threadIdx.x * 16), in(0), out(0) {}
  // Vectors p[i * NT] for i * NT < left (left counts from this thread's first); any left: the batch is counted.
  __device__ __forceinline__ void issue(const uint4* p, int left) {
    const uint32_t d = base + in * (U * NT * 16);
    if ((U - 1) * NT < left) {
#pragma unroll
      for (int i = 0; i < U; ++i) sm100::cp_async_16(d + i * (NT * 16), p + i * NT, 16);
    } else {
#pragma unroll
      for (int i = 0; i < U - 1; ++i)
        if (i * NT < left) sm100::cp_async_16(d + i * (NT * 16), p + i * NT, 16);
    }
    sm100::cp_async_commit();
    in = in == S - 1 ? 0 : in + 1;
  }
  // The oldest batch, with S - 1 issued since the start of it or later.
  __device__ __forceinline__ void take(uint4* w) {
    sm100::cp_async_wait<S - 2>();
    const uint32_t d = base + out * (U * NT * 16);
#pragma unroll
    for (int i = 0; i < U; ++i)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w) : "r"(d + i * (NT * 16)) : "memory");
    out = out == S - 1 ? 0 : out + 1;
  }
};

// A block's piece of a row's gradient: dz = pair(z) for every class of the
// piece, two at a time.
constexpr int kGradBatch = 4, kGradStages = 3;
// Pieces of a row: about sixteen vectors a thread, fewer where the rows alone leave SMs idle.
inline int grad_pieces(int64_t nrows, int C, int es, int threads) {
  const int64_t nv = ((int64_t)C * es + 15) / 16 + 1;
  int64_t most = (nv + threads * 2 - 1) / (threads * 2), p = (nv + threads * 16 - 1) / (threads * 16);
  if (threads == kWarpRow) return 1;
  while (p < most && nrows * p < 4 * kSMs) ++p;
  return (int)p;
}
template <typename T, int NT_>
struct GradPiece {
  static constexpr int VE = Vec<T>::kElems, U = kGradBatch, NT = NT_;
  VecRow<T> x, y;
  int v0, v1, f0, f1;
  VecRing<NT, U, kGradStages> ring;
  __device__ __forceinline__ GradPiece(const T* z, T* dz, int C, int piece, int pieces, void* smem)
      : x(z, C), y(dz, C), ring(smem) {
    const int per = (x.nv + pieces - 1) / pieces;
    v0 = min(piece * per, x.nv);
    v1 = min(v0 + per, x.nv);
    f0 = max(v0, x.first_full());
    f1 = min(v1, x.end_full());
    for (int b = 0; b < kGradStages - 1; ++b) fetch(b);
  }
  __device__ __forceinline__ void fetch(int b) {
    const int v = f0 + b * (U * NT) + (int)threadIdx.x;
    ring.issue(x.p + v, f1 - v);
  }
  __device__ __forceinline__ bool has(int c) const {
    const int v = (c + x.off) / VE;
    return v >= v0 && v < v1;
  }
  template <typename Pair>
  __device__ __forceinline__ void write(Pair&& pair) {
    T* row = const_cast<T*>(y.row);
    uint4* out = const_cast<uint4*>(y.p) + f0 + threadIdx.x;
    const bool same = x.off == y.off;   // both rows break into vectors at the same classes
    int b = 0;
    for (int left = f1 - f0 - (int)threadIdx.x; left > -(int)threadIdx.x; left -= U * NT, ++b) {
      uint4 w[U];
      ring.take(w);
      fetch(b + kGradStages - 1);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (i * NT >= left) break;
        float g[VE];
        Vec<T>::split(w[i], g);
#pragma unroll
        for (int j = 0; j < VE; j += 2) {
          const float2 q = pair(make_float2(g[j], g[j + 1]));
          g[j] = q.x;
          g[j + 1] = q.y;
        }
        const int at = b * (U * NT) + i * NT;
        if (same) out[at] = Vec<T>::join(g);
        else
          for (int j = 0; j < VE; ++j) row[x.cls(f0 + at + (int)threadIdx.x) + j] = Elem<T>::from_f(g[j]);
      }
    }
    // the partial vectors at the row's ends, one element a thread
    auto edge = [&](int c) {
      if (c >= 0 && c < x.C) row[c] = Elem<T>::from_f(pair(make_float2(Elem<T>::to_f(x.row[c]), 0.f)).x);
    };
    if (f0 > v0 && threadIdx.x < VE) edge(x.cls(v0) + threadIdx.x);
    if (f1 < v1 && f1 >= f0 && threadIdx.x >= NT - VE) edge(x.cls(f1) + threadIdx.x - (NT - VE));
  }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this block's shared variable in block `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_map(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sm100::smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float cluster_ld_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t cluster_ld_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ Run cluster_ld_run(const Run* p, uint32_t rank) {
  const uint32_t a = cluster_map(p, rank);
  return {cluster_ld_f32(a), cluster_ld_f32(a + 4), cluster_ld_f32(a + 8)};
}

// The vectors of the rows that a block (of a cluster) takes in turn, batch by
// batch and ahead across the rows' ends, so that the memory stays busy while
// a row is finished. skip(row): neither read nor taken.
template <typename T, int NT, int U, int S, typename Skip>
struct RowStream {
  VecRing<NT, U, S> ring;
  const T* z;
  const View& v;
  int64_t nrows, step, row;   // row: the one that is read ahead
  int C, cs, cr;
  const uint4* p;
  int left;                   // full vectors of it not asked for yet
  Skip skip;
  bool skip_next;
  __device__ __forceinline__ RowStream(void* smem, const T* z_, const View& v_, int64_t nrows_, int C_, int cs_, int cr_,
                                       Skip skip_)
      : ring(smem), z(z_), v(v_), nrows(nrows_), step(gridDim.x / cs_), row(blockIdx.x / cs_), C(C_), cs(cs_), cr(cr_),
        left(0), skip(skip_), skip_next(false) {
    skip_next = row < nrows && skip(row);
    open();
    for (int s = 0; s < S - 1; ++s) ahead();
  }
  // This block's share of a row: vectors [v0, v1), the whole ones [f0, f1).
  __device__ __forceinline__ void share(const VecRow<T>& x, int* v0, int* v1, int* f0, int* f1) const {
    const int per = cs == 1 ? x.nv : (x.nv + cs - 1) / cs;
    *v0 = min(cr * per, x.nv);
    *v1 = min(*v0 + per, x.nv);
    *f0 = max(*v0, x.first_full());
    *f1 = min(*v1, x.end_full());
  }
  __device__ __forceinline__ void open() {   // at `row`, or the first one after it that has something to read
    while (row < nrows) {
      const bool sk = skip_next;
      skip_next = row + step < nrows && skip(row + step);   // loaded a row early
      if (!sk) {
        const VecRow<T> x(z + v.base(row), C);
        int v0, v1, f0, f1;
        share(x, &v0, &v1, &f0, &f1);
        left = f1 - f0;
        p = x.p + f0 + threadIdx.x;
        if (left > 0) return;
      }
      row += step;
    }
    left = 0;
  }
  __device__ __forceinline__ void ahead() {
    ring.issue(p, left - (int)threadIdx.x);
    p += U * NT;
    left -= U * NT;
    if (left <= 0 && row < nrows) {
      row += step;
      open();
    }
  }
  __device__ __forceinline__ void take(uint4* w) {
    ring.take(w);
    ahead();
  }
};

// The runs of a cluster's blocks joined, in every lane of the calling warp.
__device__ __forceinline__ Run run_cluster(const Run* mine, int cs, float k) {
  const int lane = threadIdx.x & 31;
  Run r = lane < cs ? cluster_ld_run(mine, lane) : run_empty();
#pragma unroll
  for (int o = 8; o; o >>= 1)
    r = run_merge(r, Run{__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o),
                         __shfl_xor_sync(0xffffffffu, r.u, o)}, k);
  return {__shfl_sync(0xffffffffu, r.m, 0), __shfl_sync(0xffffffffu, r.s, 0), __shfl_sync(0xffffffffu, r.u, 0)};
}

// Blocks that share a row: as many as bring the rows to two blocks an SM, in
// powers of two up to 8 (16 were slower: one row of 131072 took 25 us, not 16),
// while each keeps a few vectors a thread.
inline int cluster_size(int64_t nrows, int C, int es, int threads) {
  int cs = 1;
  while (cs < 8 && nrows * cs * 2 <= 2 * kSMs && (int64_t)C * es >= (int64_t)threads * 16 * 2 * (cs * 2)) cs *= 2;
  return cs;
}

template <typename K, typename A>
inline cudaError_t launch_cluster(K* kernel, int64_t grid, int threads, int cs, size_t smem, cudaStream_t st, const A& a) {
  if (blocks_per_sm(kernel, threads, smem) < 1) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  if (cs > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace rows
}  // namespace r4c
