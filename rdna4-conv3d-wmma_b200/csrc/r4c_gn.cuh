// r4c_gn.cuh — group normalisation with an activation on channels-last activations: the kernels.
//
// x is (N, S, C), C innermost, in G groups of Cg = C / G channels; m = Cg * S elements a group and sample.
//   mean, rstd = statistics of a (sample, group), rstd = (var + eps)^-1/2 with the biased variance
//   z = (x - mean) * (rstd * w) + b,  y = act(z)
// Backward of a given dy, with xh = (x - mean) * rstd and dz = dy * act'(z):
//   dw = sum dz * xh,  db = sum dz  (over samples and voxels)
//   A = mean over the group of dz * w,  B = mean over the group of dz * w * xh
//   dx = rstd * (dz * w - A - xh * B)
// Two passes over the data each way: sums, then the element-wise result (the statistics of a group need all of it).
// Both are bound by memory: forward 3, backward 5 activations read or written. Samples that fit the shared memory
// of a cluster take one. [4,24,64,128,128] bf16 with silu (201 MB): forward 108 us (5.6 TB/s), backward 173 us (5.8
// TB/s), with relu 100 us forward (6.0 TB/s); with x in 8 bits too 132 and 193 us, where neither the memory (3.3 to 4.0
// TB/s) nor the issue slots (60 to 65 %, 160 to 190 instructions a warp and vector) are full.
//
// A thread owns a vector of V neighbouring elements in every R-th row of its block's range, so its channels and with
// them the parameters stay in registers. A row is a voxel's channels, or L / C voxels together where C is no multiple
// of V (L = lcm(C, V)), so that odd channel counts still move 16 bytes at a time; what is left of a sample before its
// first whole vector and behind its last whole row (its edges) goes element by element. Rows wider than a block's
// threads are cut into channel tiles.
//
// Sums: a thread keeps sum (x - p) and sum (x - p)^2 in fp32 around its own first value p, so nothing cancels where
// |mean| >> std, and an outlier as p spoils one thread's few elements at most; backward sum dz and sum dz (x - mean).
// Threads, blocks and samples add in fp64, in a fixed order: same bits on every run.
#pragma once

#include <algorithm>

#include "r4c_internal.h"
#include "r4c_q8.cuh"

namespace r4c {
namespace gn {

constexpr int kThreads = 256;   // at most, per block
// Blocks that fit an SM beside each other (the registers that each kernel may take follow from it).
constexpr int kStatsBlocks = 4, kApplyBlocks = 4, kBwdBlocks = 3;
// Blocks an SM that each pass runs in. The forward's two and two fit beside each other, so the second pass has started
// when the sums end; short sums take one block an SM (fewer parts to join). Measured, sums 4 + y 4 / 2 + 4 / 2 + 2 / 1 + 2
// (us): [4,24,64,128,128] - / 104 / 101 / 110, [4,48,32,64,64] 26.7 / 24.0 / 23.2 / 24.3, [2,32,33,47,50] fp32 17.1 /
// 15.2 / 14.6 / 13.9, [2,30,37,41,53] 18.8 / 15.9 / 16.3 / 14.9. Backward, sums 3 / 2 / 1 with dx 3: [4,24,64,128,128] 170
// / 173 / 198, [4,48,32,64,64] 40 / 42 / 47, [2,32,33,47,50] 23.8 / 23.1 / 22.8, [3,40,21,35,45] kept 16.7 / 15.2 / 14.3.
constexpr int kStatsFit = 2, kApplyFit = 2, kBwdSumsFit = 3, kBwdFit = 3;
constexpr int64_t kShortSums = 48;   // tiles of rows an SM, below which sums are short
// Vectors of a thread on their way at a time, plus one.
constexpr int kFwdAhead = 8, kBwdAhead = 4;
// Samples that a cluster keeps on chip: vectors of a thread at most (forward; backward, which keeps dy too), groups of
// a channel tile at most.
constexpr int kSmallFwd = 16, kSmallBwd = 8, kSmallGroups = 256;

struct Geo {
  int64_t sample;    // elements of a sample, S * C
  int64_t rows;      // rows of L elements of a sample (with edges: of the longest)
  int64_t chunk;     // rows of a block, a multiple of R
  int64_t samples, blocks;   // blocks of one channel tile: samples * nb
  double inv_m;      // 1 / (Cg * S)
  float eps, slope;
  int act, pdtype, format;
  int L, C, G, Cg;
  int lanes;         // vectors of a row in a channel tile (L / V when there is one tile)
  int tiles;
  int R;             // rows that a block's threads cover at a time
  int chunk_tiles;   // chunk / R
  int nb;            // blocks of a sample and channel tile (the cluster's, where one keeps a sample)
  int edges;         // samples do not part into whole rows that start on a vector
  int np;            // parts of a sample's sums that the second pass reads: blocks of the first times channel tiles
  int wide_params;   // w and b are fp32 on 16 bytes, and a thread's channels follow each other
  int pack;          // the forward writes x in 8 bits too
  int small;         // vectors that a thread keeps in shared memory (small samples), or 0: two passes
};

// The same data in another number of blocks a sample.
inline Geo split(Geo g, int nb) {
  g.chunk = std::max<int64_t>(1, ((g.rows + nb - 1) / nb + g.R - 1) / g.R) * g.R;
  g.chunk_tiles = (int)(g.chunk / g.R);
  g.nb = (int)std::max<int64_t>(1, (g.rows + g.chunk - 1) / g.chunk);
  g.blocks = g.samples * g.nb;
  return g;
}

// V elements of T, moved as one word; in fp32 as pairs, for the packed arithmetic (two fp32 an instruction: half the
// issue slots, which bound these kernels before the memory does).
template <int V> constexpr int kPairs = (V + 1) / 2;

template <typename T, int V>
struct Vec {
  static constexpr int B = V * (int)sizeof(T);
  uint32_t w[B >= 4 ? B / 4 : 1];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (B >= 4 ? B / 4 : 1); ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (B == 16) {
      const uint4 r = *reinterpret_cast<const uint4*>(p);
      w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
    } else if constexpr (B == 8) {
      const uint2 r = *reinterpret_cast<const uint2*>(p);
      w[0] = r.x, w[1] = r.y;
    } else if constexpr (B == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (B == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (B == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (B == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  }
  __device__ __forceinline__ void to_f(float2 (&f)[kPairs<V>]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < V; ++k) (k & 1 ? f[k / 2].y : f[k / 2].x) = __uint_as_float(w[k]);
      if constexpr (V == 1) f[0].y = 0.f;
    } else if constexpr (V == 1) {
      const uint16_t h = (uint16_t)w[0];
      f[0] = make_float2(Elem<T>::to_f(*reinterpret_cast<const T*>(&h)), 0.f);
    } else {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        if constexpr (__is_same(T, __nv_bfloat16))
          f[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
        else
          f[k] = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      }
    }
  }
  __device__ __forceinline__ void from_f(const float2 (&f)[kPairs<V>]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < V; ++k) w[k] = __float_as_uint(k & 1 ? f[k / 2].y : f[k / 2].x);
    } else if constexpr (V == 1) {
      const T h = Elem<T>::from_f(f[0].x);
      w[0] = *reinterpret_cast<const uint16_t*>(&h);
    } else {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        if constexpr (__is_same(T, __nv_bfloat16)) {
          const __nv_bfloat162 h = __float22bfloat162_rn(f[k]);
          w[k] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __float22half2_rn(f[k]);
          w[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
  }
};

// The activation that a backward reads: x itself, or the values of its 8 bits.
template <typename T, int V, bool Q>
struct Source;
template <typename T, int V>
struct Source<T, V, false> {
  Vec<T, V> v;
  __device__ __forceinline__ void zero() { v.zero(); }
  __device__ __forceinline__ void load(const void* x, const uint8_t*, int64_t at) { v.load(static_cast<const T*>(x) + at); }
  __device__ __forceinline__ void to_f(int, float2 (&f)[kPairs<V>]) const { v.to_f(f); }
};
template <typename T, int V>
struct Source<T, V, true> {
  q8::Codes<V> c;
  int byte;
  __device__ __forceinline__ void zero() {
    c.w[0] = 0;
    if constexpr (V > 4) c.w[1] = 0;
    byte = 0;
  }
  __device__ __forceinline__ void load(const void* x, const uint8_t* exps, int64_t at) {
    c = q8::load_codes<V>(static_cast<const uint8_t*>(x) + at);
    byte = exps[at / q8::kBlock];
  }
  __device__ __forceinline__ void to_f(int format, float2 (&f)[kPairs<V>]) const {
    float e[V];
    q8::decode<T, V>(c, byte, format, e);
#pragma unroll
    for (int k = 0; k < kPairs<V>; ++k) f[k] = make_float2(e[2 * k], V > 1 ? e[V > 1 ? 2 * k + 1 : 0] : 0.f);
  }
};

__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// A copy of BYTES bytes into shared memory that runs beside the thread (two bytes, which the hardware has no such copy
// for, are moved at once).
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  } else if constexpr (BYTES >= 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
  } else if constexpr (BYTES == 2) {
    const uint16_t v = *static_cast<const uint16_t*>(from);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(v) : "memory");
  } else {
    const uint32_t v = *static_cast<const uint8_t*>(from);
    asm volatile("st.shared.u8 [%0], %1;" ::"r"(to), "r"(v) : "memory");
  }
}

// A thread's next vectors of x (and dy), D - 1 of them on their way in its own slots of shared memory: what the memory's
// latency needs in flight (some 100 KB an SM) costs no registers, and no thread waits for another. Slots are constants
// in loops unrolled by D, addresses are counted up: these kernels issue instructions two cycles out of three.
template <typename T, int V, bool Q, bool DY, int D>
struct Ring {
  static constexpr int XS = Q ? 1 : (int)sizeof(T), XB = V * XS, YB = V * (int)sizeof(T);
  static constexpr int kDy = D * kThreads * XB, kExp = kDy + (DY ? D * kThreads * YB : 0);
  static constexpr int kBytes = kExp + (Q ? D * kThreads * 4 : 0);
  const char *x, *dy;             // the next vector to start
  const uint8_t* exps;
  int64_t at, step;               // its element, and the elements from one to the next
  uint32_t got;                   // the element of the next vector to take, its low bits
  uint32_t slot;                  // this thread's first slots
  const char* mem;

  __device__ __forceinline__ Ring(char* smem, const void* x_, const T* dy_, const uint8_t* exps_, int64_t at_,
                                  int64_t step_) {
    at = at_;
    step = step_;
    x = static_cast<const char*>(x_) + at * XS;
    dy = DY ? reinterpret_cast<const char*>(dy_ + at) : nullptr;
    exps = exps_;
    got = (uint32_t)at;
    slot = shared_at(smem);
    mem = smem;
  }
  // starts the next vector into slot i, if the thread has it
  __device__ __forceinline__ void start(int i, bool has) {
    if (has) {
      copy_async<XB>(slot + (i * kThreads + threadIdx.x) * XB, x);
      if constexpr (DY) copy_async<YB>(slot + kDy + (i * kThreads + threadIdx.x) * YB, dy);
      if constexpr (Q)            // the word that holds the block's exponent
        copy_async<4>(slot + kExp + (i * kThreads + threadIdx.x) * 4, exps + (at / q8::kBlock & ~(int64_t)3));
    }
    x += step * XS;
    if constexpr (DY) dy += step * (int)sizeof(T);
    if constexpr (Q) at += step;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the oldest has landed (D - 2 were started after it)
  __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory"); }
  __device__ __forceinline__ void drain() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
  __device__ __forceinline__ void get(int i, Source<T, V, Q>& v) const {
    const char* p = mem + (i * kThreads + threadIdx.x) * XB;
    if constexpr (Q) {
      v.c = q8::load_codes<V>(reinterpret_cast<const uint8_t*>(p));
      const uint32_t w = *reinterpret_cast<const uint32_t*>(mem + kExp + (i * kThreads + threadIdx.x) * 4);
      v.byte = (int)__byte_perm(w, 0, 0x4440 | (got / q8::kBlock & 3));
    } else {
      v.v.load(reinterpret_cast<const T*>(p));
    }
  }
  __device__ __forceinline__ void get_dy(int i, Vec<T, V>& d) const {
    d.load(reinterpret_cast<const T*>(mem + kDy + (i * kThreads + threadIdx.x) * YB));
  }
  __device__ __forceinline__ void next() {
    if constexpr (Q) got += (uint32_t)step;
  }
};

__device__ __forceinline__ float param(const void* p, int dtype, int c, float none) {
  if (!p) return none;
  if (dtype == R4C_F32) return __ldg(static_cast<const float*>(p) + c);
  if (dtype == R4C_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
  return __half2float(static_cast<const __half*>(p)[c]);
}

__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / (1 + e^-z): for 16-bit results the hardware's exponential and reciprocal (relative error about 2^-21, the
// result's own half step is 2^-9 or 2^-12), the library's in full precision for fp32. (One reciprocal for two elements
// would let a neighbour's NaN, perhaps another group's, change the last bit.)
template <typename T>
__device__ __forceinline__ float2 sigmoid(float2 z) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(1.f / (1.f + expf(-z.x)), 1.f / (1.f + expf(-z.y)));
  } else {
    const float2 t = __fmul2_rn(z, two(-1.44269504f));
    const float2 e = __fadd2_rn(make_float2(ex2(t.x), ex2(t.y)), two(1.f));
    return make_float2(rcp(e.x), rcp(e.y));
  }
}

// erfc(u) e^(u^2) = c1 t + c2 t^2 + .. with t = 1 / (1 + p u), fitted here for the least relative error over u from 0 to
// 9.6: in fp32 arithmetic 2^-20 of itself with seven terms (16-bit results), 7 units of 2^-24 with nine (fp32 results).
// For v = u sqrt(2): p / sqrt(2), and half of each coefficient, the last first.
template <typename T> struct Erfc;
template <> struct Erfc<float> {
  static constexpr int kTerms = 9;
  static constexpr float kP = 0.26516503f;
  static __device__ __forceinline__ constexpr float c(int i) {
    constexpr float k[kTerms] = {0.0308482982f, -0.144037649f, 0.21694681f, -0.11553812f, 0.13742201f,
                                 0.0605195016f, 0.102715209f, 0.105316751f, 0.105807208f};
    return k[i];
  }
};
template <> struct Erfc<__half> {
  static constexpr int kTerms = 7;
  static constexpr float kP = 0.26382154f;
  static __device__ __forceinline__ constexpr float c(int i) {
    constexpr float k[kTerms] = {-0.0694223195f, 0.20446232f, -0.07747785f, 0.149382889f, 0.0801644474f, 0.107790627f,
                                 0.1050997f};
    return k[i];
  }
};
template <> struct Erfc<__nv_bfloat16> : Erfc<__half> {};

// Phi(z) and e^(-z^2/2). Left of 0 Phi is wanted relative to itself, so it is taken from erfc: Phi(-v) =
// erfc(v / sqrt(2)) / 2 (1 + erf would cancel: nothing of it is left from z = -5.6 in fp32). The same exponential serves
// both; with CUDA's erfcf in fp32 [2,32,33,47,50] took 17.4 us forward and 31.4 us for the gradients, now 14.0 and 20.5.
// Infinities and NaN: Phi is 1, 0 and NaN.
template <typename T>
__device__ __forceinline__ void normal(float2 z, float2& phi, float2& e) {
  if constexpr (sizeof(T) == 4) {
    e = make_float2(expf(-0.5f * z.x * z.x), expf(-0.5f * z.y * z.y));
  } else {
    const float2 q = __fmul2_rn(__fmul2_rn(z, z), two(-0.72134752f));
    e = make_float2(ex2(q.x), ex2(q.y));
  }
  const float2 d = __ffma2_rn(make_float2(fabsf(z.x), fabsf(z.y)), two(Erfc<T>::kP), two(1.f));
  const float2 t = make_float2(rcp(d.x), rcp(d.y));
  float2 p = two(Erfc<T>::c(0));
#pragma unroll
  for (int i = 1; i < Erfc<T>::kTerms; ++i) p = __ffma2_rn(p, t, two(Erfc<T>::c(i)));
  p = __fmul2_rn(__fmul2_rn(p, t), e);
  const float2 c = __ffma2_rn(p, two(-1.f), two(1.f));
  phi = make_float2(z.x < 0.f ? p.x : c.x, z.y < 0.f ? p.y : c.y);
}

// ACT: the activation, or -1: read from the descriptor, in kernels that also take samples with edges and narrow vectors
// (channels that are no multiple of a vector: rarer, so one kernel for all activations; the others stay lighter by the
// edges' code: 204 against 214 us for the gradients of [4,24,64,128,128] kept in 8 bits).
template <typename T, int ACT>
__device__ __forceinline__ float2 act_value(float2 z, float slope) {
  if constexpr (ACT == R4C_ACT_RELU) return make_float2(z.x <= 0.f ? 0.f : z.x, z.y <= 0.f ? 0.f : z.y);   // NaN stays
  if constexpr (ACT == R4C_ACT_LEAKY_RELU) {
    const float2 s = __fmul2_rn(z, two(slope));
    return make_float2(z.x <= 0.f ? s.x : z.x, z.y <= 0.f ? s.y : z.y);
  }
  if constexpr (ACT == R4C_ACT_SILU) return __fmul2_rn(z, sigmoid<T>(z));
  if constexpr (ACT == R4C_ACT_GELU) {
    float2 phi, e;
    normal<T>(z, phi, e);
    return __fmul2_rn(z, phi);
  }
  return z;
}
// dy * act'(z)
template <typename T, int ACT>
__device__ __forceinline__ float2 act_grad(float2 dy, float2 z, float slope) {
  if constexpr (ACT == R4C_ACT_RELU) return make_float2(z.x <= 0.f ? 0.f : dy.x, z.y <= 0.f ? 0.f : dy.y);
  if constexpr (ACT == R4C_ACT_LEAKY_RELU) {
    const float2 s = __fmul2_rn(dy, two(slope));
    return make_float2(z.x <= 0.f ? s.x : dy.x, z.y <= 0.f ? s.y : dy.y);
  }
  if constexpr (ACT == R4C_ACT_SILU) {
    const float2 s = sigmoid<T>(z);
    // s (1 + z (1 - s))
    return __fmul2_rn(__fmul2_rn(dy, s), __ffma2_rn(z, __ffma2_rn(s, two(-1.f), two(1.f)), two(1.f)));
  }
  if constexpr (ACT == R4C_ACT_GELU) {
    float2 phi, e;
    normal<T>(z, phi, e);
    return __fmul2_rn(dy, __ffma2_rn(__fmul2_rn(z, e), two(0.39894228f), phi));
  }
  return dy;
}
template <typename T, int ACT, int P>
__device__ __forceinline__ void act_values(float2 (&z)[P], int act, float slope) {
  if constexpr (ACT >= 0) {
#pragma unroll
    for (int k = 0; k < P; ++k) z[k] = act_value<T, ACT>(z[k], slope);
  } else {
    switch (act) {
      case R4C_ACT_RELU: act_values<T, R4C_ACT_RELU>(z, act, slope); break;
      case R4C_ACT_LEAKY_RELU: act_values<T, R4C_ACT_LEAKY_RELU>(z, act, slope); break;
      case R4C_ACT_SILU: act_values<T, R4C_ACT_SILU>(z, act, slope); break;
      case R4C_ACT_GELU: act_values<T, R4C_ACT_GELU>(z, act, slope); break;
    }
  }
}
// dy becomes dy * act'(z)
template <typename T, int ACT, int P>
__device__ __forceinline__ void act_grads(float2 (&dy)[P], const float2 (&z)[P], int act, float slope) {
  if constexpr (ACT >= 0) {
#pragma unroll
    for (int k = 0; k < P; ++k) dy[k] = act_grad<T, ACT>(dy[k], z[k], slope);
  } else {
    switch (act) {
      case R4C_ACT_RELU: act_grads<T, R4C_ACT_RELU>(dy, z, act, slope); break;
      case R4C_ACT_LEAKY_RELU: act_grads<T, R4C_ACT_LEAKY_RELU>(dy, z, act, slope); break;
      case R4C_ACT_SILU: act_grads<T, R4C_ACT_SILU>(dy, z, act, slope); break;
      case R4C_ACT_GELU: act_grads<T, R4C_ACT_GELU>(dy, z, act, slope); break;
    }
  }
}

// Where a block's threads stand: sample n, part b of it, channel tile, and a thread's lane and row. A thread's rows are
// row, row + R, .. of the block's rows: one in each of the first `mine` of its `tiles` tiles of R rows. Divisions by
// run-time sizes cost tens of instructions, which a short kernel feels: each thread makes two, the rest is counted up.
struct Place {
  int64_t n;
  int64_t at;           // the thread's first element
  int64_t step;         // elements from one tile of rows to the next
  int tiles, mine;
  int b, tile, lane, row;
  int j0, j1;           // the channel tile's elements of a row
  int c, gi, in_group;  // the thread's first channel, its group and its place there
  int shift;            // the channel of a row's first element
  int ga, gb;           // the channel tile's groups
  bool active;
};
template <int V>
__device__ __forceinline__ Place place(const Geo& g) {
  Place p;
  if (g.nb == 1) {
    p.n = blockIdx.x;
    p.b = 0;
  } else {
    const unsigned n = blockIdx.x / (unsigned)g.nb;
    p.n = n;
    p.b = (int)(blockIdx.x - n * g.nb);
  }
  p.tile = blockIdx.y;
  p.row = (int)(threadIdx.x / (unsigned)g.lanes);
  p.lane = (int)threadIdx.x - p.row * g.lanes;
  p.j0 = p.tile * g.lanes * V;
  p.j1 = min(p.j0 + g.lanes * V, g.L);
  const int j = p.j0 + p.lane * V;
  p.active = p.row < g.R && j < p.j1;
  int64_t first = p.n * g.sample, rows = g.rows;
  p.shift = 0;
  if (g.edges) {
    const int head = (int)(-first & (V - 1));
    p.shift = head < g.C ? head : head % g.C;
    first += head;
    if (g.sample - head < rows * g.L) --rows;
  }
  p.c = g.L == g.C ? j : (int)((unsigned)(j + p.shift) % (unsigned)g.C);
  p.gi = (int)((unsigned)p.c / (unsigned)g.Cg);
  p.in_group = p.c - p.gi * g.Cg;
  if (g.tiles == 1) {
    p.ga = 0;
    p.gb = g.G;
  } else {
    p.ga = (int)((unsigned)p.j0 / (unsigned)g.Cg);
    p.gb = (int)((unsigned)(p.j1 - 1) / (unsigned)g.Cg) + 1;
  }
  const int64_t r0 = p.b * g.chunk;
  const int64_t left = min(g.chunk, rows - r0);
  p.tiles = left == g.chunk ? g.chunk_tiles : left > 0 ? (int)((left + g.R - 1) / g.R) : 0;
  const int64_t last = left - (int64_t)(p.tiles - 1) * g.R;    // rows of the last tile
  p.mine = p.active ? p.tiles - (p.row < last ? 0 : 1) : 0;
  if (p.mine < 0) p.mine = 0;
  p.at = first + (r0 + p.row) * g.L + j;
  p.step = (int64_t)g.R * g.L;
  return p;
}

// A sample's edges, which its first block works on: elements [first, first + head) and [tail_at, tail_at + tail).
struct Edges {
  int64_t first, tail_at;
  int head, tail, tail_c;   // tail_c: the tail's first channel
  template <int V>
  static __device__ __forceinline__ Edges of(const Geo& g, const Place& p) {
    Edges e;
    e.first = p.n * g.sample;
    e.head = (int)(-e.first & (V - 1));
    if (e.head > g.sample) e.head = (int)g.sample;
    int64_t rows = g.rows;
    if (g.sample - e.head < rows * g.L) --rows;
    const int64_t inside = e.head + (rows > 0 ? rows * g.L : 0);
    e.tail_at = e.first + inside;
    e.tail = (int)(g.sample - inside);
    e.tail_c = (int)(inside % g.C);
    return e;
  }
  // f(element) for those of channel c
  template <typename F>
  __device__ __forceinline__ void each_of(const Geo& g, int c, F f) const {
    for (int i = c; i < head; i += g.C) f(first + i);
    for (int i = c >= tail_c ? c - tail_c : c - tail_c + g.C; i < tail; i += g.C) f(tail_at + i);
  }
  // f(element, channel) for this thread's share of all
  template <typename F>
  __device__ __forceinline__ void each(const Geo& g, F f) const {
    for (int i = threadIdx.x; i < head + tail; i += blockDim.x) {
      if (i < head) f(first + i, i % g.C);
      else f(tail_at + (i - head), (tail_c + (i - head)) % g.C);
    }
  }
};

// f(column k of the thread, its channel, its group) for its V columns, in order.
template <int V, typename F>
__device__ __forceinline__ void each_column(const Geo& g, const Place& p, F f) {
  int c = p.c, gi = p.gi, in = p.in_group;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    f(k, c, gi);
    ++c;
    if (++in == g.Cg) {
      in = 0;
      ++gi;
    }
    if (c == g.C) c = gi = in = 0;
  }
}
__device__ __forceinline__ void put(float2* f, int k, float v) { (k & 1 ? f[k / 2].y : f[k / 2].x) = v; }

// Neighbouring threads for each of `items` sums: the largest power of two that the block has, at most a warp.
__device__ __forceinline__ int threads_per(int items, int threads) {
  int t = 32;
  while (t > 1 && t * items > threads) t >>= 1;
  return t;
}
template <typename S>
__device__ __forceinline__ void join(S& a, S& b, int width) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o < width) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }
}

// f(item, sub, tp, a, c) adds the terms of item that are thread `sub`'s of `tp`; out(item, a, c) gets the sums. Every
// thread of the block calls it (the shuffles need whole warps; blocks are multiples of 32 threads).
template <typename S, typename F, typename Out>
__device__ __forceinline__ void each_sum(int items, F f, Out out) {
  const int tp = threads_per(items, blockDim.x), sub = threadIdx.x & (tp - 1);
  const int first = threadIdx.x / tp, per = blockDim.x / tp;    // (tp is a power of two)
  for (int base = 0; base < items; base += per) {
    const int i = base + first;
    S a = 0, c = 0;
    if (i < items) f(i, sub, tp, a, c);
    join(a, c, tp);
    if (i < items && sub == 0) out(i, a, c);
  }
}
// each_sum's threads of an item shared out over columns and rows of a table: the rows' share.
__device__ __forceinline__ int row_threads(int tp, int rows) {
  int t = 1;
  while (2 * t <= tp && 2 * t <= rows) t *= 2;
  return t;
}

// Launched while the kernel before it may still run: what that one wrote may be read from here on.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// What the kernel before this one wrote, while this one may already have run: the pointers are not __restrict__ (which
// would promise that nothing changes it) and the loads are volatile, so that none goes ahead of the wait, which makes all
// that was written visible. (Loads past the L1, ld.relaxed.gpu, take the parameters' sums 4 us longer at [4,48,32,64,64]:
// neighbouring channels share sectors.)
__device__ __forceinline__ double2 from_previous(const double2* p) {
  double2 v;
  asm volatile("ld.global.v2.f64 {%0, %1}, [%2];" : "=d"(v.x), "=d"(v.y) : "l"(p) : "memory");
  return v;
}
// Adds p[i * stride] for i = first, first + step, .. below end, in that order, U loads on their way at a time.
template <int U>
__device__ __forceinline__ void add_previous(const double2* p, int64_t first, int64_t step, int64_t end, int64_t stride, double& a,
                                             double& c) {
  for (int64_t i = first; i < end; i += U * step) {
    double2 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = make_double2(0.0, 0.0);
      if (i + u * step < end) v[u] = from_previous(p + (i + u * step) * stride);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a += v[u].x;
      c += v[u].y;
    }
  }
}

// The thread's parameters: z = (x - mean) * a + b with a = rstd * w. The mean is not taken into b, in 16-bit types neither:
// 2^-24 of |mean| a is not small against xh where a group has next to no spread, and sums of dz * x would cancel against
// mean * sum dz. w and b do not wait for the statistics.
// SHARED: the means' negatives lie in shared memory, per column, and are read for each vector (for the gradients of
// vectors of 8, whose registers would spill: [4,24,64,128,128] bf16 silu 175 us in registers, 170 so, kept in 8 bits 232
// and 193).
template <int V> constexpr bool kSharedMeans = V == 8;
template <typename T, int V, bool SHARED = false>
struct Affine {
  float2 nmu[SHARED ? 1 : kPairs<V>], a[kPairs<V>], b[kPairs<V>];
  float4* means;         // SHARED: the thread's columns'; threads of row 0 write them
  __device__ __forceinline__ void params(const Geo& g, const Place& p, const void* gamma, const void* beta) {
#pragma unroll
    for (int k = 0; k < kPairs<V>; ++k) {
      if constexpr (!SHARED) nmu[k] = two(0.f);
      b[k] = two(0.f);
      a[k] = two(1.f);
    }
    if (!p.active) return;
    if (V % 4 == 0 && g.wide_params) {          // fp32, on 16 bytes, channels without a wrap
#pragma unroll
      for (int k = 0; k < V / 4; ++k) {
        if (gamma) {
          const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(gamma) + p.c) + k);
          a[2 * k] = make_float2(v.x, v.y);
          a[2 * k + 1] = make_float2(v.z, v.w);
        }
        if (beta) {
          const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(beta) + p.c) + k);
          b[2 * k] = make_float2(v.x, v.y);
          b[2 * k + 1] = make_float2(v.z, v.w);
        }
      }
    } else {
      each_column<V>(g, p, [&](int k, int c, int) {
        put(a, k, param(gamma, g.pdtype, c, 1.f));
        put(b, k, param(beta, g.pdtype, c, 0.f));
      });
    }
  }
  template <typename Stat>
  __device__ __forceinline__ void stats(const Geo& g, const Place& p, Stat stat) {
    if (!p.active) return;
    float2 r[kPairs<V>];
    if constexpr (V == 1) r[0] = two(0.f);
    float2 q = make_float2(0.f, 0.f);
    int have = -1;
    each_column<V>(g, p, [&](int k, int, int gi) {
      if (gi != have) q = stat(gi);
      have = gi;
      if constexpr (!SHARED) put(nmu, k, -q.x);
      else if (p.row == 0) reinterpret_cast<float*>(means)[k] = -q.x;
      put(r, k, q.y);
    });
#pragma unroll
    for (int k = 0; k < kPairs<V>; ++k) a[k] = __fmul2_rn(a[k], r[k]);
  }
  // x becomes x - mean; z of it
  __device__ __forceinline__ float2 z(int k, float2& x) const {
    if constexpr (SHARED) {
      const float4 m = means[k / 2];
      x = __fadd2_rn(x, k & 1 ? make_float2(m.z, m.w) : make_float2(m.x, m.y));
    } else {
      x = __fadd2_rn(x, nmu[k]);
    }
    return __ffma2_rn(x, a[k], b[k]);
  }
};

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
// A thread's sums around its first value.
template <typename T, int V>
struct Moments {
  float2 np[kPairs<V>], s1[kPairs<V>], s2[kPairs<V>];
  int count;
  __device__ __forceinline__ void zero() {
    count = 0;
#pragma unroll
    for (int k = 0; k < kPairs<V>; ++k) np[k] = s1[k] = s2[k] = two(0.f);
  }
  __device__ __forceinline__ void pivot(const Vec<T, V>& v) {
    v.to_f(np);
#pragma unroll
    for (int k = 0; k < kPairs<V>; ++k) np[k] = __fmul2_rn(np[k], two(-1.f));
  }
  __device__ __forceinline__ void add(const Vec<T, V>& v) {
    float2 f[kPairs<V>];
    v.to_f(f);
    ++count;
#pragma unroll
    for (int k = 0; k < kPairs<V>; ++k) {
      const float2 d = __fadd2_rn(f[k], np[k]);
      s1[k] = __fadd2_rn(s1[k], d);
      s2[k] = __ffma2_rn(d, d, s2[k]);
    }
  }
  // (sum x - o, sum (x - o)^2) of column k in fp64
  __device__ __forceinline__ double2 sums(int k, double o) const {
    const double q = -(double)(k & 1 ? np[k / 2].y : np[k / 2].x) - o, a = k & 1 ? s1[k / 2].y : s1[k / 2].x;
    const double s = k & 1 ? s2[k / 2].y : s2[k / 2].x, c = count;
    return make_double2(c * q + a, s + 2.0 * q * a + c * q * q);
  }
};

// A group's origin in a sample: its first element. Sums are joined about it, so that fp64 keeps a variance far below
// mean^2 (about zero, a group that is 30000 throughout had one of some 1e-7 instead of 0, against an eps of 1e-5).
template <typename T>
__device__ __forceinline__ float origin(const Geo& g, const Place& p, const T* __restrict__ x, int gi) {
  return Elem<T>::to_f(x[p.n * g.sample + (int64_t)gi * g.Cg]);
}

// The block's sums of each of its groups: out(group, sum x - o, sum (x - o)^2), o = origin_of(group of the tile).
template <typename T, int V, typename Origin, typename Out>
__device__ __forceinline__ void block_moments(const Geo& g, const Place& p, const Moments<T, V>& m,
                                              const T* __restrict__ x, double2* __restrict__ red, Origin origin_of,
                                              Out out) {
  // a thread whose columns all belong to one group adds them first
  const bool merged = V > 1 && g.L == g.C && (g.Cg & (V - 1)) == 0;
  if (p.active) {
    if (merged) {
      const double o = origin_of(p.gi - p.ga);
      double2 t = m.sums(0, o);
#pragma unroll
      for (int k = 1; k < V; ++k) {
        const double2 v = m.sums(k, o);
        t.x += v.x;
        t.y += v.y;
      }
      red[threadIdx.x] = t;
    } else {
      each_column<V>(g, p, [&](int k, int, int gi) { red[k * kThreads + threadIdx.x] = m.sums(k, origin_of(gi - p.ga)); });
    }
  }
  __syncthreads();
  const int tp = threads_per(p.gb - p.ga, blockDim.x), tr = row_threads(tp, g.R), tc = tp / tr;
  each_sum<double>(p.gb - p.ga, [&](int i, int sub, int, double& a, double& c) {
    const int gi = p.ga + i, sr = sub & (tr - 1), sc = sub / tr;
    int lo = gi * g.Cg, hi = lo + g.Cg;
    if (g.tiles > 1) {
      lo = max(lo, p.j0) - p.j0;
      hi = min(hi, p.j1) - p.j0;
    }
    if (merged) {
      for (int l = lo / V + sc; l < hi / V; l += tc)
        for (int r = sr; r < g.R; r += tr) {
          const double2 v = red[r * g.lanes + l];
          a += v.x;
          c += v.y;
        }
    } else {
      for (int base = 0; base < g.L; base += g.C)         // once, unless a row holds several voxels
        for (int ch = lo + sc; ch < hi; ch += tc) {
          const int j = base + (ch >= p.shift ? ch - p.shift : ch - p.shift + g.C);
          for (int r = sr; r < g.R; r += tr) {
            const double2 v = red[(j % V) * kThreads + r * g.lanes + j / V];
            a += v.x;
            c += v.y;
          }
        }
    }
    if (g.edges && p.b == 0) {
      const Edges e = Edges::of<V>(g, p);
      const double o = origin_of(i);
      for (int ch = lo + sub; ch < hi; ch += tp)
        e.each_of(g, ch, [&](int64_t at) {
          const double v = Elem<T>::to_f(x[at]) - o;
          a += v;
          c += v * v;
        });
    }
  }, [&](int i, double a, double c) { out(p.ga + i, a, c); });
}

// Mean and rstd from the sums about the group's origin; (var + eps)^-1/2 from the fp32 reciprocal root and one step of
// Newton's method in fp64 (2^-22 becomes 2^-43; an fp64 root and division would be a hundred instructions in a row).
__device__ __forceinline__ float2 mean_rstd_of(const Geo& g, double a, double c, double o) {
  const double from_o = a * g.inv_m, mean = o + from_o;
  double var = c * g.inv_m - from_o * from_o;
  if (var < 0.0) var = 0.0;
  const double v = var + (double)g.eps;
  const float f = (float)v, r0 = rsqrtf(f);
  if (!(f >= 1e-30f && f <= 1e30f)) return make_float2((float)mean, (float)(1.0 / sqrt(v)));
  const double r = r0;
  return make_float2((float)mean, (float)(r * (1.5 - 0.5 * v * r * r)));
}

// part[((n * nb + b) * tiles + tile) * G + g] = (sum x - o, sum (x - o)^2) of the block's share of group g.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, kStatsBlocks) stats_kernel(const T* __restrict__ x,
                                                                       const __grid_constant__ Geo g,
                                                                       double2* __restrict__ part) {
  using R = Ring<T, V, false, false, kFwdAhead>;
  __shared__ __align__(16) char smem[R::kBytes > V * kThreads * 16 ? R::kBytes : V * kThreads * 16];
  __shared__ float origins[V * kThreads];     // of the tile's groups, no more than its columns
  let_next_start();
  const Place p = place<V>(g);
  R ring(smem, x, nullptr, nullptr, p.at, p.step);
#pragma unroll
  for (int i = 0; i < kFwdAhead - 1; ++i) ring.start(i, i < p.mine);
  for (int i = threadIdx.x; i < p.gb - p.ga; i += blockDim.x) origins[i] = origin(g, p, x, p.ga + i);
  Moments<T, V> m;
  m.zero();
  if (p.mine > 0) {
    Vec<T, V> a;
    a.load(x + p.at);
    m.pivot(a);
  }
#pragma unroll 1
  for (int t = 0; t < p.mine; t += kFwdAhead) {
#pragma unroll
    for (int i = 0; i < kFwdAhead; ++i) {
      if (t + i >= p.mine) break;
      Source<T, V, false> a;
      ring.wait();
      ring.get(i, a);
      ring.start((i + kFwdAhead - 1) % kFwdAhead, t + i + kFwdAhead - 1 < p.mine);
      m.add(a.v);
    }
  }
  ring.drain();
  __syncthreads();
  double2* out = part + ((int64_t)blockIdx.x * g.tiles + p.tile) * g.G;
  if (g.tiles > 1)
    for (int i = threadIdx.x; i < g.G; i += blockDim.x)
      if (i < p.ga || i >= p.gb) out[i] = make_double2(0.0, 0.0);
  block_moments<T, V>(g, p, m, x, reinterpret_cast<double2*>(smem), [&](int i) { return origins[i]; },
                      [&](int gi, double a, double c) { out[gi] = make_double2(a, c); });
}

// y of one vector at element `at`, into `to`, and its 8 bits (PACK: a block of 32 elements lies in 32 / V neighbouring
// threads, all with or all without a row here; every thread of the warp calls it).
template <typename T, int V, int ACT, bool PACK>
__device__ __forceinline__ void apply_one(const Vec<T, V>& v, const Affine<T, V>& k, const Geo& g, bool in, int64_t at,
                                          T* __restrict__ to, uint8_t* __restrict__ codes,
                                          uint8_t* __restrict__ exps) {
  float2 f[kPairs<V>];
  v.to_f(f);
  if constexpr (PACK) {
    float e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = i & 1 ? f[i / 2].y : f[i / 2].x;
    bool finite;
    const int byte = q8::exponent_byte(q8::block_amax<T>(v.w, 0xffffffffu, &finite), g.format);
    const q8::Codes<V> c = q8::encode<V>(e, byte, g.format, finite);
    if (in) {
      q8::store_codes<V>(codes + at, c);
      if (((uint32_t)at & (q8::kBlock - 1)) == 0) exps[at / q8::kBlock] = (uint8_t)byte;
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) f[i] = k.z(i, f[i]);
  act_values<T, ACT>(f, g.act, g.slope);
  Vec<T, V> r;
  r.from_f(f);
  if (in) r.store(to);
}

// y of a sample's edges.
template <typename T, int V, int ACT, typename Stat>
__device__ __forceinline__ void apply_edges(const Geo& g, const Place& p, const T* __restrict__ x, const void* gamma,
                                            const void* beta, T* __restrict__ y, Stat stat) {
  Edges::of<V>(g, p).each(g, [&](int64_t at, int c) {
    const float2 s = stat((int)((unsigned)c / (unsigned)g.Cg));
    float2 z[1] = {two(fmaf(Elem<T>::to_f(x[at]) - s.x, s.y * param(gamma, g.pdtype, c, 1.f),
                            param(beta, g.pdtype, c, 0.f)))};
    act_values<T, ACT>(z, g.act, g.slope);
    y[at] = Elem<T>::from_f(z[0].x);
  });
}

// From the last row to the first: what the sums read last is what the L2 cache still has.
template <typename T, int V, int ACT, bool PACK>
__global__ void __launch_bounds__(kThreads, kApplyBlocks) apply_kernel(
    const T* __restrict__ x, const void* __restrict__ gamma, const void* __restrict__ beta,
    const __grid_constant__ Geo g, const double2* part, float2* __restrict__ mean_rstd,
    T* __restrict__ y, uint8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  using R = Ring<T, V, false, false, kFwdAhead>;
  extern __shared__ __align__(16) char smem[];
  float2* stat = reinterpret_cast<float2*>(smem + R::kBytes);
  const Place p = place<V>(g);
  // (x is older than the kernel before this one)
  const int skip = p.tiles - p.mine;       // 1 for a thread without a row in the last tile
  int64_t at = p.at + (p.tiles - 1) * p.step;
  T* to = y + at;
  R ring(smem, x, nullptr, nullptr, at, -p.step);
#pragma unroll
  for (int i = 0; i < kFwdAhead - 1; ++i) ring.start(i, i >= skip && i < p.tiles);
  Affine<T, V> k;
  k.params(g, p, gamma, beta);
  for (int i = threadIdx.x; i < p.gb - p.ga; i += blockDim.x) stat[i].x = origin(g, p, x, p.ga + i);
  __syncthreads();
  wait_for_previous();
  const double2* src = part + p.n * g.np * g.G + p.ga;
  each_sum<double>(p.gb - p.ga, [&](int i, int sub, int tp, double& a, double& c) {
    add_previous<4>(src + i, sub, tp, g.np, g.G, a, c);
  }, [&](int i, double a, double c) { stat[i] = mean_rstd_of(g, a, c, stat[i].x); });
  __syncthreads();
  if (p.b == 0)
    for (int i = threadIdx.x; i < p.gb - p.ga; i += blockDim.x) mean_rstd[p.n * g.G + p.ga + i] = stat[i];
  k.stats(g, p, [&](int gi) { return stat[gi - p.ga]; });
#pragma unroll 1
  for (int t = 0; t < p.tiles; t += kFwdAhead) {
#pragma unroll
    for (int i = 0; i < kFwdAhead; ++i) {
      if (t + i >= p.tiles) break;
      const bool in = t + i >= skip;
      Source<T, V, false> v;
      ring.wait();
      if (PACK) v.zero();
      if (in) ring.get(i, v);
      const int next = t + i + kFwdAhead - 1;
      ring.start((i + kFwdAhead - 1) % kFwdAhead, next >= skip && next < p.tiles);
      if (PACK || in) apply_one<T, V, ACT, PACK>(v.v, k, g, in, at, to, codes, exps);
      at -= p.step;
      to -= p.step;
    }
  }
  if (ACT < 0 && g.edges && p.b == 0) apply_edges<T, V, ACT>(g, p, x, gamma, beta, y, [&](int gi) { return stat[gi - p.ga]; });
}

// ---------------------------------------------------------------------------
// Backward: sums
// ---------------------------------------------------------------------------
// dz and x - mean of one vector.
template <typename T, int V, int ACT, bool Q, bool SHARED>
__device__ __forceinline__ void grad_one(const Source<T, V, Q>& v, const Vec<T, V>& d, const Affine<T, V, SHARED>& k,
                                         const Geo& g,
                                         float2 (&xm)[kPairs<V>], float2 (&dz)[kPairs<V>]) {
  v.to_f(g.format, xm);
  d.to_f(dz);
  float2 z[kPairs<V>];
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) z[i] = k.z(i, xm[i]);
  act_grads<T, ACT>(dz, z, g.act, g.slope);
}

// dz and x - mean of one element of channel c.
template <typename T, int ACT, bool Q>
__device__ __forceinline__ float2 grad_edge(const Geo& g, const T* __restrict__ dy, const void* __restrict__ x,
                                            const uint8_t* __restrict__ exps, const void* gamma, const void* beta,
                                            int64_t at, int c, float2 stat) {
  Source<T, 1, Q> v;
  float2 xm[1], dz[1] = {make_float2(Elem<T>::to_f(dy[at]), 0.f)};
  v.load(x, exps, at);
  v.to_f(g.format, xm);
  const float a = stat.y * param(gamma, g.pdtype, c, 1.f), b = param(beta, g.pdtype, c, 0.f);
  xm[0].x -= stat.x;
  const float2 z[1] = {make_float2(fmaf(xm[0].x, a, b), 0.f)};
  act_grads<T, ACT>(dz, z, g.act, g.slope);
  return make_float2(dz[0].x, xm[0].x);
}

// The block's (sum dz, sum dz * (x - mean)) of a thread's columns: cpart gets them per channel (the second times rstd),
// out(group, ..) the same times w, summed over the tile's channels of the group.
// edge(element, channel, stat): an edge's dz and x - mean. A thread's sums are fp32, everything from there on is fp64:
// sums that nearly vanish would be left with the roundings of the parts.
template <int V, bool EDGES, typename Stat, typename Edge, typename Out>
__device__ __forceinline__ void block_grads(const Geo& g, const Place& p, const float2 (&s1)[kPairs<V>],
                                            const float2 (&s2)[kPairs<V>], const void* gamma, float2* __restrict__ red,
                                            double2* __restrict__ cols, double2* __restrict__ cpart, Stat stat, Edge edge,
                                            Out out) {
#pragma unroll
  for (int k = 0; k < V; ++k)
    red[k * kThreads + threadIdx.x] = k & 1 ? make_float2(s1[k / 2].y, s2[k / 2].y) : make_float2(s1[k / 2].x, s2[k / 2].x);
  __syncthreads();
  const int nch = g.tiles == 1 ? g.C : p.j1 - p.j0;
  each_sum<double>(nch, [&](int i, int sub, int tp, double& a, double& c) {
    for (int j = i >= p.shift ? i - p.shift : i - p.shift + g.C; j < (g.tiles == 1 ? g.L : nch); j += g.C)
      for (int r = sub; r < g.R; r += tp) {
        const float2 v = red[(j % V) * kThreads + r * g.lanes + j / V];
        a += v.x;
        c += v.y;
      }
    if (EDGES && g.edges && p.b == 0 && sub == 0) {
      const float2 s = stat((int)((unsigned)i / (unsigned)g.Cg));
      Edges::of<V>(g, p).each_of(g, i, [&](int64_t at) {
        const float2 e = edge(at, i, s);
        a += e.x;
        c = fma((double)e.x, (double)e.y, c);
      });
    }
  }, [&](int i, double a, double c) {
    const int ch = p.j0 + i;
    const float2 m = stat((int)((unsigned)ch / (unsigned)g.Cg));
    const double2 s = make_double2(a, c * m.y);
    cols[i] = s;
    cpart[(int64_t)blockIdx.x * g.C + ch] = s;
  });
  __syncthreads();
  each_sum<double>(p.gb - p.ga, [&](int i, int sub, int tp, double& a, double& c) {
    const int lo = max((p.ga + i) * g.Cg, p.j0), hi = min((p.ga + i + 1) * g.Cg, p.j0 + nch);
    for (int ch = lo + sub; ch < hi; ch += tp) {
      const double w = param(gamma, g.pdtype, ch, 1.f);
      a = fma(w, cols[ch - p.j0].x, a);
      c = fma(w, cols[ch - p.j0].y, c);
    }
  }, [&](int i, double a, double c) { out(p.ga + i, a, c); });
}

// cpart[(n * nb + b) * C + c] = (sum dz, sum dz * xh) of the block's rows, and
// gpart[((n * nb + b) * tiles + tile) * G + g] = the same times w, summed over the tile's channels of the group.
template <typename T, int V, int ACT, bool Q>
__global__ void __launch_bounds__(kThreads, kBwdBlocks) bwd_sums_kernel(
    const T* __restrict__ dy, const void* __restrict__ x, const uint8_t* __restrict__ exps,
    const float2* __restrict__ mean_rstd, const void* __restrict__ gamma, const void* __restrict__ beta,
    const __grid_constant__ Geo g, double2* __restrict__ cpart, double2* __restrict__ gpart) {
  using R = Ring<T, V, Q, true, kBwdAhead>;
  constexpr int kTable = V * kThreads * (int)sizeof(float2);
  constexpr int kLoop = R::kBytes + (kSharedMeans<V> ? V * kThreads * (int)sizeof(float) : 0);
  __shared__ __align__(16) char smem[kLoop > 3 * kTable ? kLoop : 3 * kTable];
  let_next_start();
  const Place p = place<V>(g);
  R ring(smem, x, dy, exps, p.at, p.step);
#pragma unroll
  for (int i = 0; i < kBwdAhead - 1; ++i) ring.start(i, i < p.mine);
  const float2* stats = mean_rstd + p.n * g.G;
  Affine<T, V, kSharedMeans<V>> k;
  k.means = reinterpret_cast<float4*>(smem + R::kBytes) + p.lane * (V / 4);
  k.params(g, p, gamma, beta);
  k.stats(g, p, [&](int gi) { return stats[gi]; });
  if constexpr (kSharedMeans<V>) __syncthreads();
  float2 a1[kPairs<V>], a2[kPairs<V>];
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) a1[i] = a2[i] = two(0.f);
#pragma unroll 1
  for (int t = 0; t < p.mine; t += kBwdAhead) {
#pragma unroll
    for (int i = 0; i < kBwdAhead; ++i) {
      if (t + i >= p.mine) break;
      Source<T, V, Q> v;
      Vec<T, V> d;
      ring.wait();
      ring.get(i, v);
      ring.get_dy(i, d);
      ring.next();
      ring.start((i + kBwdAhead - 1) % kBwdAhead, t + i + kBwdAhead - 1 < p.mine);
      float2 xm[kPairs<V>], dz[kPairs<V>];
      grad_one<T, V, ACT, Q>(v, d, k, g, xm, dz);
#pragma unroll
      for (int j = 0; j < kPairs<V>; ++j) {
        a1[j] = __fadd2_rn(a1[j], dz[j]);
        a2[j] = __ffma2_rn(dz[j], xm[j], a2[j]);
      }
    }
  }
  ring.drain();
  __syncthreads();
  double2* out = gpart + ((int64_t)blockIdx.x * g.tiles + p.tile) * g.G;
  if (g.tiles > 1)
    for (int i = threadIdx.x; i < g.G; i += blockDim.x)
      if (i < p.ga || i >= p.gb) out[i] = make_double2(0.0, 0.0);
  block_grads<V, (ACT < 0)>(g, p, a1, a2, gamma, reinterpret_cast<float2*>(smem), reinterpret_cast<double2*>(smem + kTable), cpart,
                 [&](int gi) { return stats[gi]; },
                 [&](int64_t at, int c, float2 s) { return grad_edge<T, ACT, Q>(g, dy, x, exps, gamma, beta, at, c, s); },
                 [&](int gi, double a, double c) { out[gi] = make_double2(a, c); });
}

// ---------------------------------------------------------------------------
// Backward: dx, and the gradients of weight and bias
// ---------------------------------------------------------------------------
// dw, db: a warp, or a block, sums a channel over the (sample, block) parts, in a fixed order.
constexpr int64_t kWideParts = 2048;      // from here on a block a channel (70,000 parts of 16 channels: 160 -> 21 us)
__device__ __forceinline__ void param_grads(const double2* cpart, int64_t parts, int C, int c,
                                            float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int lane = threadIdx.x & 31;
  double u = 0.0, v = 0.0;
  add_previous<8>(cpart + c, lane, 32, parts, C, u, v);
  join(u, v, 32);
  if (lane == 0) {
    if (dbeta) dbeta[c] = (float)u;
    if (dgamma) dgamma[c] = (float)v;
  }
}
inline __global__ void __launch_bounds__(kThreads) params_kernel(const double2* cpart, int64_t parts, int C,
                                                                 float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ double2 warps[kThreads / 32];
  wait_for_previous();
  if (parts < kWideParts) {
    const int c = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    if (c < C) param_grads(cpart, parts, C, c, dgamma, dbeta);
    return;
  }
  const int c = blockIdx.x;
  double u = 0.0, v = 0.0;
  add_previous<8>(cpart + c, threadIdx.x, kThreads, parts, C, u, v);
  join(u, v, 32);
  if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = make_double2(u, v);
  __syncthreads();
  if (threadIdx.x == 0) {
    u = v = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) {
      u += warps[i].x;
      v += warps[i].y;
    }
    if (dbeta) dbeta[c] = (float)u;
    if (dgamma) dgamma[c] = (float)v;
  }
}

// dx of one vector; k1, k2: rstd * A, rstd^2 * B.
template <typename T, int V, int ACT, bool Q, bool SHARED>
__device__ __forceinline__ Vec<T, V> dx_one(const Source<T, V, Q>& v, const Vec<T, V>& d, const Affine<T, V, SHARED>& k,
                                            const float2 (&k1)[kPairs<V>], const float2 (&k2)[kPairs<V>], const Geo& g) {
  float2 xm[kPairs<V>], dz[kPairs<V>];
  grad_one<T, V, ACT, Q>(v, d, k, g, xm, dz);
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i)
    dz[i] = __ffma2_rn(dz[i], k.a[i], __fmul2_rn(__ffma2_rn(xm[i], k2[i], k1[i]), two(-1.f)));
  Vec<T, V> r;
  r.from_f(dz);
  return r;
}

// The thread's rstd * A and rstd^2 * B from its groups'.
template <int V>
__device__ __forceinline__ void thread_coef(const Geo& g, const Place& p, const float2* coef, float2 (&k1)[kPairs<V>],
                                            float2 (&k2)[kPairs<V>]) {
  if constexpr (V == 1) k1[0] = k2[0] = two(0.f);
  each_column<V>(g, p, [&](int k, int, int gi) {
    const float2 q = coef[gi - p.ga];
    put(k1, k, q.x);
    put(k2, k, q.y);
  });
}
// dx = dz * rstd * w - (first + second * (x - mean)).
__device__ __forceinline__ float2 coef_of(const Geo& g, float2 stat, double a, double c) {
  const double rstd = stat.y, first = rstd * a * g.inv_m, second = rstd * rstd * c * g.inv_m;
  return make_float2((float)first, (float)second);
}

// dx of a sample's edges.
template <typename T, int V, int ACT, bool Q>
__device__ __forceinline__ void dx_edges(const Geo& g, const Place& p, const T* __restrict__ dy,
                                         const void* __restrict__ x, const uint8_t* __restrict__ exps, const void* gamma,
                                         const void* beta, const float2* __restrict__ stats, const float2* coef,
                                         T* __restrict__ dx) {
  Edges::of<V>(g, p).each(g, [&](int64_t at, int c) {
    const int gi = (int)((unsigned)c / (unsigned)g.Cg);
    const float2 s = stats[gi], q = coef[gi - p.ga];
    const float2 e = grad_edge<T, ACT, Q>(g, dy, x, exps, gamma, beta, at, c, s);
    dx[at] = Elem<T>::from_f(fmaf(e.x, s.y * param(gamma, g.pdtype, c, 1.f), -fmaf(e.y, q.y, q.x)));
  });
}

// Blocks from g.blocks on sum the parameters' gradients, beside the others.
template <typename T, int V, int ACT, bool Q>
__global__ void __launch_bounds__(kThreads, kBwdBlocks) bwd_dx_kernel(
    const T* __restrict__ dy, const void* __restrict__ x, const uint8_t* __restrict__ exps,
    const float2* __restrict__ mean_rstd, const void* __restrict__ gamma, const void* __restrict__ beta,
    const __grid_constant__ Geo g, int64_t parts, const double2* cpart, const double2* gpart,
    T* __restrict__ dx, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  using R = Ring<T, V, Q, true, kBwdAhead>;
  extern __shared__ __align__(16) char smem[];
  float2* coef = reinterpret_cast<float2*>(smem + R::kBytes);   // per group of the tile: rstd * A, rstd^2 * B
  if (blockIdx.x >= g.blocks) {
    wait_for_previous();
    const int warps = blockDim.x / 32;
    const int64_t c = ((blockIdx.x - g.blocks) * gridDim.y + blockIdx.y) * warps + threadIdx.x / 32;
    if (c < g.C) param_grads(cpart, parts, g.C, (int)c, dgamma, dbeta);
    return;
  }
  const Place p = place<V>(g);
  const float2* stats = mean_rstd + p.n * g.G;
  // (what it reads is older than the kernel before this one)
  const int skip = p.tiles - p.mine;       // 1 for a thread without a row in the last tile
  const int64_t at = p.at + (p.tiles - 1) * p.step;
  T* to = dx + at;
  R ring(smem, x, dy, exps, at, -p.step);
#pragma unroll
  for (int i = 0; i < kBwdAhead - 1; ++i) ring.start(i, i >= skip && i < p.tiles);
  Affine<T, V, kSharedMeans<V>> k;
  k.means = reinterpret_cast<float4*>(coef + g.lanes * V) + p.lane * (V / 4);
  k.params(g, p, gamma, beta);
  k.stats(g, p, [&](int gi) { return stats[gi]; });
  wait_for_previous();
  const double2* src = gpart + p.n * g.np * g.G + p.ga;
  each_sum<double>(p.gb - p.ga, [&](int i, int sub, int tp, double& a, double& c) {
    add_previous<4>(src + i, sub, tp, g.np, g.G, a, c);
  }, [&](int i, double a, double c) { coef[i] = coef_of(g, stats[p.ga + i], a, c); });
  __syncthreads();
  if (p.mine > 0) {
    float2 k1[kPairs<V>], k2[kPairs<V>];
    thread_coef<V>(g, p, coef, k1, k2);
#pragma unroll 1
    for (int t = 0; t < p.tiles; t += kBwdAhead) {
#pragma unroll
      for (int i = 0; i < kBwdAhead; ++i) {
        if (t + i >= p.tiles) break;
        const bool in = t + i >= skip;
        Source<T, V, Q> v;
        Vec<T, V> d;
        ring.wait();
        if (in) {
          ring.get(i, v);
          ring.get_dy(i, d);
        }
        ring.next();
        const int next = t + i + kBwdAhead - 1;
        ring.start((i + kBwdAhead - 1) % kBwdAhead, next >= skip && next < p.tiles);
        if (in) dx_one<T, V, ACT, Q>(v, d, k, k1, k2, g).store(to);
        to -= p.step;
      }
    }
  }
  if (ACT < 0 && g.edges && p.b == 0) dx_edges<T, V, ACT, Q>(g, p, dy, x, exps, gamma, beta, stats, coef, dx);
  ring.drain();
}

// ---------------------------------------------------------------------------
// Small samples: one launch, data in shared memory
// ---------------------------------------------------------------------------
// A cluster of g.nb blocks keeps a sample's groups (all, or a channel tile of whole groups) in its shared memory, up to
// g.small vectors a thread, between the sums and the result: every element is read once, nothing goes through memory
// in between, and one launch does what two did. The blocks' sums are exchanged through shared memory. The loops stay
// rolled: code that runs once is paced by its own fetches (vectors in registers, unrolled: 8.5 us for [4,192,8,16,16]
// where two passes took 7.7).
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ double2 remote(const double2* p, uint32_t rank) {
  double2 v;
  asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];"
               : "=d"(v.x), "=d"(v.y) : "r"(in_block(shared_at(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Sums over the cluster's blocks of what each has in `mine` per group: out(group of the tile, sum, sum). Returns with
// an arrival on the cluster's barrier that the caller waits for before it exits (others may still read `mine`).
template <typename Out>
__device__ __forceinline__ void cluster_sums(const Geo& g, int groups, const double2* mine, Out out) {
  if (g.nb > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  each_sum<double>(groups, [&](int i, int sub, int tp, double& a, double& c) {
    for (int r = sub; r < g.nb; r += tp) {
      const double2 v = g.nb > 1 ? remote(mine + i, r) : mine[i];
      a += v.x;
      c += v.y;
    }
  }, out);
  __syncthreads();
  if (g.nb > 1) cluster_arrive();
}

// Bytes of a small kernel's shared memory: its vectors, then the blocks' tables, then each group's two results.
template <typename T, int V>
constexpr int small_fwd_bytes(int vectors) {
  return vectors * kThreads * V * (int)sizeof(T) + V * kThreads * (int)sizeof(double2) +
         kSmallGroups * (int)(sizeof(double2) + sizeof(float2));
}
template <typename T, int V, bool Q>
constexpr int small_bwd_bytes(int vectors, int lanes) {
  return vectors * kThreads * V * ((Q ? 1 : (int)sizeof(T)) + (int)sizeof(T)) + V * kThreads * (int)sizeof(float2) +
         V * lanes * (int)sizeof(double2) + kSmallGroups * (int)(sizeof(double2) + sizeof(float2));
}

template <typename T, int V, int ACT, bool PACK>
__global__ void __launch_bounds__(kThreads) fwd_small_kernel(const T* __restrict__ x, const void* __restrict__ gamma,
                                                             const void* __restrict__ beta,
                                                             const __grid_constant__ Geo g,
                                                             float2* __restrict__ mean_rstd, T* __restrict__ y,
                                                             uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ exps) {
  constexpr int B = V * (int)sizeof(T);
  extern __shared__ __align__(16) char smem[];
  double2* red = reinterpret_cast<double2*>(smem + g.small * kThreads * B);
  double2* mine = red + V * kThreads;
  float2* stat = reinterpret_cast<float2*>(mine + kSmallGroups);
  const Place p = place<V>(g);
  const int groups = p.gb - p.ga;
  const char* own = smem + threadIdx.x * B;
  for (int t = 0; t < p.mine; ++t) copy_async<B>(shared_at(own) + t * kThreads * B, x + p.at + t * p.step);
  for (int i = threadIdx.x; i < groups; i += blockDim.x) stat[i].x = origin(g, p, x, p.ga + i);
  Affine<T, V> k;
  k.params(g, p, gamma, beta);
  asm volatile("cp.async.wait_all;" ::: "memory");
  Moments<T, V> m;
  m.zero();
#pragma unroll 2
  for (int t = 0; t < p.mine; ++t) {
    Vec<T, V> v;
    v.load(reinterpret_cast<const T*>(own + t * kThreads * B));
    if (t == 0) m.pivot(v);
    m.add(v);
  }
  __syncthreads();
  block_moments<T, V>(g, p, m, x, red, [&](int i) { return stat[i].x; },
                      [&](int gi, double a, double c) { mine[gi - p.ga] = make_double2(a, c); });
  cluster_sums(g, groups, mine, [&](int i, double a, double c) { stat[i] = mean_rstd_of(g, a, c, stat[i].x); });
  if (p.b == 0)
    for (int i = threadIdx.x; i < groups; i += blockDim.x) mean_rstd[p.n * g.G + p.ga + i] = stat[i];
  k.stats(g, p, [&](int gi) { return stat[gi - p.ga]; });
#pragma unroll 2
  for (int t = 0; t < p.tiles; ++t) {
    Vec<T, V> v;
    v.zero();
    if (t < p.mine) v.load(reinterpret_cast<const T*>(own + t * kThreads * B));
    apply_one<T, V, ACT, PACK>(v, k, g, t < p.mine, p.at + t * p.step, y + p.at + t * p.step, codes, exps);
  }
  if (ACT < 0 && g.edges && p.b == 0) apply_edges<T, V, ACT>(g, p, x, gamma, beta, y, [&](int gi) { return stat[gi - p.ga]; });
  if (g.nb > 1) cluster_wait();
}

template <typename T, int V, int ACT, bool Q>
__global__ void __launch_bounds__(kThreads)
    bwd_small_kernel(const T* __restrict__ dy, const void* __restrict__ x, const uint8_t* __restrict__ exps,
                     const float2* __restrict__ mean_rstd, const void* __restrict__ gamma,
                     const void* __restrict__ beta, const __grid_constant__ Geo g, double2* __restrict__ cpart,
                     T* __restrict__ dx) {
  constexpr int XB = V * (Q ? 1 : (int)sizeof(T)), YB = V * (int)sizeof(T);
  extern __shared__ __align__(16) char smem[];
  char* dys = smem + g.small * kThreads * XB;
  float2* red = reinterpret_cast<float2*>(dys + g.small * kThreads * YB);
  double2* cols = reinterpret_cast<double2*>(red + V * kThreads);
  double2* mine = cols + V * g.lanes;
  float2* coef = reinterpret_cast<float2*>(mine + kSmallGroups);
  let_next_start();
  const Place p = place<V>(g);
  const int groups = p.gb - p.ga;
  const char *own = smem + threadIdx.x * XB, *own_dy = dys + threadIdx.x * YB;
  for (int t = 0; t < p.mine; ++t) {
    copy_async<XB>(shared_at(own) + t * kThreads * XB,
                   static_cast<const char*>(x) + (p.at + t * p.step) * (Q ? 1 : (int)sizeof(T)));
    copy_async<YB>(shared_at(own_dy) + t * kThreads * YB, dy + p.at + t * p.step);
  }
  const float2* stats = mean_rstd + p.n * g.G;
  Affine<T, V> k;
  k.params(g, p, gamma, beta);
  k.stats(g, p, [&](int gi) { return stats[gi]; });
  auto get = [&](int t, Source<T, V, Q>& v, Vec<T, V>& d) {
    if constexpr (Q) {
      v.c = q8::load_codes<V>(reinterpret_cast<const uint8_t*>(own + t * kThreads * XB));
      v.byte = exps[(p.at + t * p.step) / q8::kBlock];
    } else {
      v.v.load(reinterpret_cast<const T*>(own + t * kThreads * XB));
    }
    d.load(reinterpret_cast<const T*>(own_dy + t * kThreads * YB));
  };
  float2 s1[kPairs<V>], s2[kPairs<V>];
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) s1[i] = s2[i] = two(0.f);
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
  for (int t = 0; t < p.mine; ++t) {
    Source<T, V, Q> v;
    Vec<T, V> d;
    get(t, v, d);
    float2 xm[kPairs<V>], dz[kPairs<V>];
    grad_one<T, V, ACT, Q>(v, d, k, g, xm, dz);
#pragma unroll
    for (int j = 0; j < kPairs<V>; ++j) {
      s1[j] = __fadd2_rn(s1[j], dz[j]);
      s2[j] = __ffma2_rn(dz[j], xm[j], s2[j]);
    }
  }
  block_grads<V, (ACT < 0)>(g, p, s1, s2, gamma, red, cols, cpart, [&](int gi) { return stats[gi]; },
                 [&](int64_t at, int c, float2 s) { return grad_edge<T, ACT, Q>(g, dy, x, exps, gamma, beta, at, c, s); },
                 [&](int gi, double a, double c) { mine[gi - p.ga] = make_double2(a, c); });
  cluster_sums(g, groups, mine, [&](int i, double a, double c) { coef[i] = coef_of(g, stats[p.ga + i], a, c); });
  if (p.mine > 0) {
    float2 k1[kPairs<V>], k2[kPairs<V>];
    thread_coef<V>(g, p, coef, k1, k2);
#pragma unroll 2
    for (int t = 0; t < p.mine; ++t) {
      Source<T, V, Q> v;
      Vec<T, V> d;
      get(t, v, d);
      dx_one<T, V, ACT, Q>(v, d, k, k1, k2, g).store(dx + p.at + t * p.step);
    }
  }
  if (ACT < 0 && g.edges && p.b == 0) dx_edges<T, V, ACT, Q>(g, p, dy, x, exps, gamma, beta, stats, coef, dx);
  if (g.nb > 1) cluster_wait();
}

// ---------------------------------------------------------------------------
// Launches, one translation unit per element type (r4c_gn_*.cu)
// ---------------------------------------------------------------------------
struct FwdArgs {
  const void *x, *gamma, *beta;
  void* y;
  float2* mean_rstd;
  double2* part;
  uint8_t *codes, *exps;    // null: not wanted
  int sums_nb;              // blocks a sample of the sums
};
struct BwdArgs {
  const void *dy, *x, *gamma, *beta;
  const uint8_t* exps;      // null: x is the activation itself
  const float2* mean_rstd;
  void* dx;                 // null: not wanted
  float *dgamma, *dbeta;    // null: not wanted
  double2 *cpart, *gpart;
  int sums_nb;              // blocks a sample of the sums
};

template <typename T> cudaError_t launch_fwd(const FwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s);
template <typename T> cudaError_t launch_bwd(const BwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s);

}  // namespace gn
}  // namespace r4c
