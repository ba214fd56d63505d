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
// Both are bound by memory: forward 3, backward 5 activations read or written.
//
// A thread owns a vector of V neighbouring elements in every R-th row of its block's range, so its channels and with
// them the parameters stay in registers. A row is a voxel's channels, or L / C voxels together where C is no multiple
// of V (L = lcm(C, V)), so that odd channel counts still move 16 bytes at a time. Rows wider than a block's threads
// are cut into channel tiles.
//
// Sums: a thread keeps sum (x - p) and sum (x - p)^2 in fp32 around its own first value p, so nothing cancels where
// |mean| >> std, and an outlier as p spoils one thread's few elements at most; threads, blocks and samples add in
// fp64 about zero, in a fixed order: same bits on every run.
#pragma once

#include "r4c_internal.h"
#include "r4c_q8.cuh"

namespace r4c {
namespace gn {

constexpr int kThreads = 256;   // at most, per block

struct Geo {
  int64_t sample;    // elements of a sample, S * C
  int64_t rows;      // rows of L elements of a sample
  int64_t chunk;     // rows of a block, a multiple of R
  int64_t blocks;    // samples * nb: blocks of one channel tile
  double inv_m;      // 1 / (Cg * S)
  float eps, slope;
  int act, pdtype, format;
  int L, C, G, Cg;
  int lanes;         // vectors of a row in a channel tile (L / V when there is one tile)
  int tiles;
  int R;             // rows that a block's threads cover at a time
  int nb;            // blocks of a sample and channel tile
};

// V elements of T, moved as one word.
template <int B> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

template <typename T, int V>
struct Vec {
  using W = typename Word<V * sizeof(T)>::type;
  W raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = raw; }
  __device__ __forceinline__ void to_f(float (&f)[V]) const {
    const T* p = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Elem<T>::to_f(p[i]);
  }
  __device__ __forceinline__ void from_f(const float (&f)[V]) {
    T* p = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = Elem<T>::from_f(f[i]);
  }
};

// The activation that a backward reads: x itself, or the values of its 8 bits.
template <typename T, int V, bool Q>
struct Source;
template <typename T, int V>
struct Source<T, V, false> {
  Vec<T, V> v;
  __device__ __forceinline__ void load(const void* x, const uint8_t*, int64_t at) { v.load(static_cast<const T*>(x) + at); }
  __device__ __forceinline__ void to_f(int, float (&f)[V]) const { v.to_f(f); }
};
template <typename T, int V>
struct Source<T, V, true> {
  q8::Codes<V> c;
  int byte;
  __device__ __forceinline__ void load(const void* x, const uint8_t* exps, int64_t at) {
    c = q8::load_codes<V>(static_cast<const uint8_t*>(x) + at);
    byte = exps[at / q8::kBlock];
  }
  __device__ __forceinline__ void to_f(int format, float (&f)[V]) const { q8::decode<T, V>(c, byte, format, f); }
};

__device__ __forceinline__ float param(const void* p, int dtype, int c, float none) {
  if (!p) return none;
  if (dtype == R4C_F32) return __ldg(static_cast<const float*>(p) + c);
  if (dtype == R4C_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
  return __half2float(static_cast<const __half*>(p)[c]);
}

// 1 / (1 + e^-z): for 16-bit results the hardware's exponential and reciprocal (relative error about 2^-21, the
// result's own half step is 2^-9 or 2^-12), the library's in full precision for fp32.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-z));
  return __fdividef(1.f, 1.f + __expf(-z));
}

template <typename T>
__device__ __forceinline__ float act_value(float z, int act, float slope) {
  switch (act) {
    case R4C_ACT_RELU: return z <= 0.f ? 0.f : z;              // NaN stays
    case R4C_ACT_LEAKY_RELU: return z <= 0.f ? z * slope : z;
    case R4C_ACT_SILU: return z * sigmoid<T>(z);
    case R4C_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678f));
    default: return z;
  }
}
template <typename T>
__device__ __forceinline__ float act_slope(float z, int act, float slope) {
  switch (act) {
    case R4C_ACT_RELU: return z <= 0.f ? 0.f : 1.f;
    case R4C_ACT_LEAKY_RELU: return z <= 0.f ? slope : 1.f;
    case R4C_ACT_SILU: {
      const float s = sigmoid<T>(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    case R4C_ACT_GELU: {
      const float e = sizeof(T) == 4 ? expf(-0.5f * z * z) : __expf(-0.5f * z * z);
      return fmaf(z, e * 0.39894228f, 0.5f * (1.f + erff(z * 0.70710678f)));
    }
    default: return 1.f;
  }
}

// Where a block's threads stand: sample n, part b of it, channel tile, and a thread's lane and row.
struct Place {
  int64_t n;
  int b, tile, lane, row;
  int j0, j1;         // the tile's elements of a row
  int ga, gb;         // the tile's groups
  bool active;
};
template <int V>
__device__ __forceinline__ Place place(const Geo& g) {
  Place p;
  p.n = blockIdx.x / g.nb;
  p.b = (int)(blockIdx.x - p.n * g.nb);
  p.tile = blockIdx.y;
  p.lane = threadIdx.x % g.lanes;
  p.row = threadIdx.x / g.lanes;
  p.j0 = p.tile * g.lanes * V;
  p.j1 = min(p.j0 + g.lanes * V, g.L);
  p.ga = g.tiles == 1 ? 0 : p.j0 / g.Cg;
  p.gb = g.tiles == 1 ? g.G : (p.j1 - 1) / g.Cg + 1;
  p.active = p.row < g.R && p.j0 + p.lane * V < p.j1;
  return p;
}

// Neighbouring threads for each of `items` sums: the largest power of two that the block has, at most a warp.
__device__ __forceinline__ int threads_per(int items, int threads) {
  int t = 32;
  while (t > 1 && t * items > threads) t >>= 1;
  return t;
}

// ---------------------------------------------------------------------------
// Forward: sums
// ---------------------------------------------------------------------------
// part[((n * nb + b) * tiles + tile) * G + g] = (sum x, sum x^2) of the block's share of group g.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) stats_kernel(const T* __restrict__ x, const Geo g,
                                                         double2* __restrict__ part) {
  constexpr int U = 4;
  __shared__ double2 red[V * kThreads];
  const Place p = place<V>(g);
  const int64_t r0 = p.b * g.chunk, r1 = min(r0 + g.chunk, g.rows);
  float s1[V], s2[V], pv[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s1[k] = s2[k] = pv[k] = 0.f;
  int cnt = 0;
  if (p.active && r0 + p.row < r1) {
    const T* src = x + p.n * g.sample + p.j0 + p.lane * V;
    {
      Vec<T, V> a;
      a.load(src + (r0 + p.row) * g.L);
      a.to_f(pv);
    }
    for (int64_t r = r0 + p.row; r < r1; r += U * g.R) {
      Vec<T, V> a[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u * g.R < r1) a[u].load(src + (r + u * g.R) * g.L);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u * g.R >= r1) break;
        float f[V];
        a[u].to_f(f);
        ++cnt;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = f[k] - pv[k];
          s1[k] += d;
          s2[k] = fmaf(d, d, s2[k]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const double q = pv[k], a = s1[k], c = cnt;
    red[k * kThreads + threadIdx.x] = make_double2(c * q + a, (double)s2[k] + 2.0 * q * a + c * q * q);
  }
  __syncthreads();
  const int groups = p.gb - p.ga, tp = threads_per(groups, blockDim.x);
  const int sub = threadIdx.x % tp;
  double2* out = part + ((int64_t)blockIdx.x * g.tiles + p.tile) * g.G;
  if (g.tiles > 1)
    for (int i = threadIdx.x; i < g.G; i += blockDim.x)
      if (i < p.ga || i >= p.gb) out[i] = make_double2(0.0, 0.0);
  const int reps = g.L / g.C;
  // the loop bound is the same for every thread of a warp: the shuffles below need all lanes
  for (int base = 0; base < groups; base += blockDim.x / tp) {
    const int gi = p.ga + base + threadIdx.x / tp;
    double a = 0.0, c = 0.0;
    if (gi < p.gb && threadIdx.x / tp < blockDim.x / tp) {
      const int lo = max(gi * g.Cg, g.tiles == 1 ? 0 : p.j0), hi = min((gi + 1) * g.Cg, g.tiles == 1 ? g.C : p.j1);
      const int w = hi - lo, total = reps * w * g.R;
      for (int e = sub; e < total; e += tp) {
        const int row = e % g.R, q = e / g.R;
        const int j = (q / w) * g.C + lo + q % w - p.j0;
        const double2 v = red[(j % V) * kThreads + row * g.lanes + j / V];
        a += v.x;
        c += v.y;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (o < tp) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        c += __shfl_xor_sync(0xffffffffu, c, o);
      }
    }
    if (sub == 0 && gi < p.gb && threadIdx.x / tp < blockDim.x / tp) out[gi] = make_double2(a, c);
  }
}

// ---------------------------------------------------------------------------
// Forward: y
// ---------------------------------------------------------------------------
// Mean and rstd of the tile's groups from the blocks' partial sums, into shared memory.
__device__ __forceinline__ void finish_stats(const Geo& g, const Place& p, const double2* __restrict__ part,
                                             float2* stat) {
  const int groups = p.gb - p.ga, tp = threads_per(groups, blockDim.x), sub = threadIdx.x % tp;
  const int np = g.nb * g.tiles;
  const double2* src = part + p.n * np * g.G;
  for (int base = 0; base < groups; base += blockDim.x / tp) {
    const int gi = p.ga + base + threadIdx.x / tp;
    const bool own = gi < p.gb && threadIdx.x / tp < blockDim.x / tp;
    double a = 0.0, c = 0.0;
    if (own)
      for (int i = sub; i < np; i += tp) {
        const double2 v = src[(int64_t)i * g.G + gi];
        a += v.x;
        c += v.y;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (o < tp) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        c += __shfl_xor_sync(0xffffffffu, c, o);
      }
    }
    if (own && sub == 0) {
      const double mean = a * g.inv_m;
      double var = c * g.inv_m - mean * mean;
      if (var < 0.0) var = 0.0;
      stat[gi - p.ga] = make_float2((float)mean, (float)(1.0 / sqrt(var + (double)g.eps)));
    }
  }
  __syncthreads();
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) apply_kernel(const T* __restrict__ x, const void* __restrict__ gamma,
                                                         const void* __restrict__ beta, const Geo g,
                                                         const double2* __restrict__ part,
                                                         float2* __restrict__ mean_rstd, T* __restrict__ y) {
  constexpr int U = 4;
  extern __shared__ float2 stat[];
  const Place p = place<V>(g);
  finish_stats(g, p, part, stat);
  if (p.b == 0)
    for (int i = threadIdx.x; i < p.gb - p.ga; i += blockDim.x) mean_rstd[p.n * g.G + p.ga + i] = stat[i];
  if (!p.active) return;
  float mu[V], a[V], b[V];
  const int j = p.j0 + p.lane * V;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (j + k) % g.C;
    const float2 s = stat[c / g.Cg - p.ga];
    mu[k] = s.x;
    a[k] = s.y * param(gamma, g.pdtype, c, 1.f);
    b[k] = param(beta, g.pdtype, c, 0.f);
  }
  const int64_t r0 = p.b * g.chunk, r1 = min(r0 + g.chunk, g.rows), at = p.n * g.sample + j;
  for (int64_t r = r0 + p.row; r < r1; r += U * g.R) {
    Vec<T, V> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u * g.R < r1) v[u].load(x + at + (r + u * g.R) * g.L);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * g.R >= r1) break;
      float f[V];
      v[u].to_f(f);
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = act_value<T>(fmaf(f[k] - mu[k], a[k], b[k]), g.act, g.slope);
      v[u].from_f(f);
      v[u].store(y + at + (r + u * g.R) * g.L);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward: sums
// ---------------------------------------------------------------------------
// cpart[(n * nb + b) * C + c] = (sum dz, sum dz * xh) of the block's rows, and
// gpart[((n * nb + b) * tiles + tile) * G + g] = the same times w, summed over the tile's channels of the group.
template <typename T, int V, bool Q>
__global__ void __launch_bounds__(kThreads) bwd_sums_kernel(const T* __restrict__ dy, const void* __restrict__ x,
                                                            const uint8_t* __restrict__ exps,
                                                            const float2* __restrict__ mean_rstd,
                                                            const void* __restrict__ gamma,
                                                            const void* __restrict__ beta, const Geo g,
                                                            float2* __restrict__ cpart, float2* __restrict__ gpart) {
  constexpr int U = 4;
  __shared__ float2 red[V * kThreads];
  __shared__ float2 cols[V * kThreads];     // per column of the tile, (j1 - j0) <= V * kThreads
  const Place p = place<V>(g);
  const int64_t r0 = p.b * g.chunk, r1 = min(r0 + g.chunk, g.rows);
  float s1[V], s2[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s1[k] = s2[k] = 0.f;
  if (p.active) {
    float mu[V], a[V], b[V], rs[V];
    const int j = p.j0 + p.lane * V;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (j + k) % g.C;
      const float2 s = mean_rstd[p.n * g.G + c / g.Cg];
      mu[k] = s.x;
      rs[k] = s.y;
      a[k] = s.y * param(gamma, g.pdtype, c, 1.f);
      b[k] = param(beta, g.pdtype, c, 0.f);
    }
    const int64_t at = p.n * g.sample + j;
    for (int64_t r = r0 + p.row; r < r1; r += U * g.R) {
      Source<T, V, Q> v[U];
      Vec<T, V> d[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u * g.R < r1) {
          v[u].load(x, exps, at + (r + u * g.R) * g.L);
          d[u].load(dy + at + (r + u * g.R) * g.L);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u * g.R >= r1) break;
        float f[V], h[V];
        v[u].to_f(g.format, f);
        d[u].to_f(h);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float xm = f[k] - mu[k];
          const float dz = h[k] * act_slope<T>(fmaf(xm, a[k], b[k]), g.act, g.slope);
          s1[k] += dz;
          s2[k] = fmaf(dz, xm, s2[k]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) s2[k] *= rs[k];
  }
#pragma unroll
  for (int k = 0; k < V; ++k) red[k * kThreads + threadIdx.x] = make_float2(s1[k], s2[k]);
  __syncthreads();
  const int ncol = p.j1 - p.j0;
  {
    const int tp = threads_per(ncol, blockDim.x), sub = threadIdx.x % tp;
    for (int base = 0; base < ncol; base += blockDim.x / tp) {
      const int j = base + threadIdx.x / tp;
      const bool own = j < ncol && threadIdx.x / tp < blockDim.x / tp;
      float u = 0.f, v = 0.f;
      if (own)
        for (int r = sub; r < g.R; r += tp) {
          const float2 e = red[(j % V) * kThreads + r * g.lanes + j / V];
          u += e.x;
          v += e.y;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        if (o < tp) {
          u += __shfl_xor_sync(0xffffffffu, u, o);
          v += __shfl_xor_sync(0xffffffffu, v, o);
        }
      }
      if (own && sub == 0) cols[j] = make_float2(u, v);
    }
  }
  __syncthreads();
  const int reps = g.L / g.C, nch = g.tiles == 1 ? g.C : ncol;
  for (int i = threadIdx.x; i < nch; i += blockDim.x) {
    float2 s = cols[i];
    for (int q = 1; q < reps; ++q) {
      const float2 e = cols[q * g.C + i];
      s.x += e.x;
      s.y += e.y;
    }
    cols[i] = s;                            // columns of one channel are this thread's alone
    cpart[(int64_t)blockIdx.x * g.C + p.j0 + i] = s;
  }
  __syncthreads();
  float2* out = gpart + ((int64_t)blockIdx.x * g.tiles + p.tile) * g.G;
  for (int i = threadIdx.x; i < g.G; i += blockDim.x) {
    float u = 0.f, v = 0.f;
    const int lo = max(i * g.Cg, p.j0), hi = min((i + 1) * g.Cg, p.j0 + nch);
    for (int c = lo; c < hi; ++c) {
      const float w = param(gamma, g.pdtype, c, 1.f);
      u = fmaf(w, cols[c - p.j0].x, u);
      v = fmaf(w, cols[c - p.j0].y, v);
    }
    out[i] = make_float2(u, v);
  }
}

// ---------------------------------------------------------------------------
// Backward: dx, and the gradients of weight and bias
// ---------------------------------------------------------------------------
template <typename T, int V, bool Q>
__global__ void __launch_bounds__(kThreads) bwd_dx_kernel(const T* __restrict__ dy, const void* __restrict__ x,
                                                          const uint8_t* __restrict__ exps,
                                                          const float2* __restrict__ mean_rstd,
                                                          const void* __restrict__ gamma,
                                                          const void* __restrict__ beta, const Geo g,
                                                          const float2* __restrict__ gpart, T* __restrict__ dx) {
  constexpr int U = 4;
  extern __shared__ float2 coef[];          // per group of the tile: rstd * A, rstd^2 * B
  const Place p = place<V>(g);
  {
    const int groups = p.gb - p.ga, tp = threads_per(groups, blockDim.x), sub = threadIdx.x % tp;
    const int np = g.nb * g.tiles;
    const float2* src = gpart + p.n * np * g.G;
    for (int base = 0; base < groups; base += blockDim.x / tp) {
      const int gi = p.ga + base + threadIdx.x / tp;
      const bool own = gi < p.gb && threadIdx.x / tp < blockDim.x / tp;
      double u = 0.0, v = 0.0;
      if (own)
        for (int i = sub; i < np; i += tp) {
          const float2 e = src[(int64_t)i * g.G + gi];
          u += e.x;
          v += e.y;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        if (o < tp) {
          u += __shfl_xor_sync(0xffffffffu, u, o);
          v += __shfl_xor_sync(0xffffffffu, v, o);
        }
      }
      if (own && sub == 0) {
        const double r = mean_rstd[p.n * g.G + gi].y;
        coef[gi - p.ga] = make_float2((float)(r * u * g.inv_m), (float)(r * r * v * g.inv_m));
      }
    }
    __syncthreads();
  }
  if (!p.active) return;
  float mu[V], a[V], b[V], k1[V], k2[V];
  const int j = p.j0 + p.lane * V;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (j + k) % g.C;
    const float2 s = mean_rstd[p.n * g.G + c / g.Cg];
    const float2 q = coef[c / g.Cg - p.ga];
    mu[k] = s.x;
    a[k] = s.y * param(gamma, g.pdtype, c, 1.f);
    b[k] = param(beta, g.pdtype, c, 0.f);
    k1[k] = q.x;
    k2[k] = q.y;
  }
  const int64_t r0 = p.b * g.chunk, r1 = min(r0 + g.chunk, g.rows), at = p.n * g.sample + j;
  for (int64_t r = r0 + p.row; r < r1; r += U * g.R) {
    Source<T, V, Q> v[U];
    Vec<T, V> d[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u * g.R < r1) {
        v[u].load(x, exps, at + (r + u * g.R) * g.L);
        d[u].load(dy + at + (r + u * g.R) * g.L);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * g.R >= r1) break;
      float f[V], h[V];
      v[u].to_f(g.format, f);
      d[u].to_f(h);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xm = f[k] - mu[k];
        const float dz = h[k] * act_slope<T>(fmaf(xm, a[k], b[k]), g.act, g.slope);
        h[k] = fmaf(dz, a[k], -fmaf(xm, k2[k], k1[k]));
      }
      d[u].from_f(h);
      d[u].store(dx + at + (r + u * g.R) * g.L);
    }
  }
}

// dw, db: a warp a channel over the (sample, block) sums, in a fixed order.
inline __global__ void __launch_bounds__(kThreads) params_kernel(const float2* __restrict__ cpart, int64_t parts, int C,
                                                                 float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int c = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
  if (c >= C) return;
  double u = 0.0, v = 0.0;
  for (int64_t i = lane; i < parts; i += 32) {
    const float2 e = cpart[i * C + c];
    u += e.x;
    v += e.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(0xffffffffu, u, o);
    v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  if (lane == 0) {
    if (dbeta) dbeta[c] = (float)u;
    if (dgamma) dgamma[c] = (float)v;
  }
}

// ---------------------------------------------------------------------------
// Launches, one translation unit per element type (r4c_gn_*.cu)
// ---------------------------------------------------------------------------
struct FwdArgs {
  const void *x, *gamma, *beta;
  void* y;
  float2* mean_rstd;
  double2* part;
};
struct BwdArgs {
  const void *dy, *x, *gamma, *beta;
  const uint8_t* exps;      // null: x is the activation itself
  const float2* mean_rstd;
  void* dx;                 // null: not wanted
  float *dgamma, *dbeta;    // null: not wanted
  float2 *cpart, *gpart;
};

template <typename T> cudaError_t launch_fwd(const FwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s);
template <typename T> cudaError_t launch_bwd(const BwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s);

}  // namespace gn
}  // namespace r4c
