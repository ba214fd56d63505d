// r4c_rows.cuh — rows of logits: addressing, arithmetic and the two ways of
// reading them shared by the log-probability (r4c_logp.cu) and distillation
// (r4c_distill.cu) kernels.
//
// A row is the class axis at one voxel of an (N, C, D, H, W) map or at one
// token of an (R, C) matrix; r4c_rows_desc gives its place for any strides.
//
// * Up to kTileClasses classes ("tile"): G lanes hold a whole row in
//   registers, so a kernel reads it once whatever it needs of it, and a
//   backward recomputes the softmax instead of loading saved statistics.
//   Dense rows come through shared memory: tiles of consecutive rows are one
//   contiguous piece of memory, copied with 16-byte cp.async whatever the
//   alignment of each row (105 classes of 2 bytes start on any even byte).
// * Above ("block"): a block, or a cluster of blocks when there are few rows,
//   streams over the row in 16-byte loads and keeps a running maximum and sum.
#pragma once

#include <cmath>

#include "r4c_internal.h"
#include "r4c_sm100.cuh"

namespace r4c {
namespace rows {

constexpr float kLog2e = 1.4426950408889634f;
// A rest mass 1 - sum(q) below this is the rounding of the teacher's own sum.
constexpr float kRestNoise = 1e-6f;
constexpr int kTileClasses = 1024;
constexpr int kTileThreads = 256;
constexpr int kSMs = 148;

struct View {
  int64_t inner, so, si, sc;   // inner 0: one stride walks all rows
  __device__ __forceinline__ int64_t base(int64_t r) const {
    return inner == 0 ? r * si : (r / inner) * so + (r % inner) * si;
  }
};

inline bool valid_desc(const r4c_rows_desc* d) {
  return d && d->rows >= 0 && d->inner > 0 && d->classes > 0 && std::isfinite(d->temperature) && d->temperature > 0.f;
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

// ---- 32-bit words of logits -------------------------------------------------
template <typename T> struct Word;
template <> struct Word<float> {
  static constexpr int kElems = 1;
  static __device__ __forceinline__ void split(uint32_t w, float* v) { v[0] = __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t join(const float* v) { return __float_as_uint(v[0]); }
};
template <> struct Word<__nv_bfloat16> {
  static constexpr int kElems = 2;
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

// ---- tile: rows held in registers --------------------------------------------
// Geometry of a tile launch. `staged`: rows dense and 16-byte aligned as a
// whole, read (and for a backward written) through shared memory.
struct Tile {
  int64_t nrows, ntiles;
  int C, rows_per_tile, staged, stage_bytes;
};
constexpr int kTileStages = 3;

// One lane's part of a row: E values, value e = i * kElems + h being class
// cls(e). Lanes take words cyclically (lane l words l, l + G, ...), each row
// starting at another one of them (`rot`), so that rows whose width is a
// multiple of the banks do not meet in the same bank.
template <typename T, int G, int E>
struct TileRow {
  static constexpr int kW = Word<T>::kElems, kEW = E / kW;
  float v[E];
  uint32_t live;        // bit e: v[e] is a class of the row
  int lane, rot, odd;   // odd: the row starts at the second half of a word

  __device__ __forceinline__ int word(int i) const { return lane + G * ((i + rot) & (kEW - 1)); }
  __device__ __forceinline__ int cls(int e) const { return kW * word(e / kW) + e % kW - odd; }
  // Where class c sits: true and its e when this lane holds it.
  __device__ __forceinline__ bool owns(int c, int* e) const {
    const int p = c + odd, w = p / kW;
    *e = (((w / G) - rot) & (kEW - 1)) * kW + p % kW;
    return w % G == lane;
  }
  // row: the row's first element, in shared memory (staged) or global memory.
  __device__ __forceinline__ void load(const T* row, int64_t sc, int C, bool staged) {
    const int wl = threadIdx.x & 31;
    lane = wl & (G - 1);
    live = 0;
    if (staged) {
      const uint32_t a = sm100::smem_u32(row);
      odd = kW == 2 ? (a >> 1) & 1 : 0;
      const int nw = (odd + C + kW - 1) / kW;
      rot = (nw & 1) ? 0 : G == 1 ? wl / (32 / (kEW < 32 ? kEW : 32)) : wl / G;
#pragma unroll
      for (int i = 0; i < kEW; ++i) {
        const int w = word(i);
        uint32_t x = 0;
        if (w < nw) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"((a & ~3u) + 4 * w) : "memory");
        Word<T>::split(x, v + i * kW);
#pragma unroll
        for (int h = 0; h < kW; ++h) {
          const int c = kW * w + h - odd;
          const bool ok = c >= 0 && c < C;
          if (!ok) v[i * kW + h] = -INFINITY;
          live |= (uint32_t)ok << (i * kW + h);
        }
      }
    } else {
      odd = rot = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = cls(e);
        const bool ok = c < C;
        v[e] = ok ? Elem<T>::to_f(row[c * sc]) : -INFINITY;
        live |= (uint32_t)ok << e;
      }
    }
  }
  // g[e] to the classes of `which` (a subset of live), in the row's own place or at `row`.
  __device__ __forceinline__ void store(T* row, int64_t sc, bool staged, const float* g, uint32_t which) const {
    if (staged) {
      const uint32_t a = sm100::smem_u32(row) & ~3u;
#pragma unroll
      for (int i = 0; i < kEW; ++i) {
        const uint32_t at = a + 4 * word(i);
        const uint32_t x = Word<T>::join(g + i * kW);
        const uint32_t sel = (which >> (i * kW)) & ((1u << kW) - 1u);
        if (sel == (1u << kW) - 1u) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(x) : "memory");
        else if (kW == 2 && sel == 1u) asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"((uint16_t)x) : "memory");
        else if (kW == 2 && sel == 2u)
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + 2), "h"((uint16_t)(x >> 16)) : "memory");
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (which >> e & 1) row[cls(e) * sc] = Elem<T>::from_f(g[e]);
    }
  }
};

// Copies a tile's bytes into a stage (the last chunk of the last tile in part).
__device__ __forceinline__ void tile_fetch(const Tile& t, const void* z, int64_t tile, int es, uint8_t* stage) {
  const int64_t r0 = tile * t.rows_per_tile;
  if (tile < t.ntiles) {
    const int64_t nr = t.nrows - r0 < t.rows_per_tile ? t.nrows - r0 : t.rows_per_tile;
    const int bytes = (int)(nr * t.C * es);
    const uint8_t* src = static_cast<const uint8_t*>(z) + r0 * t.C * es;
    const uint32_t dst = sm100::smem_u32(stage);
    for (int b = threadIdx.x * 16; b < bytes; b += kTileThreads * 16)
      sm100::cp_async_16(dst + b, src + b, bytes - b < 16 ? bytes - b : 16);
  }
  sm100::cp_async_commit();
}
// Writes a stage back to dense rows of dz (the block has synchronized).
template <typename T>
__device__ __forceinline__ void tile_flush(const Tile& t, void* dz, int64_t tile, const uint8_t* stage) {
  const int64_t r0 = tile * t.rows_per_tile;
  const int64_t nr = t.nrows - r0 < t.rows_per_tile ? t.nrows - r0 : t.rows_per_tile;
  const int bytes = (int)(nr * t.C * sizeof(T));
  uint8_t* dst = static_cast<uint8_t*>(dz) + r0 * t.C * sizeof(T);
  for (int b = threadIdx.x * 16; b < bytes; b += kTileThreads * 16) {
    if (bytes - b >= 16) *reinterpret_cast<uint4*>(dst + b) = *reinterpret_cast<const uint4*>(stage + b);
    else
      for (int i = b; i < bytes; i += (int)sizeof(T)) *reinterpret_cast<T*>(dst + i) = *reinterpret_cast<const T*>(stage + i);
  }
}

// Walks the tiles of a persistent block: body(row index, row pointer in
// shared or global memory, in range) for each group of G lanes and row. All
// lanes of a warp call body together; rows out of range repeat the last row.
template <typename T, int G, bool WRITES, typename Body>
__device__ __forceinline__ void tile_walk(const Tile& t, const void* z, const View& v, void* dz, Body&& body) {
  extern __shared__ __align__(16) uint8_t stages[];
  constexpr int R = kTileThreads / G;
  const int sub = threadIdx.x / G;
  if (t.staged) {
    for (int s = 0; s < kTileStages - 1; ++s)
      tile_fetch(t, z, blockIdx.x + (int64_t)s * gridDim.x, sizeof(T), stages + s * t.stage_bytes);
    int st = 0;
    for (int64_t tile = blockIdx.x; tile < t.ntiles; tile += gridDim.x) {
      sm100::cp_async_wait<kTileStages - 2>();
      __syncthreads();   // this tile has landed for everyone, the last one is done with
      tile_fetch(t, z, tile + (int64_t)(kTileStages - 1) * gridDim.x, sizeof(T),
                 stages + ((st + kTileStages - 1) % kTileStages) * t.stage_bytes);
      T* base = reinterpret_cast<T*>(stages + st * t.stage_bytes);
      const int64_t r0 = tile * t.rows_per_tile;
      const int nr = (int)(t.nrows - r0 < t.rows_per_tile ? t.nrows - r0 : t.rows_per_tile);
      for (int i = 0; i < nr; i += R) {
        const int q = i + sub, at = q < nr ? q : nr - 1;
        body(r0 + at, base + (int64_t)at * t.C, q < nr);
      }
      if (WRITES) {
        __syncthreads();
        tile_flush<T>(t, dz, tile, stages + st * t.stage_bytes);
      }
      st = (st + 1) % kTileStages;
    }
  } else {
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < t.nrows; r0 += (int64_t)gridDim.x * R) {
      const int64_t q = r0 + sub, at = q < t.nrows ? q : t.nrows - 1;
      body(at, const_cast<T*>(static_cast<const T*>(z)) + v.base(at), q < t.nrows);
    }
  }
}

// Lanes per row and values per lane by the number of classes.
struct TileKind { int g, e; };
inline TileKind tile_kind(int C) {
  if (C <= 4) return {1, 4};
  if (C <= 8) return {1, 8};
  if (C <= 16) return {1, 16};
  if (C <= 32) return {1, 32};
  if (C <= 64) return {4, 16};
  if (C <= 128) return {8, 16};
  if (C <= 256) return {16, 16};
  if (C <= 512) return {32, 16};
  return {32, 32};
}
// One tile of up to 16 KB (at least one row for each group of lanes): three
// of them in flight in each of the blocks of an SM keep the memory busy.
inline Tile make_tile(const r4c_rows_desc* d, int es, int g, bool dense) {
  Tile t;
  t.nrows = d->rows;
  t.C = d->classes;
  t.staged = dense;
  const int r = kTileThreads / g;
  int reps = (16 << 10) / (r * d->classes * es);
  reps = reps < 1 ? 1 : reps > 16 ? 16 : reps;
  // few rows: smaller tiles, so that every SM gets some
  while (reps > 1 && d->rows < (int64_t)r * reps * 2 * kSMs) reps /= 2;
  t.rows_per_tile = r * reps;
  t.ntiles = (d->rows + t.rows_per_tile - 1) / t.rows_per_tile;
  t.stage_bytes = (t.rows_per_tile * d->classes * es + 31) / 16 * 16;
  return t;
}
inline bool dense_rows(const View& v, int64_t rows, int classes, const void* p) {
  return v.inner == 0 && (v.sc == 1 || classes == 1) && (v.si == classes || rows == 1) && ((uintptr_t)p & 15) == 0;
}
// Blocks of a persistent tile launch: what shared memory and threads let an SM hold.
inline int tile_grid(const Tile& t, int threads_rows) {
  if (!t.staged) {
    const int64_t n = (t.nrows + threads_rows - 1) / threads_rows;
    return (int)(n < kSMs * 8 ? n : kSMs * 8);
  }
  int per_sm = (216 << 10) / (kTileStages * t.stage_bytes + 1024);
  per_sm = per_sm < 1 ? 1 : per_sm > 8 ? 8 : per_sm;
  return (int)(t.ntiles < kSMs * per_sm ? t.ntiles : kSMs * per_sm);
}

template <typename K, typename A>
inline cudaError_t launch_tile(K* kernel, const Tile& t, int threads_rows, cudaStream_t st, const A& a) {
  const size_t smem = t.staged ? (size_t)kTileStages * t.stage_bytes : 0;
  if (smem > 48 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kernel<<<tile_grid(t, threads_rows), kTileThreads, smem, st>>>(a);
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

// Running maximum and sums of exponentials: s = sum exp2((z - m) k),
// u = sum exp2((z - m) k) (z - m), k = log2(e) / T. m = -inf: nothing finite yet.
struct Run {
  float m, s, u;
};
__device__ __forceinline__ Run run_empty() { return {-INFINITY, 0.f, 0.f}; }
__device__ __forceinline__ Run run_merge(const Run& a, const Run& b, float k) {
  const float m = fmaxf(a.m, b.m), mm = anchor(m);
  const float da = a.m - mm, db = b.m - mm;
  const float fa = ex2(da * k), fb = ex2(db * k);
  // an empty side has s = u = 0 and a difference of -inf: bounded, so that 0 * it stays 0
  return {m, a.s * fa + b.s * fb, fa * (a.u + fmaxf(da, -1e30f) * a.s) + fb * (b.u + fmaxf(db, -1e30f) * b.s)};
}
template <int N, bool ENT>
__device__ __forceinline__ void run_add(Run& r, const float* x, float k) {
  float bm = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) bm = fmaxf(bm, x[i]);
  if (bm > r.m) {
    const float d = r.m - bm, f = ex2(d * k);
    if (ENT) r.u = f * (r.u + fmaxf(d, -1e30f) * r.s);
    r.s *= f;
    r.m = bm;
  }
  const float mm = anchor(r.m);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = x[i] - mm, e = ex2(d * k);
    r.s += e;
    if (ENT) r.u = fmaf(e, fmaxf(d, -1e30f), r.u);
  }
}
// Joins the threads' runs of a block; every thread gets the result.
template <int NT>
__device__ __forceinline__ Run run_block(Run r, float k, Run* sh) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const Run b{__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o),
                __shfl_xor_sync(0xffffffffu, r.u, o)};
    r = run_merge(r, b, k);
  }
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = r;
  __syncthreads();
  r = sh[0];
  for (int i = 1; i < NT / 32; ++i) r = run_merge(r, sh[i], k);
  return r;
}

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

// Blocks that share a row: as many as bring the rows to two blocks an SM, in
// powers of two up to 16, while each keeps a few vectors a thread.
inline int cluster_size(int64_t nrows, int C, int es, int threads) {
  int cs = 1;
  while (cs < 16 && nrows * cs * 2 <= 2 * kSMs && (int64_t)C * es >= (int64_t)threads * 16 * 2 * (cs * 2)) cs *= 2;
  return cs;
}

template <typename K, typename A>
inline cudaError_t launch_cluster(K* kernel, int64_t grid, int threads, int cs, size_t smem, cudaStream_t st, const A& a) {
  if (smem > 48 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  if (cs > 1) {
    if (cs > 8) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
    }
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
