// r4c_gn_launch.cuh — the launches of r4c_gn.cuh for one element type.
#pragma once

#include <atomic>

#include "r4c_gn.cuh"

namespace r4c {
namespace gn {

template <typename... P, typename... A>
cudaError_t launch_with(cudaLaunchAttribute at, void (*kernel)(P...), dim3 grid, int threads, size_t smem,
                        cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
// A launch that may start while the one before it in the stream still runs (it waits itself before it reads).
template <typename... P, typename... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  return launch_with(at, kernel, grid, threads, smem, s, args...);
}
template <typename... P, typename... A>
cudaError_t launch_cluster(int blocks, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                           A... args) {
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = blocks;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  return launch_with(at, kernel, grid, threads, smem, s, args...);
}

// Allows a kernel its shared memory above 48 KB, once a device.
template <typename K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<uint64_t>& devices) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (devices.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) devices.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <typename T, int V, int ACT, bool PACK>
cudaError_t fwd_small(const FwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  auto kernel = fwd_small_kernel<T, V, ACT, PACK>;
  const cudaError_t e = allow_shared(kernel, small_fwd_bytes<T, V>(kSmallFwd), allowed);
  if (e != cudaSuccess) return e;
  note_launches(1);
  return launch_cluster(g.nb, kernel, dim3((unsigned)g.blocks, g.tiles), threads, small_fwd_bytes<T, V>(g.small), s,
                        static_cast<const T*>(a.x), a.gamma, a.beta, g, a.mean_rstd, static_cast<T*>(a.y), a.codes,
                        a.exps);
}
template <typename T, int V, int ACT, bool Q>
cudaError_t bwd_small(const BwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  auto kernel = bwd_small_kernel<T, V, ACT, Q>;
  const cudaError_t e = allow_shared(kernel, small_bwd_bytes<T, V, Q>(kSmallBwd, kThreads), allowed);
  if (e != cudaSuccess) return e;
  note_launches(1);
  return launch_cluster(g.nb, kernel, dim3((unsigned)g.blocks, g.tiles), threads, small_bwd_bytes<T, V, Q>(g.small, g.lanes), s,
                        static_cast<const T*>(a.dy), a.x, a.exps, a.mean_rstd, a.gamma, a.beta, g, a.cpart,
                        static_cast<T*>(a.dx));
}

// Both passes with the SM's memory divided alike (all of it shared): blocks of the second may start beside the first's.
template <typename K>
void all_shared(K kernel, std::atomic<uint64_t>& devices) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return;
  const uint64_t bit = 1ull << dev;
  if (devices.load(std::memory_order_relaxed) & bit) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) == cudaSuccess)
    devices.fetch_or(bit, std::memory_order_relaxed);
  else
    (void)cudaGetLastError();           // (a preference)
}

template <typename T, int V, int ACT>
cudaError_t fwd_v(const FwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  const dim3 grid((unsigned)g.blocks, g.tiles);
  const T* x = static_cast<const T*>(a.x);
  if (g.small) {
    if constexpr (V * sizeof(T) == 16 && ACT >= 0)
      if (g.pack) return fwd_small<T, V, ACT, true>(a, g, threads, s);
    return fwd_small<T, V, ACT, false>(a, g, threads, s);
  }
  const size_t smem = Ring<T, V, false, false, kFwdAhead>::kBytes + sizeof(float2) * (g.tiles == 1 ? g.G : g.lanes * V);
  const Geo sums = split(g, a.sums_nb);
  static std::atomic<uint64_t> shared_s{0}, shared_a[2] = {{0}, {0}};
  all_shared(stats_kernel<T, V>, shared_s);
  stats_kernel<T, V><<<dim3((unsigned)sums.blocks, g.tiles), threads, 0, s>>>(x, sums, a.part);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  auto apply = apply_kernel<T, V, ACT, false>;
  if constexpr (V * sizeof(T) == 16 && ACT >= 0)             // (samples with edges are packed on their own)
    if (g.pack) apply = apply_kernel<T, V, ACT, true>;
  all_shared(apply, shared_a[g.pack != 0]);
  e = launch_next(apply, grid, threads, smem, s, x, a.gamma, a.beta, g, a.part, a.mean_rstd, static_cast<T*>(a.y),
                  a.codes, a.exps);
  note_launches(2);
  return e;
}

template <typename T, int V, int ACT, bool Q>
cudaError_t bwd_v(const BwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  dim3 grid((unsigned)g.blocks, g.tiles);
  const T* dy = static_cast<const T*>(a.dy);
  const bool params = a.dgamma || a.dbeta;
  const Geo sums = g.small ? g : split(g, a.sums_nb);
  auto params_next = [&] {
    note_launches(1);
    return launch_next(params_kernel, dim3(sums.blocks < kWideParts ? cdiv(g.C, kThreads / 32) : g.C), kThreads, 0, s,
                       a.cpart, sums.blocks, g.C, a.dgamma, a.dbeta);
  };
  if (g.small && a.dx) {
    const cudaError_t e = bwd_small<T, V, ACT, Q>(a, g, threads, s);
    return e != cudaSuccess || !params ? e : params_next();
  }
  using R = Ring<T, V, Q, true, kBwdAhead>;
  // each group's coefficients, then the columns' means
  constexpr size_t column = sizeof(float2) + (kSharedMeans<V> ? sizeof(float) : 0);
  const size_t smem = R::kBytes + column * g.lanes * V;
  static std::atomic<uint64_t> shared_s{0}, shared_d{0}, allowed{0};
  cudaError_t e = allow_shared(bwd_dx_kernel<T, V, ACT, Q>, R::kBytes + (int)column * kThreads * V, allowed);
  if (e != cudaSuccess) return e;
  all_shared(bwd_sums_kernel<T, V, ACT, Q>, shared_s);
  all_shared(bwd_dx_kernel<T, V, ACT, Q>, shared_d);
  bwd_sums_kernel<T, V, ACT, Q><<<dim3((unsigned)sums.blocks, g.tiles), threads, 0, s>>>(
      dy, a.x, a.exps, a.mean_rstd, a.gamma, a.beta, sums, a.cpart, a.gpart);
  note_launches(1);
  e = cudaGetLastError();
  if (e != cudaSuccess || !a.dx) return e != cudaSuccess ? e : params_next();
  const bool beside = params && sums.blocks < kWideParts;
  if (beside) grid.x += cdiv(g.C, (int64_t)g.tiles * (threads / 32));
  note_launches(1);
  e = launch_next(bwd_dx_kernel<T, V, ACT, Q>, grid, threads, smem, s, dy, a.x, a.exps, a.mean_rstd, a.gamma, a.beta,
                  g, sums.blocks, a.cpart, a.gpart, static_cast<T*>(a.dx), a.dgamma, a.dbeta);
  if (e != cudaSuccess || !params || beside) return e;
  return params_next();
}

// The widest vectors have a kernel for each activation; narrower ones and samples with edges one for all.
template <typename T, int V>
cudaError_t fwd_act(const FwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  if constexpr (V * sizeof(T) == 16) {
    if (g.edges) return fwd_v<T, V, -1>(a, g, threads, s);
    switch (g.act) {
      case R4C_ACT_NONE: return fwd_v<T, V, R4C_ACT_NONE>(a, g, threads, s);
      case R4C_ACT_RELU: return fwd_v<T, V, R4C_ACT_RELU>(a, g, threads, s);
      case R4C_ACT_LEAKY_RELU: return fwd_v<T, V, R4C_ACT_LEAKY_RELU>(a, g, threads, s);
      case R4C_ACT_SILU: return fwd_v<T, V, R4C_ACT_SILU>(a, g, threads, s);
      default: return fwd_v<T, V, R4C_ACT_GELU>(a, g, threads, s);
    }
  } else {
    return fwd_v<T, V, -1>(a, g, threads, s);
  }
}
template <typename T, int V, bool Q>
cudaError_t bwd_act(const BwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  if constexpr (V * sizeof(T) == 16) {
    if (g.edges) return bwd_v<T, V, -1, Q>(a, g, threads, s);
    switch (g.act) {
      case R4C_ACT_NONE: return bwd_v<T, V, R4C_ACT_NONE, Q>(a, g, threads, s);
      case R4C_ACT_RELU: return bwd_v<T, V, R4C_ACT_RELU, Q>(a, g, threads, s);
      case R4C_ACT_LEAKY_RELU: return bwd_v<T, V, R4C_ACT_LEAKY_RELU, Q>(a, g, threads, s);
      case R4C_ACT_SILU: return bwd_v<T, V, R4C_ACT_SILU, Q>(a, g, threads, s);
      default: return bwd_v<T, V, R4C_ACT_GELU, Q>(a, g, threads, s);
    }
  } else {
    return bwd_v<T, V, -1, Q>(a, g, threads, s);
  }
}

template <typename T>
cudaError_t launch_fwd(const FwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (V == 8) return fwd_act<T, 8>(a, g, threads, s);
  if (V == 4) return fwd_act<T, 4>(a, g, threads, s);
  if (V == 2) return fwd_act<T, 2>(a, g, threads, s);
  return fwd_act<T, 1>(a, g, threads, s);
}

template <typename T, bool Q>
cudaError_t bwd_q(const BwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (V == 8) return bwd_act<T, 8, Q>(a, g, threads, s);
  if (V == 4) return bwd_act<T, 4, Q>(a, g, threads, s);
  if (V == 2) return bwd_act<T, 2, Q>(a, g, threads, s);
  return bwd_act<T, 1, Q>(a, g, threads, s);
}
template <typename T>
cudaError_t launch_bwd(const BwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s) {
  return a.exps ? bwd_q<T, true>(a, g, V, threads, s) : bwd_q<T, false>(a, g, V, threads, s);
}

#define R4C_GN_INSTANCE(T)                                                                \
  template cudaError_t launch_fwd<T>(const FwdArgs&, const Geo&, int, int, cudaStream_t); \
  template cudaError_t launch_bwd<T>(const BwdArgs&, const Geo&, int, int, cudaStream_t);

}  // namespace gn
}  // namespace r4c
