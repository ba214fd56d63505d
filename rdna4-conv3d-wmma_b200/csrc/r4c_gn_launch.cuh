// r4c_gn_launch.cuh — the launches of r4c_gn.cuh for one element type.
#pragma once

#include "r4c_gn.cuh"

namespace r4c {
namespace gn {

template <typename T, int V>
cudaError_t fwd_v(const FwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  const dim3 grid((unsigned)g.blocks, g.tiles);
  const T* x = static_cast<const T*>(a.x);
  const size_t smem = sizeof(float2) * (g.tiles == 1 ? g.G : g.lanes * V);
  stats_kernel<T, V><<<grid, threads, 0, s>>>(x, g, a.part);
  apply_kernel<T, V><<<grid, threads, smem, s>>>(x, a.gamma, a.beta, g, a.part, a.mean_rstd, static_cast<T*>(a.y));
  note_launches(2);
  return cudaGetLastError();
}

template <typename T, int V, bool Q>
cudaError_t bwd_v(const BwdArgs& a, const Geo& g, int threads, cudaStream_t s) {
  const dim3 grid((unsigned)g.blocks, g.tiles);
  const T* dy = static_cast<const T*>(a.dy);
  const size_t smem = sizeof(float2) * (g.tiles == 1 ? g.G : g.lanes * V);
  bwd_sums_kernel<T, V, Q><<<grid, threads, 0, s>>>(dy, a.x, a.exps, a.mean_rstd, a.gamma, a.beta, g, a.cpart, a.gpart);
  note_launches(1);
  if (a.dx) {
    bwd_dx_kernel<T, V, Q><<<grid, threads, smem, s>>>(dy, a.x, a.exps, a.mean_rstd, a.gamma, a.beta, g, a.gpart,
                                                      static_cast<T*>(a.dx));
    note_launches(1);
  }
  if (a.dgamma || a.dbeta) {
    params_kernel<<<cdiv(g.C, kThreads / 32), kThreads, 0, s>>>(a.cpart, g.blocks, g.C, a.dgamma, a.dbeta);
    note_launches(1);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_fwd(const FwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (V == 8) return fwd_v<T, 8>(a, g, threads, s);
  if (V == 4) return fwd_v<T, 4>(a, g, threads, s);
  if (V == 2) return fwd_v<T, 2>(a, g, threads, s);
  return fwd_v<T, 1>(a, g, threads, s);
}

template <typename T, bool Q>
cudaError_t bwd_q(const BwdArgs& a, const Geo& g, int V, int threads, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (V == 8) return bwd_v<T, 8, Q>(a, g, threads, s);
  if (V == 4) return bwd_v<T, 4, Q>(a, g, threads, s);
  if (V == 2) return bwd_v<T, 2, Q>(a, g, threads, s);
  return bwd_v<T, 1, Q>(a, g, threads, s);
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
