// r4c_logp.cu — log-probability of a given label, entropy, log-sum-exp and
// the most probable classes of each row of logits, and the logits' gradient.
//
//   s_c = z_c / T,  m = max s,  S = sum exp(s_c - m),  lse = m + ln S
//   logp = s_t - lse,   H = ln S - (1/S) sum exp(s_c - m) (s_c - m)
//   dz_c = (1/T) [ p_c (g_lse - g_logp - g_H (ln p_c + H)) + g_logp [c = t] ],  p_c = exp(s_c - lse)
//
// The difference s_c - m is taken before it is scaled, so rows of the type's
// lowest value stay a uniform distribution instead of overflowing.
#include "r4c_rows.cuh"

namespace r4c {
namespace logp {

using namespace rows;

constexpr int kThreads = 256;

struct FwdArgs {
  const void* z;
  const int64_t* target;
  int64_t ignore, nrows;
  View v;
  int C, K;
  float inv_t;
  float *logp, *entropy, *lse, *top_logp;
  int32_t* top_index;
  float2* stats;
  int* err;
};

struct BwdArgs {
  const void* z;
  const int64_t* target;
  int64_t ignore, nrows;
  View v, dv;
  int C;
  float inv_t;
  const float* entropy;
  const float2* stats;
  const float *g_logp, *g_entropy, *g_lse;
  int gl_inc, gh_inc, gs_inc;
  void* dz;
  int* err;
};

__device__ __forceinline__ int label_of(const int64_t* target, int64_t r, int C, int64_t ignore, int* err) {
  if (!target) return -1;
  const int64_t t = target[r];
  if (t == ignore) return -1;
  if (t < 0 || t >= C) {
    atomicExch(err, 6);
    return -1;
  }
  return (int)t;
}

// One warp per row, any strides.
template <typename T>
__global__ void __launch_bounds__(kThreads) fwd_kernel(FwdArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= a.nrows) return;
  const T* z = static_cast<const T*>(a.z) + a.v.base(r);
  const float k2 = a.inv_t * kLog2e;
  float m = -INFINITY;
  for (int c = lane; c < a.C; c += 32) m = fmaxf(m, Elem<T>::to_f(z[c * a.v.sc]));
  m = warp_max(m);
  const float mm = m == -INFINITY ? 0.f : m;
  float s = 0.f, u = 0.f;
  for (int c = lane; c < a.C; c += 32) {
    const float d = Elem<T>::to_f(z[c * a.v.sc]) - mm;
    const float e = ex2(d * k2);
    s += e;
    u += e * fmaxf(d, -1e30f);
  }
  s = warp_sum(s);
  u = warp_sum(u);
  const bool bad = isnan(s), empty = s == 0.f;
  const float ln_s = empty ? -INFINITY : logf(s);
  if (lane == 0) {
    const int t = label_of(a.target, r, a.C, a.ignore, a.err);
    if (a.target) a.logp[r] = t < 0 ? 0.f : empty ? -INFINITY : (Elem<T>::to_f(z[t * a.v.sc]) - mm) * a.inv_t - ln_s;
    a.entropy[r] = empty ? 0.f : ln_s - a.inv_t * (u / s);
    a.lse[r] = mm * a.inv_t + ln_s;
    if (a.stats) a.stats[r] = make_float2(mm, ln_s);
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < a.K; ++j) {
    uint64_t best = 0;
    if (!bad) {
      for (int c = lane; c < a.C; c += 32) {
        const uint64_t key = rank_key(Elem<T>::to_f(z[c * a.v.sc]), c);
        if (key < last && key > best) best = key;
      }
      last = best = warp_max64(best);
    }
    if (lane == 0) {
      a.top_logp[r * a.K + j] = bad ? NAN : empty ? -INFINITY : (key_value(best) - mm) * a.inv_t - ln_s;
      a.top_index[r * a.K + j] = bad ? -1 : key_class(best);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) bwd_kernel(BwdArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= a.nrows) return;
  const T* z = static_cast<const T*>(a.z) + a.v.base(r);
  T* dz = static_cast<T*>(a.dz) + a.dv.base(r);
  const int t = label_of(a.target, r, a.C, a.ignore, a.err);
  const float gl = a.g_logp && t >= 0 ? a.g_logp[r * a.gl_inc] : 0.f;
  const float gh = a.g_entropy ? a.g_entropy[r * a.gh_inc] : 0.f;
  const float gs = a.g_lse ? a.g_lse[r * a.gs_inc] : 0.f;
  const float2 st = a.stats[r];
  const float h = a.entropy[r];
  const bool none = (gl == 0.f && gh == 0.f && gs == 0.f) || st.y == -INFINITY;
  for (int c = lane; c < a.C; c += 32) {
    float g = 0.f;
    if (!none) {
      const float ln_p = fmaxf((Elem<T>::to_f(z[c * a.v.sc]) - st.x) * a.inv_t, -1e30f) - st.y;
      const float p = ex2(ln_p * kLog2e);
      g = a.inv_t * (p * (gs - gl - gh * (ln_p + h)) + (c == t ? gl : 0.f));
      if (isnan(Elem<T>::to_f(z[c * a.v.sc]))) g = NAN;
    }
    dz[c * a.dv.sc] = Elem<T>::from_f(g);
  }
}

}  // namespace logp
}  // namespace r4c

using namespace r4c;

extern "C" size_t r4c_logp_stats_size(const r4c_rows_desc* d) {
  return rows::valid_desc(d) ? (size_t)d->rows * sizeof(float2) : 0;
}

extern "C" int r4c_logp_fwd(const r4c_rows_desc* d, const void* logits, const int64_t* target, int64_t ignore_index,
                            int top_k, float* logp, float* entropy, float* lse, float* top_logp, int32_t* top_index,
                            void* stats, r4c_stream_t stream) {
  if (!rows::valid_desc(d) || top_k < 0 || top_k > d->classes) return R4C_ERR_INVALID;
  if (d->rows == 0) return R4C_OK;
  if (!logits || !entropy || !lse || (target && !logp) || (top_k > 0 && (!top_logp || !top_index))) return R4C_ERR_INVALID;
  if (!rows::valid_dtype(d->dtype)) return R4C_ERR_UNSUPPORTED;
  if (top_k > R4C_TOPK_MAX) return R4C_ERR_TOO_LARGE;
  int* err = tc::device_error_flag();
  if (!err) return R4C_ERR_NO_DEVICE;
  logp::FwdArgs a{logits, target, ignore_index, d->rows, {d->inner, d->outer_stride, d->inner_stride, d->class_stride},
                  d->classes, top_k, 1.f / d->temperature, logp, entropy, lse, top_logp, top_index,
                  static_cast<float2*>(stats), err};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t grid = (d->rows + 7) / 8;
  if (grid > 0x7fffffff) return R4C_ERR_TOO_LARGE;
  if (d->dtype == R4C_BF16) logp::fwd_kernel<__nv_bfloat16><<<(int)grid, logp::kThreads, 0, s>>>(a);
  else if (d->dtype == R4C_F16) logp::fwd_kernel<__half><<<(int)grid, logp::kThreads, 0, s>>>(a);
  else logp::fwd_kernel<float><<<(int)grid, logp::kThreads, 0, s>>>(a);
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}

extern "C" int r4c_logp_bwd(const r4c_rows_desc* d, const void* logits, const int64_t* target, int64_t ignore_index,
                            const float* entropy, const void* stats, const float* g_logp, int g_logp_inc,
                            const float* g_entropy, int g_entropy_inc, const float* g_lse, int g_lse_inc,
                            void* dlogits, r4c_stream_t stream) {
  if (!rows::valid_desc(d)) return R4C_ERR_INVALID;
  if (d->rows == 0) return R4C_OK;
  if (!logits || !dlogits || !entropy || !stats || (g_logp && !target)) return R4C_ERR_INVALID;
  if (!rows::valid_dtype(d->dtype)) return R4C_ERR_UNSUPPORTED;
  int* err = tc::device_error_flag();
  if (!err) return R4C_ERR_NO_DEVICE;
  logp::BwdArgs a{logits, target, ignore_index, d->rows, {d->inner, d->outer_stride, d->inner_stride, d->class_stride},
                  {d->inner, d->grad_outer_stride, d->grad_inner_stride, d->grad_class_stride}, d->classes,
                  1.f / d->temperature, entropy, static_cast<const float2*>(stats), g_logp, g_entropy, g_lse,
                  g_logp_inc, g_entropy_inc, g_lse_inc, dlogits, err};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t grid = (d->rows + 7) / 8;
  if (grid > 0x7fffffff) return R4C_ERR_TOO_LARGE;
  if (d->dtype == R4C_BF16) logp::bwd_kernel<__nv_bfloat16><<<(int)grid, logp::kThreads, 0, s>>>(a);
  else if (d->dtype == R4C_F16) logp::bwd_kernel<__half><<<(int)grid, logp::kThreads, 0, s>>>(a);
  else logp::bwd_kernel<float><<<(int)grid, logp::kThreads, 0, s>>>(a);
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}
