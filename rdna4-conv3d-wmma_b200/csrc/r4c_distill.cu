// r4c_distill.cu — distillation from a teacher's top classes: the student's
// row of logits against K (log-probability, class) pairs of the teacher.
//
//   s_c = z_c / T,  ln p_c = s_c - lse(s);  v_j, i_j the teacher's pairs
//   renormalised:  q_j = exp(v_j) / sum exp(v)
//   rest bucket:   q_j = exp(v_j),  q_r = max(0, 1 - sum q)  against  p_r = sum of p over unlisted classes
//   L  = T^2 [ sum_j q_j (ln q_j - ln p_{i_j}) + q_r (ln q_r - ln p_r) ]
//   dL/dz_c = T [ Q p_c - q_c ]                    listed c;   Q = sum q + q_r
//           = T exp(s_c - lse_r) [ Q p_r - q_r ]   unlisted c (lse_r over the unlisted classes alone)
//
// The unlisted classes keep a log-sum-exp of their own: 1 - sum p would lose
// a student's small rest mass to cancellation, and its gradient with it.
// A pair with a negative class or a log-probability of -inf is void. A row
// without valid pairs, with weight 0 or with no finite logit takes no part.
#include "r4c_rows.cuh"

namespace r4c {
namespace distill {

using namespace rows;

constexpr int kThreads = 256;

struct Stats {           // per row, written by the forward for the backward
  float m, ln_s;         // lse = m / T + ln_s (m a logit, not yet scaled)
  float mr, ln_sr;       // the same over the unlisted classes
  float q_norm;          // ln q_j = v_j - q_norm
  float mass, q_rest;    // Q, q_r
  float w;               // the row's weight, 0: takes no part
};

struct Args {
  const void* z;
  View v, dv;
  int64_t nrows;
  int C, K, rest;
  float temp, inv_t;
  const void* t_logp;
  const void* t_index;
  int t_dtype, t_wide;
  const float* weight;
  float* row_loss;       // forward: w L
  float* row_w;          // forward: w of a row that takes part
  Stats* stats;
  const float* loss_weight;
  const float* grad;
  int grad_inc;
  void* dz;
  int* err;
};

__device__ __forceinline__ float teacher_logp(const Args& a, int64_t i) {
  if (a.t_dtype == R4C_F32) return static_cast<const float*>(a.t_logp)[i];
  if (a.t_dtype == R4C_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.t_logp)[i]);
  return __half2float(static_cast<const __half*>(a.t_logp)[i]);
}
// The pair's class, -1 when the pair is void.
__device__ __forceinline__ int teacher_class(const Args& a, int64_t i, float v) {
  const int64_t c = a.t_wide ? static_cast<const int64_t*>(a.t_index)[i] : static_cast<const int32_t*>(a.t_index)[i];
  if (c < 0 || v == -INFINITY) return -1;
  if (c >= a.C) {
    atomicExch(a.err, 6);
    return -1;
  }
  return (int)c;
}

// One warp per row, any strides.
template <typename T>
__global__ void __launch_bounds__(kThreads) fwd_kernel(Args a) {
  __shared__ int sh_idx[kThreads / 32][R4C_TOPK_MAX];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + warp;
  if (r >= a.nrows) return;
  const T* z = static_cast<const T*>(a.z) + a.v.base(r);
  const float k2 = a.inv_t * kLog2e;
  float w = a.weight ? a.weight[r] : 1.f;
  float qm = -INFINITY;
  for (int j = lane; j < a.K; j += 32) {
    const float v = teacher_logp(a, r * a.K + j);
    const int c = teacher_class(a, r * a.K + j, v);
    sh_idx[warp][j] = c;
    if (c >= 0) qm = fmaxf(qm, v);
  }
  __syncwarp();
  const bool any = __any_sync(0xffffffffu, [&] {
    bool x = false;
    for (int j = lane; j < a.K; j += 32) x |= sh_idx[warp][j] >= 0;
    return x;
  }());
  qm = warp_max(qm);
  if (!any) w = 0.f;
  Stats st{};
  float loss = 0.f;
  if (w != 0.f) {
    auto listed = [&](int c) {
      for (int j = 0; j < a.K; ++j)
        if (sh_idx[warp][j] == c) return true;
      return false;
    };
    float m = -INFINITY, mr = -INFINITY;
    for (int c = lane; c < a.C; c += 32) {
      const float x = Elem<T>::to_f(z[c * a.v.sc]);
      m = fmaxf(m, x);
      if (a.rest && x > mr && !listed(c)) mr = x;
    }
    m = warp_max(m);
    mr = warp_max(mr);
    const float mm = m == -INFINITY ? 0.f : m, mmr = mr == -INFINITY ? 0.f : mr;
    float s = 0.f, sr = 0.f;
    for (int c = lane; c < a.C; c += 32) {
      const float x = Elem<T>::to_f(z[c * a.v.sc]);
      s += ex2((x - mm) * k2);
      if (a.rest && !listed(c)) sr += ex2((x - mmr) * k2);
    }
    s = warp_sum(s);
    sr = warp_sum(sr);
    if (s == 0.f) w = 0.f;   // no finite logit
    st.m = mm;
    st.ln_s = logf(s);
    st.mr = mmr;
    st.ln_sr = logf(sr);
    st.q_norm = 0.f;
    if (!a.rest) {
      float qs = 0.f;
      for (int j = lane; j < a.K; j += 32)
        if (sh_idx[warp][j] >= 0) qs += expf(teacher_logp(a, r * a.K + j) - qm);
      st.q_norm = qm + logf(warp_sum(qs));
    }
    float sum_q = 0.f;
    for (int j = lane; j < a.K; j += 32) {
      const int c = sh_idx[warp][j];
      if (c < 0) continue;
      const float ln_q = teacher_logp(a, r * a.K + j) - st.q_norm, q = expf(ln_q);
      sum_q += q;
      if (!(q == 0.f)) loss += q * (ln_q - ((Elem<T>::to_f(z[c * a.v.sc]) - mm) * a.inv_t - st.ln_s));
    }
    sum_q = warp_sum(sum_q);
    loss = warp_sum(loss);
    if (a.rest) {
      const float qr = 1.f - sum_q;
      st.q_rest = qr >= kRestNoise ? qr : 0.f;
      if (st.q_rest > 0.f)
        loss += st.q_rest * (logf(st.q_rest) - ((mmr - mm) * a.inv_t + (st.ln_sr - st.ln_s)));
    }
    st.mass = sum_q + st.q_rest;
    loss *= a.temp * a.temp;
  }
  st.w = w;
  if (lane == 0) {
    a.row_loss[r] = w == 0.f ? 0.f : w * loss;
    if (a.row_w) a.row_w[r] = w;
    a.stats[r] = st;
  }
}

// loss_weight = (sum of row losses / sum of weights, sum of weights), summed in a fixed order in double.
__global__ void __launch_bounds__(1024) mean_kernel(const float* loss, const float* w, int64_t n, float* loss_weight) {
  __shared__ double sh[2][1024];
  double s = 0.0, t = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    s += loss[i];
    t += w[i];
  }
  sh[0][threadIdx.x] = s;
  sh[1][threadIdx.x] = t;
  __syncthreads();
  for (int off = 512; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) {
      sh[0][threadIdx.x] += sh[0][threadIdx.x + off];
      sh[1][threadIdx.x] += sh[1][threadIdx.x + off];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    loss_weight[0] = (float)(sh[0][0] / sh[1][0]);   // no row takes part: NaN
    loss_weight[1] = (float)sh[1][0];
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) bwd_kernel(Args a) {
  __shared__ int sh_idx[kThreads / 32][R4C_TOPK_MAX];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + warp;
  if (r >= a.nrows) return;
  const T* z = static_cast<const T*>(a.z) + a.v.base(r);
  T* dz = static_cast<T*>(a.dz) + a.dv.base(r);
  const Stats st = a.stats[r];
  if (st.w == 0.f) {
    for (int c = lane; c < a.C; c += 32) dz[c * a.dv.sc] = Elem<T>::from_f(0.f);
    return;
  }
  for (int j = lane; j < a.K; j += 32)
    sh_idx[warp][j] = teacher_class(a, r * a.K + j, teacher_logp(a, r * a.K + j));
  __syncwarp();
  const float scale = a.temp * st.w * a.grad[r * a.grad_inc] / (a.loss_weight ? a.loss_weight[1] : 1.f);
  const float base = a.rest ? st.mr : st.m, ln_b = a.rest ? st.ln_sr : st.ln_s;
  const float p_r = expf((st.mr - st.m) * a.inv_t + (st.ln_sr - st.ln_s));
  const float coef = a.rest ? st.mass * p_r - st.q_rest : st.mass;
  for (int c = lane; c < a.C; c += 32) {
    const float x = Elem<T>::to_f(z[c * a.v.sc]);
    float q = 0.f;
    bool listed = false;
    for (int j = 0; j < a.K; ++j)
      if (sh_idx[warp][j] == c) {
        listed = true;
        q += expf(teacher_logp(a, r * a.K + j) - st.q_norm);
      }
    float g;
    if (listed) g = st.mass * ex2(((x - st.m) * a.inv_t - st.ln_s) * kLog2e) - q;
    else g = x == -INFINITY ? 0.f : coef * ex2(((x - base) * a.inv_t - ln_b) * kLog2e);
    dz[c * a.dv.sc] = Elem<T>::from_f(scale * g);
  }
}

}  // namespace distill
}  // namespace r4c

using namespace r4c;

namespace {
int check(const r4c_rows_desc* d, int k, const void* t_logp, int t_dtype, const void* t_index, int index_bits) {
  if (!rows::valid_desc(d) || k <= 0 || (index_bits != 32 && index_bits != 64)) return R4C_ERR_INVALID;
  if (d->rows > 0 && (!t_logp || !t_index)) return R4C_ERR_INVALID;
  if (!rows::valid_dtype(d->dtype) || !rows::valid_dtype(t_dtype)) return R4C_ERR_UNSUPPORTED;
  if (k > R4C_TOPK_MAX || d->rows > (int64_t)0x7fffffff * 8) return R4C_ERR_TOO_LARGE;
  return R4C_OK;
}
distill::Args make_args(const r4c_rows_desc* d, const void* logits, int k, const void* t_logp, int t_dtype,
                        const void* t_index, int index_bits, int rest, const float* weight, void* stats) {
  distill::Args a{};
  a.z = logits;
  a.v = {d->inner, d->outer_stride, d->inner_stride, d->class_stride};
  a.dv = {d->inner, d->grad_outer_stride, d->grad_inner_stride, d->grad_class_stride};
  a.nrows = d->rows;
  a.C = d->classes;
  a.K = k;
  a.rest = rest != 0;
  a.temp = d->temperature;
  a.inv_t = 1.f / d->temperature;
  a.t_logp = t_logp;
  a.t_index = t_index;
  a.t_dtype = t_dtype;
  a.t_wide = index_bits == 64;
  a.weight = weight;
  a.stats = static_cast<distill::Stats*>(stats);
  return a;
}
}  // namespace

extern "C" size_t r4c_distill_stats_size(const r4c_rows_desc* d) {
  return rows::valid_desc(d) ? (size_t)d->rows * sizeof(distill::Stats) : 0;
}
extern "C" size_t r4c_distill_workspace_size(const r4c_rows_desc* d) {
  return rows::valid_desc(d) ? (size_t)d->rows * 2 * sizeof(float) : 0;
}

extern "C" int r4c_distill_fwd(const r4c_rows_desc* d, const void* logits, int k, const void* teacher_logp,
                               int teacher_dtype, const void* teacher_index, int index_bits, int rest,
                               const float* weight, float* row_loss, float* loss_weight, void* stats, void* ws,
                               size_t ws_bytes, r4c_stream_t stream) {
  const int rc = check(d, k, teacher_logp, teacher_dtype, teacher_index, index_bits);
  if (rc != R4C_OK) return rc;
  if ((!row_loss && !loss_weight) || (d->rows > 0 && (!logits || !stats))) return R4C_ERR_INVALID;
  if (d->rows > 0 && (!ws || ws_bytes < r4c_distill_workspace_size(d))) return R4C_ERR_WORKSPACE;
  distill::Args a = make_args(d, logits, k, teacher_logp, teacher_dtype, teacher_index, index_bits, rest, weight, stats);
  a.err = tc::device_error_flag();
  if (!a.err) return R4C_ERR_NO_DEVICE;
  a.row_loss = row_loss ? row_loss : static_cast<float*>(ws);
  a.row_w = loss_weight ? static_cast<float*>(ws) + d->rows : nullptr;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int grid = (int)((d->rows + 7) / 8);
  if (d->rows > 0) {
    if (d->dtype == R4C_BF16) distill::fwd_kernel<__nv_bfloat16><<<grid, distill::kThreads, 0, s>>>(a);
    else if (d->dtype == R4C_F16) distill::fwd_kernel<__half><<<grid, distill::kThreads, 0, s>>>(a);
    else distill::fwd_kernel<float><<<grid, distill::kThreads, 0, s>>>(a);
    note_launches(1);
  }
  if (loss_weight) {
    distill::mean_kernel<<<1, 1024, 0, s>>>(a.row_loss, a.row_w, d->rows, loss_weight);
    note_launches(1);
  }
  return cudaGetLastError() == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}

extern "C" int r4c_distill_bwd(const r4c_rows_desc* d, const void* logits, int k, const void* teacher_logp,
                               int teacher_dtype, const void* teacher_index, int index_bits, int rest,
                               const float* weight, const float* loss_weight, const float* grad, int grad_inc,
                               const void* stats, void* dlogits, r4c_stream_t stream) {
  const int rc = check(d, k, teacher_logp, teacher_dtype, teacher_index, index_bits);
  if (rc != R4C_OK) return rc;
  if (d->rows == 0) return R4C_OK;
  if (!logits || !dlogits || !grad || !stats) return R4C_ERR_INVALID;
  distill::Args a = make_args(d, logits, k, teacher_logp, teacher_dtype, teacher_index, index_bits, rest, weight,
                              const_cast<void*>(stats));
  a.err = tc::device_error_flag();
  if (!a.err) return R4C_ERR_NO_DEVICE;
  a.loss_weight = loss_weight;
  a.grad = grad;
  a.grad_inc = grad_inc;
  a.dz = dlogits;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int grid = (int)((d->rows + 7) / 8);
  if (d->dtype == R4C_BF16) distill::bwd_kernel<__nv_bfloat16><<<grid, distill::kThreads, 0, s>>>(a);
  else if (d->dtype == R4C_F16) distill::bwd_kernel<__half><<<grid, distill::kThreads, 0, s>>>(a);
  else distill::bwd_kernel<float><<<grid, distill::kThreads, 0, s>>>(a);
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}
