// r4c_distill.cuh — distillation from a teacher's top classes: the student's
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
#pragma once

#include "r4c_rows.cuh"

namespace r4c {
namespace distill {

using namespace rows;

struct Stats {           // per streamed row, written by the forward for the backward
  float m, s;            // lse = m / T + ln s (m a logit, not yet scaled)
  float mr, sr;          // the same over the unlisted classes
  float qm, qs;          // q_j = exp(v_j - qm) / qs
  float mass, q_rest;    // Q, q_r
  float w;               // the row's weight, 0: takes no part
};

constexpr int kParts = kSMs * 32;   // most blocks of a forward: each leaves one partial sum

struct Args {
  const void* z;
  View v, dv;
  Tile tile;
  int64_t nrows;
  int C, K, rest, segs;
  int even;              // short rows: K even and the pairs 8-byte aligned
  float temp, inv_t;
  const void* t_logp;
  const void* t_index;
  int t_dtype, t_wide;
  float t_round;         // the largest relative rounding of 16-bit log-probabilities, 0 for fp32
  const float* weight;
  float* row_loss;       // forward: w L per row, or null
  double* part;          // forward: (sum w L, sum w) of each block, or null
  float* loss;           // the mean and the sum of weights, written by a launch of one block itself
  float* total;
  Stats* stats;
  const float* total_weight;
  const float* grad;
  int grad_inc;
  void* dz;
  int* err;
};

// PLAIN: fp32 log-probabilities and 32-bit classes; else what the types say.
template <bool PLAIN>
__device__ __forceinline__ float teacher_logp(const Args& a, int64_t first, int i) {
  if (PLAIN || a.t_dtype == R4C_F32) return __ldg(static_cast<const float*>(a.t_logp) + first + i);
  if (a.t_dtype == R4C_BF16) return __bfloat162float((static_cast<const __nv_bfloat16*>(a.t_logp) + first)[i]);
  return __half2float((static_cast<const __half*>(a.t_logp) + first)[i]);
}
// The class of a pair as the kernels use it, -1 when the pair is void.
template <typename I>
__device__ __forceinline__ int valid_class(const Args& a, I c, float v) {
  if (c < 0 || v == -INFINITY) return -1;
  if (c >= a.C) {
    atomicExch(a.err, 6);
    return -1;
  }
  return (int)c;
}
template <bool PLAIN>
__device__ __forceinline__ int teacher_class(const Args& a, int64_t first, int i, float v) {
  if (PLAIN || !a.t_wide) return valid_class(a, __ldg(static_cast<const int32_t*>(a.t_index) + first + i), v);
  return valid_class(a, __ldg(static_cast<const long long*>(a.t_index) + first + i), v);
}
// T g / W of the row; its weight comes on top.
__device__ __forceinline__ float grad_scale(const Args& a, int64_t r) {
  return a.temp * a.grad[r * a.grad_inc] / (a.total_weight ? a.total_weight[0] : 1.f);
}
// A block's (sum of losses, sum of weights), in a fixed order.
template <int NT>
__device__ __forceinline__ void leave_part(double loss, double w, const Args& a) {
  __shared__ double sh[2][NT / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, o);
    w += __shfl_xor_sync(0xffffffffu, w, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sh[0][threadIdx.x >> 5] = loss;
    sh[1][threadIdx.x >> 5] = w;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NT / 32; ++i) {
      loss += sh[0][i];
      w += sh[1][i];
    }
    if (gridDim.x == 1) {
      a.loss[0] = (float)(loss / w);   // no row takes part: NaN
      a.total[0] = (float)w;
    } else {
      a.part[2 * blockIdx.x] = loss;
      a.part[2 * blockIdx.x + 1] = w;
    }
  }
}

// The terms of a row that come from its sums: r over the unlisted classes
// (rest) or all of them, l over the listed ones (rest). Probabilities are
// exponentials divided by their sum, logarithms serve the loss alone: a
// difference p - q then keeps the exponentials' own error.
struct RowSums {
  float m, s, mr, sr;
  bool empty;
  __device__ __forceinline__ RowSums(const Run& r, const Run& l, bool rest, float k) {
    const float top = rest ? fmaxf(r.m, l.m) : r.m;
    m = anchor(top);
    mr = anchor(r.m);
    sr = s = r.s;
    if (rest) s = r.s * ex2((r.m - m) * k) + l.s * ex2((l.m - m) * k);   // an empty side: 0 * 2^-inf
    empty = s == 0.f;
  }
};
// What rounding v = ln q to 16 bits takes from q at most: q (e^x - 1), x = round |v|.
__device__ __forceinline__ float pair_noise(float q, float v, float round) {
  const float x = round * fabsf(v);
  return q > 0.f ? q * fmaf(x, x, x) : 0.f;
}
// q_r from the sum of the listed q. `noise` is what the stored pairs' rounding
// explains, given only where the student has no unlisted class: mass on none
// is infinitely far off, and there it would be so for a teacher that lists
// all there is. With unlisted classes 1 - sum q is the best that is known.
__device__ __forceinline__ float rest_mass(float sum_q, float noise) {
  const float qr = 1.f - sum_q;
  return qr >= kRestNoise + noise ? qr : 0.f;
}
// q_r (ln q_r - ln p_r)
__device__ __forceinline__ float rest_loss(float qr, const RowSums& s, float inv_t) {
  return qr > 0.f ? qr * (kLn2 * (lg2(qr) - lg2(s.sr) + lg2(s.s)) - (s.mr - s.m) * inv_t) : 0.f;
}
// The factor of 2^t (t from mr) in the gradient of an unlisted class: (Q p_r - q_r) / sr, 0 without any.
__device__ __forceinline__ float rest_coef(bool rest, float mass, float qr, float m, float s, float mr, float sr, float k) {
  if (!rest) return __fdividef(mass, s);
  return sr == 0.f ? 0.f : __fdividef(mass * ex2((mr - m) * k), s) - __fdividef(qr, sr);
}
// The pairs' exponentials: few, and their difference from the student's is the gradient.
__device__ __forceinline__ float prob(float ln_q) { return expf(ln_q); }

// The kernels for rows of up to kTileClasses classes (r4c_distill_tile.cuh),
// one translation unit for each type of logits.
template <typename T>
cudaError_t launch_tiles(Args& a, bool bwd, int* blocks, cudaStream_t s);

}  // namespace distill
}  // namespace r4c
