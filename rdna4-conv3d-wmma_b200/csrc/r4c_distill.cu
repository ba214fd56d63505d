// r4c_distill.cu — distillation from a teacher's top classes: the streamed rows
// (more than 1024 classes), the mean over rows and the C entries. The
// operator and the short rows are in r4c_distill.cuh and r4c_distill_tile.cuh.
#include "r4c_distill.cuh"

namespace r4c {
namespace distill {

// ---- rows streamed -----------------------------------------------------------
// -inf in the places of a vector whose bit is set.
template <typename T>
__device__ __forceinline__ uint4 mask_vec(uint4 w, uint32_t bits) {
  constexpr int n = Word<T>::kElems;
  uint32_t* p = &w.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = bits >> (i * n);
    const uint32_t m = n == 1 ? (b & 1 ? ~0u : 0u) : (b & 1 ? 0xffffu : 0u) | (b & 2 ? 0xffff0000u : 0u);
    p[i] = (p[i] & ~m) | (Word<T>::kNegInf & m);
  }
  return w;
}

// One block (or cluster) per row. The listed classes are marked by a bit each
// (a byte per vector) in shared memory, so that the streaming loop leaves
// them out at the price of one byte load per vector; their own sum comes from
// the K pairs. For 16-bit logits the exponential unit, the issue slots and
// DRAM are at 0.65 each, and the rows' ends are between them: 4096 rows of
// 131072 bf16 classes with 64 pairs 219 us, 0.75 of a copy's rate, 204 us
// without a rest and one pair; 4096 of 65536 fp32 185 us (0.89).
// ROUNDED: a rest with 16-bit log-probabilities. Their noise takes registers
// that the others cannot spare (220 -> 234 us for the 64 pairs above).
constexpr int kBatch = 4, kStages = 2;
template <typename T, int NT, bool ROUNDED>
__global__ void __launch_bounds__(NT, 1024 / NT) fwd_block_kernel(Args a) {
  constexpr int VE = Vec<T>::kElems, U = kBatch;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ RunShared<NT> runs;
  __shared__ Run mine, joined;
  __shared__ float2 pair_sums[4];
  __shared__ float pair_noises[4];
  __shared__ int idx[R4C_TOPK_MAX];
  uint8_t* marks = dyn + VecRing<NT, U, kStages>::kBytes;
  const int tid = threadIdx.x;
  uint32_t cs = 1, cr = 0;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cs));
  if (cs > 1) cr = cluster_rank();
  const float k = a.inv_t * kLog2e;
  double sum_loss = 0.0, sum_w = 0.0;
  auto masked = [&](int64_t row) { return a.weight && a.weight[row] == 0.f; };
  RowStream<T, NT, U, kStages, decltype(masked)> stream(dyn, static_cast<const T*>(a.z), a.v, a.nrows, a.C, (int)cs,
                                                        (int)cr, masked);
  if (a.rest) {
    const int bytes = ((a.C + 2 * VE) / VE + (int)cs) / (int)cs + 8;
    for (int i = tid; i < bytes / 4 + 1; i += NT) reinterpret_cast<uint32_t*>(marks)[i] = 0;
  }
  __syncthreads();
  for (int64_t r = blockIdx.x / cs; r < a.nrows; r += stream.step) {
    const VecRow<T> x(static_cast<const T*>(a.z) + a.v.base(r), a.C);
    int v0, v1, f0, f1;
    stream.share(x, &v0, &v1, &f0, &f1);
    float w = a.weight ? a.weight[r] : 1.f;
    // the pairs; each class's first pair stands for it in the sums
    int c = -1;
    float v = 0.f;
    if (tid < a.K) {
      v = teacher_logp<false>(a, r * a.K, tid);
      c = teacher_class<false>(a, r * a.K, tid, v);
      idx[tid] = c;
    }
    const bool any = __syncthreads_or(c >= 0);
    if (w == 0.f || !any) {   // the same for all blocks of the cluster
      if (w != 0.f) {         // its vectors are on their way all the same
        uint4 y4[U];
        for (int left = f1 - f0; left > 0; left -= U * NT) stream.take(y4);
      }
      if (cr == 0 && tid == 0) {
        if (a.row_loss) a.row_loss[r] = 0.f;
        a.stats[r].w = 0.f;
      }
      __syncthreads();
      continue;
    }
    float zc = -INFINITY;
    bool first = c >= 0;
    int mark = -1;
    if (c >= 0) {
      zc = Elem<T>::to_f(x.row[c]);
      for (int i = 0; i < tid; ++i)
        if (idx[i] == c) first = false;
      if (a.rest) {
        const int vec = (c + x.off) / VE;
        if (vec >= v0 && vec < v1) {
          mark = (vec - v0) * 8 + (c + x.off) % VE;
          atomicOr(reinterpret_cast<uint32_t*>(marks) + (mark >> 5), 1u << (mark & 31));
        }
      }
    }
    __syncthreads();
    Run2 part = run2_empty();
    const uint8_t* mk = marks + (f0 - v0 + tid);
    for (int left = f1 - f0; left > 0; left -= U * NT, mk += U * NT) {
      uint4 y4[U];
      stream.take(y4);
      if (left >= U * NT) {
        if (a.rest) {
#pragma unroll
          for (int i = 0; i < U; ++i)
            if (const uint32_t b = mk[i * NT]) y4[i] = mask_vec<T>(y4[i], b);
        }
        float vm = Vec<T>::top(y4[0]);
#pragma unroll
        for (int i = 1; i < U; ++i) vm = fmaxf(vm, Vec<T>::top(y4[i]));
        run2_raise<false>(part, vm, k);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          float y[VE];
          Vec<T>::split(y4[i], y);
          run2_add<VE, false>(part, y, k);
        }
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (tid + i * NT >= left) break;
          if (a.rest)
            if (const uint32_t b = mk[i * NT]) y4[i] = mask_vec<T>(y4[i], b);
          run2_raise<false>(part, Vec<T>::top(y4[i]), k);
          float y[VE];
          Vec<T>::split(y4[i], y);
          run2_add<VE, false>(part, y, k);
        }
      }
    }
    auto edge = [&](int vec, int j) {   // one element of a partial vector
      const int e = x.cls(vec) + j;
      if (e >= 0 && e < a.C && !(a.rest && (marks[vec - v0] >> j & 1)))
        run2_one<false>(part, Elem<T>::to_f(x.row[e]), k);
    };
    if (f0 > v0 && tid < VE) edge(v0, tid);
    if (f1 < v1 && f1 >= f0 && tid >= NT - VE) edge(f1, tid - (NT - VE));
    Run run = run_block<NT>(part.join(), k, runs);
    if (mark >= 0) reinterpret_cast<uint32_t*>(marks)[mark >> 5] = 0;
    if (cs > 1) {
      if (tid == 0) mine = run;
      cluster_sync();
      if (cr == 0) {
        if (tid < 32) {
          run = run_cluster(&mine, (int)cs, k);
          if (tid == 0) joined = run;
        }
        __syncthreads();
        run = joined;
      }
    }
    if (cr == 0) {
      Run l{first ? zc : -INFINITY, first && zc != -INFINITY ? 1.f : 0.f, 0.f};
      if (isnan(zc)) l = {0.f, zc, 0.f};
      if (a.rest) l = run_block<NT>(l, k, runs);
      const RowSums s(run, l, a.rest, k);
      // renormalised: ln sum exp(v) of the pairs, by the same joining
      float q0 = 0.f, qs = 1.f;
      if (!a.rest) {
        const Run q = run_block<NT>(Run{c >= 0 ? v : -INFINITY, c >= 0 ? 1.f : 0.f, 0.f}, kLog2e, runs);
        q0 = q.m;
        qs = q.s;
      }
      float q = 0.f, loss = 0.f;
      if (c >= 0) {
        q = prob(v - q0) / qs;
        if (!(q == 0.f)) loss = q * ((v - q0) - kLn2 * log2f(qs) - (zc - s.m) * a.inv_t + kLn2 * log2f(s.s));
      }
      __syncthreads();
      // (the sums of K <= 128 numbers: the first four warps hold them)
      if (ROUNDED) {
        const float noise = group_sum<32>(pair_noise(q, v, a.t_round));
        if ((tid & 31) == 0 && tid < 128) pair_noises[tid >> 5] = noise;
      }
      q = group_sum<32>(q);
      loss = group_sum<32>(loss);
      if ((tid & 31) == 0 && tid < 128) pair_sums[tid >> 5] = make_float2(q, loss);
      __syncthreads();
      if (tid == 0) {
        float sum_q = 0.f;
        loss = 0.f;
        for (int i = 0; i < 4 && i < NT / 32; ++i) {
          sum_q += pair_sums[i].x;
          loss += pair_sums[i].y;
        }
        float noise = 0.f;
        if (ROUNDED && s.sr == 0.f)
          for (int i = 0; i < 4 && i < NT / 32; ++i) noise += pair_noises[i];
        const float qr = a.rest ? rest_mass(sum_q, noise) : 0.f;
        if (s.empty) w = 0.f;
        loss = w == 0.f ? 0.f : w * a.temp * a.temp * (loss + rest_loss(qr, s, a.inv_t));
        if (a.row_loss) a.row_loss[r] = loss;
        sum_loss += loss;
        sum_w += w;
        a.stats[r] = {s.m, s.s, s.mr, s.sr, q0, qs, a.rest ? sum_q + qr : 1.f, qr, w};
      }
    }
    if (cs > 1) cluster_sync();
    else __syncthreads();
  }
  if (a.part) leave_part<NT>(sum_loss, sum_w, a);
}

// Elementwise from the row's saved sums, one block per piece of a row; the
// listed classes are written over at the end. Memory bounds it: 4096 rows of
// 131072 bf16 classes 326 us, a copy's rate.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) bwd_block_kernel(Args a) {
  __shared__ int idx[R4C_TOPK_MAX];
  __shared__ float qj[R4C_TOPK_MAX];
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / a.segs;
  T* dz = static_cast<T*>(a.dz) + a.dv.base(r);
  extern __shared__ __align__(16) uint8_t ring[];
  GradPiece<T, NT> piece(static_cast<const T*>(a.z) + a.v.base(r), dz, a.C, blockIdx.x % a.segs, a.segs, ring);
  const Stats st = a.stats[r];
  if (st.w == 0.f) {
    piece.write([](float2) { return make_float2(0.f, 0.f); });
    return;
  }
  int c = -1;
  if (tid < a.K) {
    const float v = teacher_logp<false>(a, r * a.K, tid);
    c = teacher_class<false>(a, r * a.K, tid, v);
    idx[tid] = c;
    qj[tid] = c < 0 ? 0.f : prob(v - st.qm) / st.qs;
  }
  const float k = a.inv_t * kLog2e, scale = st.w * grad_scale(a, r), mr = a.rest ? st.mr : st.m;
  const float coef = scale * rest_coef(a.rest, st.mass, st.q_rest, st.m, st.s, st.mr, st.sr, k);
  const float2 m2 = {-mr, -mr}, k2 = {k, k}, c2 = {coef, coef};
  piece.write([&](float2 z) {
    const float2 t = __fmul2_rn(__fadd2_rn(z, m2), k2);
    return __fmul2_rn(make_float2(ex2(t.x), ex2(t.y)), c2);
  });
  __syncthreads();   // the block's own stores come before these
  if (c >= 0 && piece.has(c)) {
    float q = 0.f;
    bool first = true;
    for (int i = 0; i < a.K; ++i) {
      if (idx[i] != c) continue;
      if (i < tid) first = false;
      q += qj[i];
    }
    const float p = prob((Elem<T>::to_f(piece.x.row[c]) - st.m) * a.inv_t) / st.s;
    if (first) dz[c] = Elem<T>::from_f(scale * (st.mass * p - q));
  }
}

// loss = sum w L / sum w, total_weight = sum w: the blocks' partial sums in a fixed order.
constexpr int kMeanThreads = 256;
__global__ void __launch_bounds__(kMeanThreads) mean_kernel(const double* part, int n, float* loss, float* total_weight) {
  __shared__ double sh[2][kMeanThreads];
  double s = 0.0, w = 0.0;
  for (int i = threadIdx.x; i < n; i += kMeanThreads) {
    s += part[2 * i];
    w += part[2 * i + 1];
  }
  sh[0][threadIdx.x] = s;
  sh[1][threadIdx.x] = w;
  __syncthreads();
  for (int off = kMeanThreads / 2; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) {
      sh[0][threadIdx.x] += sh[0][threadIdx.x + off];
      sh[1][threadIdx.x] += sh[1][threadIdx.x + off];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    loss[0] = (float)(sh[0][0] / sh[1][0]);   // no row takes part: NaN
    total_weight[0] = (float)sh[1][0];
  }
}

// ---- launches ----------------------------------------------------------------
// Shared memory for the marks of a block's share of the vectors.
template <typename T>
size_t mark_bytes(int C, int cs) {
  return (size_t)((C + 2 * Vec<T>::kElems) / Vec<T>::kElems + cs) / cs + 16;
}
constexpr size_t kMostMarks = 128 << 10;

template <typename T, int NT, bool ROUNDED>
cudaError_t launch_fwd_rows(const Args& a, int* blocks, cudaStream_t s) {
  int cs = cluster_size(a.nrows, a.C, sizeof(T), NT);
  while (a.rest && cs < 8 && mark_bytes<T>(a.C, cs) > kMostMarks) cs *= 2;
  const size_t smem = VecRing<NT, kBatch, kStages>::kBytes + (a.rest ? mark_bytes<T>(a.C, cs) : 0);
  const int64_t most = (int64_t)kSMs * blocks_per_sm(fwd_block_kernel<T, NT, ROUNDED>, NT, smem) / cs * cs;
  int64_t grid = a.nrows * cs;
  if (grid > most) grid = most;   // (0: launch_cluster gives the error)
  *blocks = (int)grid;
  return launch_cluster(fwd_block_kernel<T, NT, ROUNDED>, grid, NT, cs, smem, s, a);
}
template <typename T, int NT>
cudaError_t launch_fwd_block(const Args& a, int* blocks, cudaStream_t s) {
  return a.rest && a.t_round > 0.f ? launch_fwd_rows<T, NT, true>(a, blocks, s) : launch_fwd_rows<T, NT, false>(a, blocks, s);
}

template <typename T>
cudaError_t launch_fwd(Args& a, int* blocks, cudaStream_t s) {
  if (a.C <= kTileClasses) return launch_tiles<T>(a, false, blocks, s);
  if (row_threads(a.C, sizeof(T), a.K) == kWarpRow) return launch_fwd_block<T, kWarpRow>(a, blocks, s);
  return launch_fwd_block<T, kLongRow>(a, blocks, s);
}
template <typename T>
cudaError_t launch_bwd(Args& a, cudaStream_t s) {
  int blocks;
  if (a.C <= kTileClasses) return launch_tiles<T>(a, true, &blocks, s);
  const int threads = row_threads(a.C, sizeof(T), a.K) == kWarpRow ? kWarpRow : kGradRow;
  a.segs = grad_pieces(a.nrows, a.C, sizeof(T), threads);
  if (a.nrows * a.segs > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (threads == kWarpRow)
    return launch_cluster(bwd_block_kernel<T, kWarpRow>, a.nrows, kWarpRow, 1,
                          VecRing<kWarpRow, kGradBatch, kGradStages>::kBytes, s, a);
  return launch_cluster(bwd_block_kernel<T, kGradRow>, a.nrows * a.segs, kGradRow, 1,
                        VecRing<kGradRow, kGradBatch, kGradStages>::kBytes, s, a);
}

}  // namespace distill
}  // namespace r4c

using namespace r4c;

namespace {
int check(const r4c_rows_desc* d, int k, const void* t_logp, int t_dtype, const void* t_index, int index_bits, int rest) {
  if (!rows::valid_desc(d) || k <= 0 || (index_bits != 32 && index_bits != 64)) return R4C_ERR_INVALID;
  if (d->rows > 0 && (!t_logp || !t_index)) return R4C_ERR_INVALID;
  if (!rows::valid_dtype(d->dtype) || !rows::valid_dtype(t_dtype)) return R4C_ERR_UNSUPPORTED;
  if (d->classes > rows::kTileClasses && (d->class_stride != 1 || d->grad_class_stride != 1)) return R4C_ERR_UNSUPPORTED;
  if (k > R4C_TOPK_MAX) return R4C_ERR_TOO_LARGE;
  // the marks of the listed classes, spread over a cluster of 8 blocks
  if (rest && distill::mark_bytes<float>(d->classes, 8) > distill::kMostMarks) return R4C_ERR_TOO_LARGE;
  return R4C_OK;
}
// The state: the blocks' partial sums, the sum of weights, the rows' statistics.
constexpr size_t kTotalAt = (size_t)distill::kParts * 2 * sizeof(double), kStatsAt = kTotalAt + 16;

distill::Args make_args(const r4c_rows_desc* d, const void* logits, int k, const void* t_logp, int t_dtype,
                        const void* t_index, int index_bits, int rest, const float* weight, void* state) {
  distill::Args a{};
  a.z = logits;
  a.v = rows::make_view(d);
  a.dv = rows::make_grad_view(d);
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
  a.t_round = t_dtype == R4C_BF16 ? 0x1p-8f : t_dtype == R4C_F16 ? 0x1p-11f : 0.f;
  a.weight = weight;
  a.stats = reinterpret_cast<distill::Stats*>(static_cast<char*>(state) + kStatsAt);
  return a;
}
}  // namespace

extern "C" size_t r4c_distill_state_size(const r4c_rows_desc* d) {
  if (!rows::valid_desc(d)) return 0;
  return kStatsAt + (d->classes <= rows::kTileClasses ? 0 : (size_t)d->rows * sizeof(distill::Stats));
}

extern "C" int r4c_distill_fwd(const r4c_rows_desc* d, const void* logits, int k, const void* teacher_logp,
                               int teacher_dtype, const void* teacher_index, int index_bits, int rest,
                               const float* weight, float* row_loss, float* loss, void* state, size_t state_bytes,
                               r4c_stream_t stream) {
  const int rc = check(d, k, teacher_logp, teacher_dtype, teacher_index, index_bits, rest);
  if (rc != R4C_OK) return rc;
  if (d->rows == 0 && !loss) return R4C_OK;
  if ((!row_loss && !loss) || (d->rows > 0 && !logits)) return R4C_ERR_INVALID;
  if (!state || state_bytes < r4c_distill_state_size(d)) return R4C_ERR_WORKSPACE;
  if ((uintptr_t)state & 15) return R4C_ERR_ALIGN;
  distill::Args a = make_args(d, logits, k, teacher_logp, teacher_dtype, teacher_index, index_bits, rest, weight, state);
  a.err = tc::device_error_flag();
  if (!a.err) return R4C_ERR_NO_DEVICE;
  a.row_loss = row_loss;
  a.part = loss ? static_cast<double*>(state) : nullptr;
  a.loss = loss;
  a.total = reinterpret_cast<float*>(static_cast<char*>(state) + kTotalAt);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  int blocks = 0;
  if (d->rows > 0) {
    if (d->dtype == R4C_BF16) e = distill::launch_fwd<__nv_bfloat16>(a, &blocks, s);
    else if (d->dtype == R4C_F16) e = distill::launch_fwd<__half>(a, &blocks, s);
    else e = distill::launch_fwd<float>(a, &blocks, s);
    note_launches(1);
  }
  if (e == cudaSuccess && loss && blocks != 1) {
    distill::mean_kernel<<<1, distill::kMeanThreads, 0, s>>>(a.part, blocks, loss, a.total);
    e = cudaGetLastError();
    note_launches(1);
  }
  return rows::status(e);
}

extern "C" int r4c_distill_bwd(const r4c_rows_desc* d, const void* logits, int k, const void* teacher_logp,
                               int teacher_dtype, const void* teacher_index, int index_bits, int rest,
                               const float* weight, int mean, const float* grad, int grad_inc, const void* state,
                               void* dlogits, r4c_stream_t stream) {
  const int rc = check(d, k, teacher_logp, teacher_dtype, teacher_index, index_bits, rest);
  if (rc != R4C_OK) return rc;
  if (d->rows == 0) return R4C_OK;
  if (!logits || !dlogits || !grad || !state) return R4C_ERR_INVALID;
  distill::Args a = make_args(d, logits, k, teacher_logp, teacher_dtype, teacher_index, index_bits, rest, weight,
                              const_cast<void*>(state));
  a.err = tc::device_error_flag();
  if (!a.err) return R4C_ERR_NO_DEVICE;
  a.total_weight = mean ? reinterpret_cast<const float*>(static_cast<const char*>(state) + kTotalAt) : nullptr;
  a.grad = grad;
  a.grad_inc = grad_inc;
  a.dz = dlogits;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d->dtype == R4C_BF16) e = distill::launch_bwd<__nv_bfloat16>(a, s);
  else if (d->dtype == R4C_F16) e = distill::launch_bwd<__half>(a, s);
  else e = distill::launch_bwd<float>(a, s);
  note_launches(1);
  return rows::status(e);
}
