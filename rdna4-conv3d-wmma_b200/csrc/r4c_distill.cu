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

struct Stats {           // per streamed row, written by the forward for the backward
  float m, s;            // lse = m / T + ln s (m a logit, not yet scaled)
  float mr, sr;          // the same over the unlisted classes
  float qm, qs;          // q_j = exp(v_j - qm) / qs
  float mass, q_rest;    // Q, q_r
  float w;               // the row's weight, 0: takes no part
};

constexpr int kParts = kSMs * 16;   // most blocks of a forward: each leaves one partial sum

struct Args {
  const void* z;
  View v, dv;
  Tile tile;
  int64_t nrows;
  int C, K, rest, segs;
  float temp, inv_t;
  const void* t_logp;
  const void* t_index;
  int t_dtype, t_wide;
  const float* weight;
  float* row_loss;       // forward: w L per row, or null
  double* part;          // forward: (sum w L, sum w) of each block, or null
  Stats* stats;
  const float* total_weight;
  const float* grad;
  int grad_inc;
  void* dz;
  int* err;
};

__device__ __forceinline__ float teacher_logp(const Args& a, int64_t i) {
  if (a.t_dtype == R4C_F32) return __ldg(static_cast<const float*>(a.t_logp) + i);
  if (a.t_dtype == R4C_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.t_logp)[i]);
  return __half2float(static_cast<const __half*>(a.t_logp)[i]);
}
// The pair's class, -1 when the pair is void.
__device__ __forceinline__ int teacher_class(const Args& a, int64_t i, float v) {
  const int64_t c = a.t_wide ? __ldg(static_cast<const long long*>(a.t_index) + i)
                             : (int64_t)__ldg(static_cast<const int32_t*>(a.t_index) + i);
  if (c < 0 || v == -INFINITY) return -1;
  if (c >= a.C) {
    atomicExch(a.err, 6);
    return -1;
  }
  return (int)c;
}
__device__ __forceinline__ float grad_scale(const Args& a, int64_t r, float w) {
  return a.temp * w * a.grad[r * a.grad_inc] / (a.total_weight ? a.total_weight[0] : 1.f);
}
// A block's (sum of losses, sum of weights), in a fixed order.
template <int NT>
__device__ __forceinline__ void leave_part(double loss, double w, double* part) {
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
    part[2 * blockIdx.x] = loss;
    part[2 * blockIdx.x + 1] = w;
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
    const Run all = rest ? run_merge(r, l, k) : r;
    empty = all.s == 0.f;
    m = anchor(all.m);
    s = all.s;
    mr = anchor(r.m);
    sr = r.s;
  }
};
// q_r from the sum of the listed q.
__device__ __forceinline__ float rest_mass(float sum_q) {
  const float qr = 1.f - sum_q;
  return qr >= kRestNoise ? qr : 0.f;
}
// q_r (ln q_r - ln p_r)
__device__ __forceinline__ float rest_loss(float qr, const RowSums& s, float inv_t) {
  return qr > 0.f ? qr * (kLn2 * (__log2f(qr) - __log2f(s.sr) + __log2f(s.s)) - (s.mr - s.m) * inv_t) : 0.f;
}
// The factor of 2^t (t from mr) in the gradient of an unlisted class: (Q p_r - q_r) / sr, 0 without any.
__device__ __forceinline__ float rest_coef(bool rest, float mass, float qr, float m, float s, float mr, float sr, float k) {
  if (!rest) return __fdividef(mass, s);
  return sr == 0.f ? 0.f : mass * ex2((mr - m) * k) / s - qr / sr;
}
// The pairs' exponentials: few, and their difference from the student's is the gradient.
__device__ __forceinline__ float prob(float ln_q) { return expf(ln_q); }

// ---- rows in registers -------------------------------------------------------
// The teacher's pairs of a row, lane l of the group taking pairs l, l + G,
// ...; the first kSlots of a lane stay in registers, more are read again.
constexpr int kSlots = 2;
struct Pair {
  float v, z;   // the teacher's log-probability, the student's logit
  int c;        // class, -1: void
};

template <typename T, int G, int E, bool VEC, bool BWD>
__global__ void __launch_bounds__(kTileThreads) tile_kernel(Args a) {
  constexpr int ES = (int)sizeof(T);
  const float k = a.inv_t * kLog2e;
  const bool rest = a.rest;
  double sum_loss = 0.0, sum_w = 0.0;
  tile_walk<T, G, BWD>(a.tile, a.v, a.z, a.dv, a.dz, [&](int64_t r, uint32_t row, bool in) {
    const int lane = threadIdx.x & (G - 1);
    const int64_t p0 = r * a.K;
    float w = a.weight ? a.weight[r] : 1.f;
    auto read = [&](int j) {   // from memory: the row in shared memory changes below
      Pair p;
      p.v = teacher_logp(a, p0 + j);
      p.c = teacher_class(a, p0 + j, p.v);
      return p;
    };
    auto logit = [&](int c) { return Elem<T>::to_f(static_cast<const T*>(a.z)[a.v.base(r) + c * a.v.sc]); };
    Pair held[kSlots];
    float qm = -INFINITY;
    bool any = false;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      held[s].c = -1;
      if (s * G < a.K && lane + s * G < a.K) {
        held[s] = read(lane + s * G);
        if (held[s].c >= 0) {
          held[s].z = sh_get<T>(row + held[s].c * ES);
          qm = fmaxf(qm, held[s].v);
          any = true;
        }
      }
    }
    for (int j = lane + kSlots * G; j < a.K; j += G) {
      const Pair p = read(j);
      if (p.c >= 0) {
        qm = fmaxf(qm, p.v);
        any = true;
      }
    }
    if (G > 1) any = group_any<G>(any);
    if (!any) w = 0.f;
    // f(pair, its number) for each valid pair of this lane
    auto pairs = [&](auto&& f) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (s * G < a.K && held[s].c >= 0) f(held[s], lane + s * G);
      for (int j = lane + kSlots * G; j < a.K; j += G) {
        Pair p = read(j);
        if (p.c < 0) continue;
        p.z = logit(p.c);
        f(p, j);
      }
    };
    // Is a class listed twice? Each pair leaves its number at its class and
    // looks whether it is still there; the logits are put back after that.
    bool twice = false;
    if ((rest || BWD) && a.K > 1) {
      __syncwarp();
      if (in) pairs([&](const Pair& p, int j) { sh_put<T>(row + p.c * ES, (float)(j + 1)); });
      __syncwarp();
      if (in) pairs([&](const Pair& p, int j) { twice |= sh_get<T>(row + p.c * ES) != (float)(j + 1); });
      if (G > 1) twice = group_any<G>(twice);
      __syncwarp();
    }
    // With a rest the listed classes leave the row; their own sum comes from the pairs.
    if ((rest || BWD) && in && (rest || a.K > 1))
      pairs([&](const Pair& p, int) { sh_put<T>(row + p.c * ES, rest ? -INFINITY : p.z); });
    __syncwarp();
    TileRow<T, G, E, VEC> x;
    x.load(row, a.C);
    if (G > 1) __syncwarp();   // read by all before any of it is written over
    auto first = [&](const Pair& p, int j) {   // of the pairs with this class
      if (!twice) return true;
      for (int i = 0; i < j; ++i)
        if (read(i).c == p.c) return false;
      return true;
    };
    Run u = run_empty(), l = run_empty();
    {
      Run2 part = run2_empty();
      part.m = x.max();
      run2_add<E, false>(part, x.v, k);
      u = part.join();
      u.s = group_sum<G>(u.s);
    }
    if (rest) {
      pairs([&](const Pair& p, int) { l.m = fmaxf(l.m, p.z); });
      l.m = group_max<G>(l.m);
      const float lm = anchor(l.m);
      pairs([&](const Pair& p, int j) { if (first(p, j)) l.s += ex2((p.z - lm) * k); });
      l.s = group_sum<G>(l.s);
    }
    const RowSums s(u, l, rest, k);
    if (s.empty) w = 0.f;
    float q0 = 0.f, qi = 1.f;   // q_j = exp(v_j - q0) qi
    if (!rest) {
      float qs = 0.f;
      q0 = anchor(group_max<G>(qm));
      pairs([&](const Pair& p, int) { qs += prob(p.v - q0); });
      qi = 1.f / group_sum<G>(qs);
    }
    float sum_q = 1.f, qr = 0.f;
    if (rest) {
      sum_q = 0.f;
      pairs([&](const Pair& p, int) { sum_q += prob(p.v); });
      sum_q = group_sum<G>(sum_q);
      qr = rest_mass(sum_q);
    }
    if constexpr (!BWD) {
      const float c0 = kLn2 * (__log2f(qi) + __log2f(s.s)) - q0;
      float loss = 0.f;
      pairs([&](const Pair& p, int) {
        const float q = prob(p.v - q0) * qi;
        if (!(q == 0.f)) loss += q * (p.v + c0 - (p.z - s.m) * a.inv_t);
      });
      loss = group_sum<G>(loss) + rest_loss(qr, s, a.inv_t);
      if (in && lane == 0) {
        loss = w == 0.f ? 0.f : w * a.temp * a.temp * loss;
        if (a.row_loss) a.row_loss[r] = loss;
        sum_loss += loss;
        sum_w += w;
      }
    } else {
      const float scale = w == 0.f ? 0.f : grad_scale(a, r, w), mass = rest ? sum_q + qr : 1.f;
      const float coef = w == 0.f ? 0.f : scale * rest_coef(rest, mass, qr, s.m, s.s, s.mr, s.sr, k);
      const float2 m2 = {-s.mr, -s.mr}, k2 = {k, k}, c2 = {coef, coef};
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 t = __fmul2_rn(__fadd2_rn(make_float2(x.v[e], x.v[e + 1]), m2), k2);
        const float2 g = __fmul2_rn(make_float2(ex2(t.x), ex2(t.y)), c2);
        x.v[e] = w == 0.f ? 0.f : g.x;
        x.v[e + 1] = w == 0.f ? 0.f : g.y;
      }
      if (in) x.store(x.v);
      __syncwarp();
      if (in && w != 0.f) {
        const float mass_s = mass / s.s;
        pairs([&](const Pair& p, int j) {
          float q = prob(p.v - q0) * qi;
          if (twice) {   // the class's first pair writes, with all its q
            if (!first(p, j)) return;
            q = 0.f;
            for (int i = 0; i < a.K; ++i) {
              const Pair o = read(i);
              if (o.c == p.c) q += prob(o.v - q0) * qi;
            }
          }
          sh_put<T>(row + p.c * ES, scale * (mass_s * prob((p.z - s.m) * a.inv_t) - q));
        });
      }
    }
  });
  if (!BWD && a.part) leave_part<kTileThreads>(sum_loss, sum_w, a.part);
}

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
// the K pairs.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) fwd_block_kernel(Args a) {
  constexpr int VE = Vec<T>::kElems, U = 4;
  extern __shared__ __align__(16) uint8_t marks[];
  __shared__ Run runs[NT / 32];
  __shared__ Run mine;
  __shared__ int idx[R4C_TOPK_MAX];
  const int tid = threadIdx.x;
  uint32_t cs = 1, cr = 0;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cs));
  if (cs > 1) cr = cluster_rank();
  const float k = a.inv_t * kLog2e;
  double sum_loss = 0.0, sum_w = 0.0;
  if (a.rest) {
    const int bytes = ((a.C + 2 * VE) / VE + (int)cs) / (int)cs + 8;
    for (int i = tid; i < bytes / 4 + 1; i += NT) reinterpret_cast<uint32_t*>(marks)[i] = 0;
  }
  __syncthreads();
  for (int64_t r = blockIdx.x / cs; r < a.nrows; r += gridDim.x / cs) {
    const VecRow<T> x(static_cast<const T*>(a.z) + a.v.base(r), a.C);
    const int per = (x.nv + (int)cs - 1) / (int)cs;
    const int v0 = min((int)cr * per, x.nv), v1 = min(v0 + per, x.nv);
    const int f0 = max(v0, x.first_full()), f1 = min(v1, x.end_full());
    float w = a.weight ? a.weight[r] : 1.f;
    // the pairs; each class's first pair stands for it in the sums
    int c = -1;
    float v = 0.f;
    if (tid < a.K) {
      v = teacher_logp(a, r * a.K + tid);
      c = teacher_class(a, r * a.K + tid, v);
      idx[tid] = c;
    }
    const bool any = __syncthreads_or(c >= 0);
    if (!any || w == 0.f) {   // the same for all blocks of the cluster
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
    int at = f0 + tid;
    const uint4* p = x.p + at;
    const uint8_t* mk = marks + (at - v0);
    for (; at + (U - 1) * NT < f1; at += U * NT, p += U * NT, mk += U * NT) {
      uint4 y4[U];
#pragma unroll
      for (int i = 0; i < U; ++i) y4[i] = __ldg(p + i * NT);
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
    }
    for (; at < f1; at += NT, p += NT, mk += NT) {
      uint4 y4 = __ldg(p);
      if (a.rest)
        if (const uint32_t b = *mk) y4 = mask_vec<T>(y4, b);
      run2_raise<false>(part, Vec<T>::top(y4), k);
      float y[VE];
      Vec<T>::split(y4, y);
      run2_add<VE, false>(part, y, k);
    }
    auto edge = [&](int vec, int j) {   // one element of a partial vector
      const int e = x.cls(vec) + j;
      if (e >= 0 && e < a.C && !(a.rest && (marks[vec - v0] >> j & 1)))
        run2_one<false>(part, Elem<T>::to_f(x.row[e]), k);
    };
    if (f0 > v0 && tid < VE) edge(v0, tid);
    if (f1 < v1 && f1 >= f0 && tid >= 32 && tid < 32 + VE) edge(f1, tid - 32);
    Run run = run_block<NT>(part.join(), k, runs);
    if (mark >= 0) reinterpret_cast<uint32_t*>(marks)[mark >> 5] = 0;
    if (cs > 1) {
      if (tid == 0) mine = run;
      cluster_sync();
      if (cr == 0)
        for (uint32_t q = 1; q < cs; ++q) run = run_merge(run, cluster_ld_run(&mine, q), k);
    }
    if (cr == 0) {
      __syncthreads();   // runs is free again
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
      q = group_sum<32>(q);
      loss = group_sum<32>(loss);
      if ((tid & 31) == 0) runs[tid >> 5] = {q, loss, 0.f};
      __syncthreads();
      if (tid == 0) {
        float sum_q = 0.f;
        loss = 0.f;
        for (int i = 0; i < 4; ++i) {
          sum_q += runs[i].m;
          loss += runs[i].s;
        }
        const float qr = a.rest ? rest_mass(sum_q) : 0.f;
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
  if (a.part) leave_part<NT>(sum_loss, sum_w, a.part);
}

// One block per piece of a row; the listed classes are written over at the end.
template <typename T>
__global__ void __launch_bounds__(kGradThreads) bwd_block_kernel(Args a) {
  __shared__ int idx[R4C_TOPK_MAX];
  __shared__ float qj[R4C_TOPK_MAX];
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / a.segs;
  T* dz = static_cast<T*>(a.dz) + a.dv.base(r);
  GradPiece<T> piece(static_cast<const T*>(a.z) + a.v.base(r), dz, a.C, blockIdx.x % a.segs, a.segs);
  const Stats st = a.stats[r];
  if (st.w == 0.f) {
    piece.write([](float2) { return make_float2(0.f, 0.f); });
    return;
  }
  int c = -1;
  if (tid < a.K) {
    const float v = teacher_logp(a, r * a.K + tid);
    c = teacher_class(a, r * a.K + tid, v);
    idx[tid] = c;
    qj[tid] = c < 0 ? 0.f : prob(v - st.qm) / st.qs;
  }
  const float k = a.inv_t * kLog2e, scale = grad_scale(a, r, st.w), mr = a.rest ? st.mr : st.m;
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
template <typename T, bool BWD>
cudaError_t launch_tiles(Args& a, int* blocks, cudaStream_t s) {
  const TileKind kind = tile_kind(a.C, sizeof(T));
  a.tile = make_tile(a.nrows, a.C, sizeof(T), kind.g,
                     dense_rows(a.v, a.nrows, a.C, a.z) && (!BWD || dense_rows(a.dv, a.nrows, a.C, a.dz)));
  *blocks = tile_grid(a.tile);
  return for_tile_kind<T>(kind, [&](auto c) {
    return launch_tile(tile_kernel<T, decltype(c)::G, decltype(c)::E, decltype(c)::VEC, BWD>, a.tile, s, a);
  });
}

// Shared memory for the marks of a block's share of the vectors.
template <typename T>
size_t mark_bytes(int C, int cs) {
  return (size_t)((C + 2 * Vec<T>::kElems) / Vec<T>::kElems + cs) / cs + 16;
}
constexpr size_t kMostMarks = 160 << 10;

template <typename T, int NT>
cudaError_t launch_fwd_block(const Args& a, int* blocks, cudaStream_t s) {
  int cs = cluster_size(a.nrows, a.C, sizeof(T), NT);
  while (a.rest && cs < 16 && mark_bytes<T>(a.C, cs) > kMostMarks) cs *= 2;
  const int64_t most = (int64_t)kSMs * (1024 / NT) / cs * cs;
  int64_t grid = a.nrows * cs;
  if (grid > most) grid = most;
  *blocks = (int)grid;
  return launch_cluster(fwd_block_kernel<T, NT>, grid, NT, cs, a.rest ? mark_bytes<T>(a.C, cs) : 0, s, a);
}

template <typename T>
cudaError_t launch_fwd(Args& a, int* blocks, cudaStream_t s) {
  if (a.C <= kTileClasses) return launch_tiles<T, false>(a, blocks, s);
  if ((int64_t)a.C * sizeof(T) <= 16 << 10) return launch_fwd_block<T, 128>(a, blocks, s);
  return launch_fwd_block<T, 256>(a, blocks, s);
}
template <typename T>
cudaError_t launch_bwd(Args& a, cudaStream_t s) {
  int blocks;
  if (a.C <= kTileClasses) return launch_tiles<T, true>(a, &blocks, s);
  a.segs = grad_pieces(a.C, sizeof(T));
  if (a.nrows * a.segs > 0x7fffffff) return cudaErrorInvalidConfiguration;
  bwd_block_kernel<T><<<(unsigned)(a.nrows * a.segs), kGradThreads, 0, s>>>(a);
  return cudaGetLastError();
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
  // the marks of the listed classes, spread over a cluster of 16 blocks
  if (rest && distill::mark_bytes<float>(d->classes, 16) > distill::kMostMarks) return R4C_ERR_TOO_LARGE;
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
  if ((!row_loss && !loss) || (d->rows > 0 && !logits)) return R4C_ERR_INVALID;
  if (!state || state_bytes < r4c_distill_state_size(d)) return R4C_ERR_WORKSPACE;
  if ((uintptr_t)state & 15) return R4C_ERR_ALIGN;
  distill::Args a = make_args(d, logits, k, teacher_logp, teacher_dtype, teacher_index, index_bits, rest, weight, state);
  a.err = tc::device_error_flag();
  if (!a.err) return R4C_ERR_NO_DEVICE;
  a.row_loss = row_loss;
  a.part = loss ? static_cast<double*>(state) : nullptr;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  int blocks = 0;
  if (d->rows > 0) {
    if (d->dtype == R4C_BF16) e = distill::launch_fwd<__nv_bfloat16>(a, &blocks, s);
    else if (d->dtype == R4C_F16) e = distill::launch_fwd<__half>(a, &blocks, s);
    else e = distill::launch_fwd<float>(a, &blocks, s);
    note_launches(1);
  }
  if (e == cudaSuccess && loss) {
    distill::mean_kernel<<<1, distill::kMeanThreads, 0, s>>>(
        a.part, blocks, loss, reinterpret_cast<float*>(static_cast<char*>(state) + kTotalAt));
    e = cudaGetLastError();
    note_launches(1);
  }
  return e == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
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
  return e == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}
