// r4c_logp.cu — log-probability of a given label, entropy, log-sum-exp and
// the most probable classes of each row of logits, and the logits' gradient.
//
//   s_c = z_c / T,  m = max s,  S = sum exp(s_c - m),  lse = m + ln S
//   logp = s_t - lse,   H = ln S - (1/S) sum exp(s_c - m) (s_c - m)
//   dz_c = (1/T) [ p_c (g_lse - g_logp - g_H (ln p_c + H)) + g_logp [c = t] ],  p_c = exp(s_c - lse)
//
// The difference z_c - max z is taken before it is scaled, so rows of the
// type's lowest value stay a uniform distribution instead of overflowing.
// Both directions read each logit once and are bound by memory; the kernels
// for short and long rows are described in r4c_rows.cuh.
#include "r4c_rows.cuh"

namespace r4c {
namespace logp {

using namespace rows;

struct FwdArgs {
  const void* z;
  const int64_t* target;
  int64_t ignore, nrows;
  View v;
  Tile tile;
  int C, K, pairs;   // pairs: K = 2 and the outputs 8-byte aligned
  float inv_t;
  float *logp, *entropy, *lse, *top_logp;
  int32_t* top_index;
  float2* stats;      // (max z, S) of streamed rows
  int* err;
};

struct BwdArgs {
  const void* z;
  const int64_t* target;
  int64_t ignore, nrows;
  View v, dv;
  Tile tile;
  int C, segs;
  float inv_t;
  const float* entropy;
  const float2* stats;
  const float *g_logp, *g_entropy, *g_lse;
  int gl_inc, gh_inc, gs_inc;
  void* dz;
  int* err;
};

// The row's label, -1 when it has none or takes no part.
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

// What a row's sums say; bad: NaN or +inf in the row, empty: no finite logit.
struct RowOut {
  float mm, l2s, inv_t;
  bool bad, empty;
  __device__ __forceinline__ RowOut(const Run& r, float log2_s, float it)
      : mm(anchor(r.m)), l2s(log2_s), inv_t(it), bad(isnan(r.s)), empty(r.s == 0.f) {}
  __device__ __forceinline__ float logp(float z) const { return empty ? -INFINITY : fmaf(z - mm, inv_t, -kLn2 * l2s); }
  __device__ __forceinline__ float entropy(const Run& r) const { return empty ? 0.f : kLn2 * (l2s - __fdividef(r.u, r.s)); }
  __device__ __forceinline__ float lse() const { return fmaf(mm, inv_t, kLn2 * l2s); }
};

// ---- rows in registers -------------------------------------------------------
template <typename Row>
__device__ __forceinline__ Run row_run(const Row& x, float k) {
  Run2 r = run2_empty();
  r.m = x.max();
  run2_add<sizeof(x.v) / sizeof(float), true>(r, x.v, k);   // places outside the row hold -inf and add nothing
  return r.join();
}
template <int G>
__device__ __forceinline__ void run_group(Run& r) {
  r.s = group_sum<G>(r.s);
  r.u = group_sum<G>(r.u);
}

// Keys that order a row's values, equal ones by lowest class; the least is no
// class. 16-bit types: 19 bits of the value hold it exactly, 13 the class.
template <typename T> struct TopKey {
  using type = int;
  static constexpr int kNone = (int)0x80000000;
  static __device__ __forceinline__ int make(float v, int c) {
    const int b = __float_as_int(v + 0.f);
    return ((b ^ ((b >> 31) & 0x7fffffff)) & ~0x1fff) | (0x1fff - c);
  }
  static __device__ __forceinline__ int cls(int k) { return 0x1fff - (k & 0x1fff); }
  static __device__ __forceinline__ float value(int k) {
    const int o = (k & ~0x1fff) | (k < 0 ? 0x1fff : 0);
    return __int_as_float(o ^ ((o >> 31) & 0x7fffffff));
  }
};
template <> struct TopKey<float> {
  using type = long long;
  static constexpr long long kNone = (long long)0x8000000000000000ull;
  static __device__ __forceinline__ long long make(float v, int c) { return (long long)(rank_key(v, c) ^ 0x8000000000000000ull); }
  static __device__ __forceinline__ int cls(long long k) { return key_class((uint64_t)k); }
  static __device__ __forceinline__ float value(long long k) { return key_value((uint64_t)k ^ 0x8000000000000000ull); }
};

template <typename T, int G, int E, bool VEC>
__global__ void __launch_bounds__(kTileThreads) fwd_tile_kernel(FwdArgs a) {
  const float k = a.inv_t * kLog2e;
  tile_walk<T, G, false>(a.tile, a.v, a.z, a.v, nullptr, [&](int64_t r, uint32_t row, bool in) {
    TileRow<T, G, E, VEC> x;
    x.load(row, a.C);
    Run run = row_run(x, k);
    run_group<G>(run);
    const RowOut o(run, lg2(run.s), a.inv_t);
    if (in && x.lane == 0) {
      if (a.target) {
        const int t = label_of(a.target, r, a.C, a.ignore, a.err);
        a.logp[r] = t < 0 ? 0.f : o.logp(sh_get<T>(row + t * (int)sizeof(T)));
      }
      a.entropy[r] = o.entropy(run);
      a.lse[r] = o.lse();
    }
    if (a.K == 0) return;
    // the most probable classes, one after the other
    using Key = TopKey<T>;
    typename Key::type key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = x.ok(e) ? Key::make(x.v[e], x.cls(e)) : Key::kNone;
    float* tl = a.top_logp + r * a.K;
    int32_t* ti = a.top_index + r * a.K;
    auto next = [&](float* l, int* c) {
      typename Key::type b = key[0];
#pragma unroll
      for (int e = 1; e < E; ++e) b = key[e] > b ? key[e] : b;
#pragma unroll
      for (int q = G / 2; q; q >>= 1) {
        const typename Key::type w = __shfl_xor_sync(0xffffffffu, b, q);
        b = w > b ? w : b;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) key[e] = key[e] == b ? Key::kNone : key[e];
      *l = o.bad ? NAN : o.logp(Key::value(b));
      *c = o.bad ? -1 : Key::cls(b);
    };
    if (G == 1 && a.pairs) {   // two alternatives are stored whole: half-written sectors cost twice
      float2 l;
      int2 c;
      next(&l.x, &c.x);
      next(&l.y, &c.y);
      if (in) {
        *reinterpret_cast<float2*>(tl) = l;
        *reinterpret_cast<int2*>(ti) = c;
      }
      return;
    }
    for (int j = 0; j < a.K; ++j) {
      float l;
      int c;
      next(&l, &c);
      if (in && x.lane == 0) {
        tl[j] = l;
        ti[j] = c;
      }
    }
  });
}

template <typename T, int G, int E, bool VEC>
__global__ void __launch_bounds__(kTileThreads) bwd_tile_kernel(BwdArgs a) {
  const float k = a.inv_t * kLog2e;
  tile_walk<T, G, true>(a.tile, a.v, a.z, a.dv, a.dz, [&](int64_t r, uint32_t row, bool in) {
    TileRow<T, G, E, VEC> x;
    x.load(row, a.C);
    const int t = label_of(a.target, r, a.C, a.ignore, a.err);
    const float gl = a.g_logp && t >= 0 ? a.g_logp[r * a.gl_inc] : 0.f;
    const float gh = a.g_entropy ? a.g_entropy[r * a.gh_inc] : 0.f;
    const float gs = a.g_lse ? a.g_lse[r * a.gs_inc] : 0.f;
    Run run = row_run(x, k);
    run_group<G>(run);
    const float l2s = lg2(run.s);
    const bool none = (gl == 0.f && gh == 0.f && gs == 0.f) || run.s == 0.f;
    const float h = kLn2 * (l2s - __fdividef(run.u, run.s));
    const float f = none ? 0.f : __fdividef(a.inv_t, run.s), ca = f * (gs - gl - gh * h), cb = f * gh * kLn2;
    const float mm = -anchor(run.m), lb = cb * l2s;
    const float2 m2 = {mm, mm}, k2 = {k, k};
    // 2^t (ca - cb (t - l2s))
    const float c0 = none ? 0.f : ca + lb;
    const float2 c2 = {c0, c0}, b2 = {none ? 0.f : -cb, none ? 0.f : -cb};
    float zt = 0.f;
    if (t >= 0) zt = sh_get<T>(row + t * (int)sizeof(T));
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      float2 q = __fmul2_rn(__fadd2_rn(make_float2(x.v[e], x.v[e + 1]), m2), k2);
      q = make_float2(max_nan(q.x, kFloor), max_nan(q.y, kFloor));
      q = __fmul2_rn(make_float2(ex2(q.x), ex2(q.y)), __ffma2_rn(b2, q, c2));
      x.v[e] = q.x;
      x.v[e + 1] = q.y;
    }
    if (G > 1) __syncwarp();   // every lane has read the row (and the label's logit)
    if (in) x.store(x.v);
    if (G > 1) __syncwarp();
    if (in && t >= 0 && x.lane == 0 && !none) {
      const float q = max_nan((zt + mm) * k, kFloor);
      sh_put<T>(row + t * (int)sizeof(T), fmaf(a.inv_t, gl, ex2(q) * fmaf(-cb, q, c0)));
    }
  });
}

// ---- rows streamed -----------------------------------------------------------
constexpr int kCand = 2048;   // candidate keys a block keeps while it selects

// The K largest keys of a block's part of a row, in order, into sh.top
// (0 where the part has fewer). Each thread knows the largest value of its
// own vectors and the vector it is in; the K-th largest of those is a bound
// that at least K elements reach, and few more do, so only the vectors of
// the threads that reach it are looked at again. Keys are unique (value,
// then class), which makes the result exact whatever the ties; if elements
// crowd above the bound (more than kCand) it is raised by bisection first.
struct TopShared {
  uint64_t* cand;     // kCand
  uint64_t* top;      // R4C_TOPK_MAX
  uint64_t* keys;     // a thread's best, as a lower bound
  int* active;        // threads that reach the bound
  uint64_t tau;
  int n_active, n_cand;
};

template <typename T, int NT>
__device__ void block_topk(const VecRow<T>& x, int v0, int v1, int f0, int f1, float tm, int tv, int K, bool skip,
                           TopShared& sh) {
  constexpr int VE = Vec<T>::kElems;
  const int tid = threadIdx.x;
  const bool have = tv >= 0;
  const int nd = f1 - f0 < 0 ? 0 : f1 - f0 < NT ? f1 - f0 : NT;   // threads with a vector
  sh.keys[tid] = have ? rank_key(tm, x.cls(tv) + VE - 1) : 0;
  if (tid == 0) {
    sh.n_active = 0;
    sh.n_cand = 0;
    sh.tau = 0;
  }
  for (int j = tid; j < K; j += NT) sh.top[j] = 0;
  __syncthreads();
  if (nd >= K && tid < 32) {
    uint64_t kk[NT / 32], lo = ~0ull, hi = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      kk[i] = sh.keys[tid + 32 * i];
      hi = kk[i] > hi ? kk[i] : hi;
      if (kk[i] && kk[i] < lo) lo = kk[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const uint64_t l = __shfl_xor_sync(0xffffffffu, lo, o), h = __shfl_xor_sync(0xffffffffu, hi, o);
      lo = l < lo ? l : lo;
      hi = h > hi ? h : hi;
    }
    hi += 1;   // none reach it; all nd >= K reach lo
    const int enough = K + (K >> 1) + 4;
    int reach = nd;
    while (reach > enough && hi - lo > 1) {
      const uint64_t mid = lo + ((hi - lo) >> 1);
      int c = 0;
#pragma unroll
      for (int i = 0; i < NT / 32; ++i) c += kk[i] >= mid;
      c = __reduce_add_sync(0xffffffffu, c);
      if (c >= K) {
        lo = mid;
        reach = c;
      } else {
        hi = mid;
      }
    }
    if (tid == 0) sh.tau = lo;
  }
  __syncthreads();
  uint64_t tau = sh.tau;
  if (have && rank_key(tm, x.cls(tv)) >= tau) sh.active[atomicAdd(&sh.n_active, 1)] = tid;
  __syncthreads();
  const int iters = (f1 - f0 + NT - 1) / NT;
  const int items = skip ? 0 : sh.n_active * iters;
  // every element that reaches `bound`: kept in cand (keep) or counted
  auto scan = [&](uint64_t bound, bool keep) {
    auto look = [&](float z, int c) {
      const uint64_t key = rank_key(z, c);
      if (key >= bound) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (keep && at < kCand) sh.cand[at] = key;
      }
    };
    for (int q = tid; q < items; q += NT) {
      const int v = f0 + sh.active[q / iters] + (q % iters) * NT;
      if (v < f1) {
        float y[VE];
        Vec<T>::split(__ldg(x.p + v), y);
#pragma unroll
        for (int i = 0; i < VE; ++i) look(y[i], x.cls(v) + i);
      }
    }
    if (!skip) {   // the partial vectors at the row's ends
      if (f0 > v0 && tid < VE) {
        const int c = x.cls(v0) + tid;
        if (c >= 0 && c < x.C) look(Elem<T>::to_f(x.row[c]), c);
      }
      if (f1 < v1 && f1 >= f0 && tid >= 32 && tid < 32 + VE) {
        const int c = x.cls(f1) + tid - 32;
        if (c >= 0 && c < x.C) look(Elem<T>::to_f(x.row[c]), c);
      }
    }
    __syncthreads();
    const int n = sh.n_cand;
    __syncthreads();
    if (tid == 0) sh.n_cand = 0;
    __syncthreads();
    return n;
  };
  int n = scan(tau, true);
  if (n > kCand) {
    uint64_t lo = tau, hi = ~0ull;
    while (hi - lo > 1) {
      const uint64_t mid = lo + ((hi - lo) >> 1);
      const int c = scan(mid, false);
      if (c >= K) {
        lo = mid;
        if (c <= kCand) break;
      } else {
        hi = mid;
      }
    }
    n = scan(lo, true);
    n = n < kCand ? n : kCand;
  }
  for (int i = tid; i < n; i += NT) {
    const uint64_t key = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.cand[j] > key;
    if (rank < K) sh.top[rank] = key;
  }
  __syncthreads();
}

#ifndef KS
#define KS 2
#endif
constexpr int kBatch = 4, kStages = KS;
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT) fwd_block_kernel(FwdArgs a) {
  constexpr int VE = Vec<T>::kElems, U = kBatch;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ RunShared<NT> runs;
  __shared__ Run mine;
  __shared__ TopShared top;
  const int tid = threadIdx.x;
  uint32_t cs = 1, cr = 0;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cs));
  if (cs > 1) cr = cluster_rank();
  if (TOP && tid == 0) {
    top.cand = reinterpret_cast<uint64_t*>(dyn + VecRing<NT, U, kStages>::kBytes);
    top.top = top.cand + kCand;
    top.keys = top.top + R4C_TOPK_MAX;
    top.active = reinterpret_cast<int*>(top.keys + NT);
  }
  __syncthreads();
  const float k = a.inv_t * kLog2e;
  auto none = [](int64_t) { return false; };
  RowStream<T, NT, U, kStages, decltype(none)> stream(dyn, static_cast<const T*>(a.z), a.v, a.nrows, a.C, (int)cs, (int)cr,
                                                      none);
  for (int64_t r = blockIdx.x / cs; r < a.nrows; r += stream.step) {
    const VecRow<T> x(static_cast<const T*>(a.z) + a.v.base(r), a.C);
    int v0, v1, f0, f1;
    stream.share(x, &v0, &v1, &f0, &f1);
    Run2 part = run2_empty();
    float tm = 0.f;   // the largest value of this thread's full vectors, and the first vector that has it
    int tv = -1;
    auto track = [&](float vm, int v) {
      if (TOP && (tv < 0 || vm > tm)) {
        tm = vm;
        tv = v;
      }
    };
    int v = f0 + tid;
    for (int left = f1 - f0; left > 0; left -= U * NT, v += U * NT) {
      uint4 w[U];
      stream.take(w);
      if (left >= U * NT) {
        float vm[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          vm[i] = Vec<T>::top(w[i]);
          track(vm[i], v + i * NT);
        }
        run2_raise<true>(part, fmaxf(fmaxf(vm[0], vm[1]), fmaxf(vm[2], vm[3])), k);
        run2_batch<VE, U>(part, k, [&](int i, float* y) { Vec<T>::split(i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3], y); });
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (v + i * NT >= f1) break;
          const float vm = Vec<T>::top(w[i]);
          track(vm, v + i * NT);
          run2_raise<true>(part, vm, k);
          run2_batch<VE, 1>(part, k, [&](int, float* y) { Vec<T>::split(w[i], y); });
        }
      }
    }
    if (f0 > v0 && tid < VE) {   // partial vectors: one element a thread
      const int c = x.cls(v0) + tid;
      if (c >= 0 && c < a.C) run2_one<true>(part, Elem<T>::to_f(x.row[c]), k);
    }
    if (f1 < v1 && f1 >= f0 && tid >= 32 && tid < 32 + VE) {
      const int c = x.cls(f1) + tid - 32;
      if (c >= 0 && c < a.C) run2_one<true>(part, Elem<T>::to_f(x.row[c]), k);
    }
    Run run = run_block<NT>(part.join(), k, runs);
    if (TOP) block_topk<T, NT>(x, v0, v1, f0, f1, tm, tv, a.K, isnan(run.s), top);
    if (cs > 1) {
      if (tid == 0) mine = run;
      cluster_sync();
      if (cr == 0) {
        for (uint32_t q = 1; q < cs; ++q) run = run_merge(run, cluster_ld_run(&mine, q), k);
        if (TOP) {
          // the blocks' ordered lists, side by side: a key's place is the number of larger keys in each
          for (int i = tid; i < (int)cs * a.K; i += NT)
            top.cand[i] = cluster_ld_u64(cluster_map(top.top + i % a.K, i / a.K));
          __syncthreads();
        }
      }
    }
    if (cr == 0) {
      const RowOut o(run, log2f(run.s), a.inv_t);
      if (tid == 0) {
        if (a.target) {
          const int t = label_of(a.target, r, a.C, a.ignore, a.err);
          a.logp[r] = t < 0 ? 0.f : o.logp(Elem<T>::to_f(x.row[t]));
        }
        a.entropy[r] = o.entropy(run);
        a.lse[r] = o.lse();
        if (a.stats) a.stats[r] = make_float2(o.mm, run.s);
      }
      if (TOP) {
        for (int i = tid; i < (int)cs * a.K; i += NT) {
          uint64_t key = top.top[i % a.K];
          int rank = i;
          if (cs > 1) {
            key = top.cand[i];
            rank = 0;
            for (uint32_t q = 0; key && q < cs; ++q) {
              int lo = 0, hi = a.K;
              while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (top.cand[q * a.K + mid] > key) lo = mid + 1;
                else hi = mid;
              }
              rank += lo;
            }
          }
          if (o.bad && i < a.K) {
            a.top_logp[r * a.K + i] = NAN;
            a.top_index[r * a.K + i] = -1;
          } else if (!o.bad && key && rank < a.K) {
            a.top_logp[r * a.K + rank] = o.logp(key_value(key));
            a.top_index[r * a.K + rank] = key_class(key);
          }
        }
      }
    }
    if (cs > 1) cluster_sync();   // the other blocks' sums and lists have been read
    else __syncthreads();
  }
}

// One block per piece of a row.
template <typename T>
__global__ void __launch_bounds__(kGradThreads) bwd_block_kernel(BwdArgs a) {
  extern __shared__ __align__(16) uint8_t ring[];
  const int64_t r = blockIdx.x / a.segs;
  T* dz = static_cast<T*>(a.dz) + a.dv.base(r);
  GradPiece<T> piece(static_cast<const T*>(a.z) + a.v.base(r), dz, a.C, blockIdx.x % a.segs, a.segs, ring);
  const int t = label_of(a.target, r, a.C, a.ignore, a.err);
  const float gl = a.g_logp && t >= 0 ? a.g_logp[r * a.gl_inc] : 0.f;
  const float gh = a.g_entropy ? a.g_entropy[r * a.gh_inc] : 0.f;
  const float gs = a.g_lse ? a.g_lse[r * a.gs_inc] : 0.f;
  const float2 st = a.stats[r];
  // a row without a finite logit has no gradient; a bad row's is NaN, from its statistics
  if ((gl == 0.f && gh == 0.f && gs == 0.f) || st.y == 0.f) {
    piece.write([](float2) { return make_float2(0.f, 0.f); });
    return;
  }
  const float k = a.inv_t * kLog2e, f = a.inv_t / st.y;
  const float ca = f * (gs - gl - gh * a.entropy[r]), cb = f * gh * kLn2;
  const float c0 = cb != 0.f ? fmaf(cb, log2f(st.y), ca) : ca;   // p (ca - cb log2 p) as 2^t (c0 - cb t) / S
  const float2 m2 = {-st.x, -st.x}, k2 = {k, k}, c2 = {c0, c0}, b2 = {-cb, -cb};
  auto with_entropy = [&](float2 z) {
    float2 q = __fmul2_rn(__fadd2_rn(z, m2), k2);
    q = make_float2(max_nan(q.x, kFloor), max_nan(q.y, kFloor));
    return __fmul2_rn(make_float2(ex2(q.x), ex2(q.y)), __ffma2_rn(b2, q, c2));
  };
  if (cb != 0.f) {
    piece.write(with_entropy);
  } else {
    piece.write([&](float2 z) {
      const float2 q = __fmul2_rn(__fadd2_rn(z, m2), k2);
      return __fmul2_rn(make_float2(ex2(q.x), ex2(q.y)), c2);
    });
  }
  if (t >= 0 && piece.has(t)) {   // the label's own term, over what the block has stored
    __syncthreads();
    if (threadIdx.x == 0)
      dz[t] = Elem<T>::from_f(with_entropy(make_float2(Elem<T>::to_f(piece.x.row[t]), 0.f)).x + a.inv_t * gl);
  }
}

// ---- launches ----------------------------------------------------------------
template <typename T, int NT>
cudaError_t launch_fwd_block(const FwdArgs& a, cudaStream_t s) {
  const int cs = cluster_size(a.nrows, a.C, sizeof(T), NT);
  constexpr size_t ring = VecRing<NT, kBatch, kStages>::kBytes;
  const size_t smem = ring + (a.K > 0 ? (kCand + R4C_TOPK_MAX + NT) * sizeof(uint64_t) + NT * sizeof(int) : 0);
  const int64_t most = (int64_t)kSMs * blocks_per_sm(NT, smem);
  int64_t grid = a.nrows * cs;
  if (cs == 1 && grid > most) grid = most;
  if (a.K > 0) return launch_cluster(fwd_block_kernel<T, NT, true>, grid, NT, cs, smem, s, a);
  return launch_cluster(fwd_block_kernel<T, NT, false>, grid, NT, cs, smem, s, a);
}

template <typename T>
cudaError_t launch_fwd(FwdArgs& a, cudaStream_t s) {
  if (a.C <= kTileClasses) {
    const TileKind kind = tile_kind(a.C, sizeof(T));
    a.tile = make_tile(a.nrows, a.C, sizeof(T), kind.g, dense_rows(a.v, a.nrows, a.C, a.z));
    return for_tile_kind<T>(kind, [&](auto c) {
      return launch_tile(fwd_tile_kernel<T, decltype(c)::G, decltype(c)::E, decltype(c)::VEC>, a.tile, s, a);
    });
  }
  if ((int64_t)a.C * sizeof(T) <= 16 << 10) return launch_fwd_block<T, 128>(a, s);
  return launch_fwd_block<T, 256>(a, s);
}

template <typename T>
cudaError_t launch_bwd(BwdArgs& a, cudaStream_t s) {
  if (a.C <= kTileClasses) {
    const TileKind kind = tile_kind(a.C, sizeof(T));
    a.tile = make_tile(a.nrows, a.C, sizeof(T), kind.g,
                       dense_rows(a.v, a.nrows, a.C, a.z) && dense_rows(a.dv, a.nrows, a.C, a.dz));
    return for_tile_kind<T>(kind, [&](auto c) {
      return launch_tile(bwd_tile_kernel<T, decltype(c)::G, decltype(c)::E, decltype(c)::VEC>, a.tile, s, a);
    });
  }
  a.segs = grad_pieces(a.nrows, a.C, sizeof(T));
  if (a.nrows * a.segs > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch_cluster(bwd_block_kernel<T>, a.nrows * a.segs, kGradThreads, 1,
                        VecRing<kGradThreads, kGradBatch, kGradStages>::kBytes, s, a);
}

}  // namespace logp
}  // namespace r4c

using namespace r4c;

namespace {
int check(const r4c_rows_desc* d) {
  if (!rows::valid_desc(d)) return R4C_ERR_INVALID;
  if (!rows::valid_dtype(d->dtype)) return R4C_ERR_UNSUPPORTED;
  if (d->classes > rows::kTileClasses && (d->class_stride != 1 || d->grad_class_stride != 1)) return R4C_ERR_UNSUPPORTED;
  return R4C_OK;
}
}  // namespace

extern "C" size_t r4c_logp_stats_size(const r4c_rows_desc* d) {
  if (!rows::valid_desc(d) || d->classes <= rows::kTileClasses) return 0;
  return (size_t)d->rows * sizeof(float2);
}

extern "C" int r4c_logp_fwd(const r4c_rows_desc* d, const void* logits, const int64_t* target, int64_t ignore_index,
                            int top_k, float* logp, float* entropy, float* lse, float* top_logp, int32_t* top_index,
                            void* stats, r4c_stream_t stream) {
  const int rc = check(d);
  if (rc != R4C_OK) return rc;
  if (top_k < 0 || top_k > d->classes) return R4C_ERR_INVALID;
  if (top_k > R4C_TOPK_MAX) return R4C_ERR_TOO_LARGE;
  if (d->rows == 0) return R4C_OK;
  if (!logits || !entropy || !lse || (target && !logp) || (top_k > 0 && (!top_logp || !top_index))) return R4C_ERR_INVALID;
  int* err = tc::device_error_flag();
  if (!err) return R4C_ERR_NO_DEVICE;
  const int pairs = top_k == 2 && !(((uintptr_t)top_logp | (uintptr_t)top_index) & 7);
  logp::FwdArgs a{logits, target, ignore_index, d->rows, rows::make_view(d), {}, d->classes, top_k, pairs,
                  1.f / d->temperature, logp, entropy, lse, top_logp, top_index, static_cast<float2*>(stats), err};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d->dtype == R4C_BF16) e = logp::launch_fwd<__nv_bfloat16>(a, s);
  else if (d->dtype == R4C_F16) e = logp::launch_fwd<__half>(a, s);
  else e = logp::launch_fwd<float>(a, s);
  note_launches(1);
  return e == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}

extern "C" int r4c_logp_bwd(const r4c_rows_desc* d, const void* logits, const int64_t* target, int64_t ignore_index,
                            const float* entropy, const void* stats, const float* g_logp, int g_logp_inc,
                            const float* g_entropy, int g_entropy_inc, const float* g_lse, int g_lse_inc,
                            void* dlogits, r4c_stream_t stream) {
  const int rc = check(d);
  if (rc != R4C_OK) return rc;
  if (d->rows == 0) return R4C_OK;
  if (!logits || !dlogits || !entropy || (!stats && r4c_logp_stats_size(d)) || (g_logp && !target)) return R4C_ERR_INVALID;
  int* err = tc::device_error_flag();
  if (!err) return R4C_ERR_NO_DEVICE;
  logp::BwdArgs a{logits, target, ignore_index, d->rows, rows::make_view(d), rows::make_grad_view(d), {}, d->classes,
                  0, 1.f / d->temperature, entropy, static_cast<const float2*>(stats), g_logp, g_entropy, g_lse,
                  g_logp_inc, g_entropy_inc, g_lse_inc, dlogits, err};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d->dtype == R4C_BF16) e = logp::launch_bwd<__nv_bfloat16>(a, s);
  else if (d->dtype == R4C_F16) e = logp::launch_bwd<__half>(a, s);
  else e = logp::launch_bwd<float>(a, s);
  note_launches(1);
  return e == cudaSuccess ? R4C_OK : R4C_ERR_CUDA;
}
