// r4c_logp.cu — log-probability of a given label, entropy, log-sum-exp and
// the most probable classes of each row of logits, and the logits' gradient.
//
//   s_c = z_c / T,  m = max s,  S = sum exp(s_c - m),  lse = m + ln S
//   logp = s_t - lse,   H = ln S - (1/S) sum exp(s_c - m) (s_c - m)
//   dz_c = (1/T) [ p_c (g_lse - g_logp - g_H (ln p_c + H)) + g_logp [c = t] ],  p_c = exp(s_c - lse)
//
// The difference z_c - max z is taken before it is scaled, so rows of the
// type's lowest value stay a uniform distribution instead of overflowing.
// Both directions read each logit once; how short and long rows are read is
// described in r4c_rows.cuh. Figures below: B200, kernel alone, L2 flushed;
// "of copy" is against a copy's 6.55 TB/s.
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
  int C, ign, K, pairs;   // pairs: K = 2 and the outputs 8-byte aligned
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
  int C, ign, segs;
  float inv_t;
  const float* entropy;
  const float2* stats;
  const float *g_logp, *g_entropy, *g_lse;
  int gl_inc, gh_inc, gs_inc;
  void* dz;
  int* err;
};

// The row's label, -1 when it has none or takes no part. (ign: ignore_index
// where it is a class, else -1; most labels need one comparison in 64 bits.)
__device__ __forceinline__ int label_of(const int64_t* target, int64_t r, int C, int64_t ignore, int ign, int* err) {
  if (!target) return -1;
  const int64_t t = target[r];
  if ((uint64_t)t < (uint64_t)C) return (int)t == ign ? -1 : (int)t;
  if (t != ignore) atomicExch(err, 6);
  return -1;
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

// Short rows, forward. With the whole row in the registers of G lanes the
// maximum is known before the first exponential, so there is no rescaling;
// the entropy comes from sum 2^t t in the same pass, and the alternatives
// from rounds of a maximum over unique keys (two of them, of a lane's own
// row, from one pass that keeps the two largest). What it does beyond the
// exponentials fills its issue slots (0.70 to 0.75 of them) before the memory
// is busy: 4.2M rows of 4 bf16 classes with labels and two alternatives take
// 41 us, 0.69 of copy, at 210 instructions a row, of which the alternatives
// are 70, the label 30 and the sums 27; 369k rows of 105 fp16 classes 39 us,
// 0.33 of copy. The rounds go over all of a lane's keys, so they cost far more
// than a pass: with 0, 1, 5 and 20 alternatives 369k rows of 105 bf16 classes
// take 39, 64, 98 and 225 us, fp32 (keys of 64 bits) 57, 98, 190 and 539 us;
// 4.2M rows of 4 with 1, 2 and 3 take 47, 41 and 65 us.
template <typename T, int G, int E, int UB>
__global__ void __launch_bounds__(kTileThreads) fwd_tile_kernel(FwdArgs a) {
  const float k = a.inv_t * kLog2e;
  tile_walk<T, G, false>(a.tile, a.v, a.z, a.v, nullptr, [&](int64_t r0, int r, uint32_t row, bool in) {
    TileRow<T, G, E, UB> x;
    x.load(row, a.C);
    // Two alternatives of a lane's own row: the two largest in one pass
    // (a later class takes a place only by a larger value).
    float b1 = x.v[0], b2 = -INFINITY;
    int c1 = 0, c2 = 1;
    if (G == 1 && a.pairs) {
      const bool half = x.c0 < 0;   // the first value is no class
      if (half) {
        b1 = x.v[1];
        c1 = 1;
        c2 = 2;
      } else {
        const bool up = x.v[1] > b1;
        b2 = up ? b1 : x.v[1];
        b1 = up ? x.v[1] : b1;
        c1 = up;
        c2 = !up;
      }
#pragma unroll
      for (int e = 2; e < E; ++e) {
        const bool up = x.v[e] > b1, mid = x.v[e] > b2;
        c2 = up ? c1 : mid ? e : c2;
        b2 = up ? b1 : mid ? x.v[e] : b2;
        c1 = up ? e : c1;
        b1 = up ? x.v[e] : b1;
      }
      c1 -= half;
      c2 -= half;
    }
    const Run run = tile_run(x, k);
    const RowOut o(run, lg2(run.s), a.inv_t);
    if (in && x.lane == 0) {
      if (a.target) {
        const int t = label_of(a.target + r0, r, a.C, a.ignore, a.ign, a.err);
        (a.logp + r0)[r] = t < 0 ? 0.f : o.logp(sh_get<T>(row + t * (int)sizeof(T)));
      }
      (a.entropy + r0)[r] = o.entropy(run);
      (a.lse + r0)[r] = o.lse();
    }
    if (a.K == 0) return;
    float* tl = a.top_logp + r0 * a.K + r * a.K;
    int32_t* ti = a.top_index + r0 * a.K + r * a.K;
    if (G == 1 && a.pairs) {   // stored whole: half-written sectors cost twice
      if (in) {                // (a bad row's sums are NaN and make its values NaN)
        *reinterpret_cast<float2*>(tl) = make_float2(o.logp(b1), o.logp(b2));
        *reinterpret_cast<int2*>(ti) = o.bad ? make_int2(-1, -1) : make_int2(c1, c2);
      }
      return;
    }
    // the most probable classes, one after the other, from the row as it was
    x.load(row, a.C);
    using Key = TopKey<T>;
    typename Key::type key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = Key::make(x.v[e], x.cls(e));   // past the row: -inf, ranked after every class
    if (x.c0 < 0) key[0] = Key::kNone;                                  // the half word before it is no class
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

// Short rows, backward: dz_c = 2^t (c0 - cb t) with the row's constants, then
// the label's own term. The sums are computed again: reading them back would
// be 8 bytes a row, as much as four bf16 logits (little beside a hundred, but
// that form is not built). 369k rows of 105 fp16 classes take 61 us (0.40 of
// copy, 0.73 of the issue slots).
template <typename T, int G, int E, int UB>
__global__ void __launch_bounds__(kTileThreads) bwd_tile_kernel(BwdArgs a) {
  const float k = a.inv_t * kLog2e;
  tile_walk<T, G, true>(a.tile, a.v, a.z, a.dv, a.dz, [&](int64_t r0, int r, uint32_t row, bool in) {
    TileRow<T, G, E, UB> x;
    const int t = a.target ? label_of(a.target + r0, r, a.C, a.ignore, a.ign, a.err) : -1;
    const float gl = a.g_logp && t >= 0 ? (a.g_logp + r0 * a.gl_inc)[r * a.gl_inc] : 0.f;
    const float gh = a.g_entropy ? (a.g_entropy + r0 * a.gh_inc)[r * a.gh_inc] : 0.f;
    const float gs = a.g_lse ? (a.g_lse + r0 * a.gs_inc)[r * a.gs_inc] : 0.f;
    x.load(row, a.C);
    const Run run = tile_run(x, k);   // x: the exponents
    const float l2s = lg2(run.s);
    const bool none = (gl == 0.f && gh == 0.f && gs == 0.f) || run.s == 0.f;
    const float h = kLn2 * (l2s - __fdividef(run.u, run.s));
    const float f = none ? 0.f : __fdividef(a.inv_t, run.s), ca = f * (gs - gl - gh * h), cb = f * gh * kLn2;
    const float mm = -anchor(run.m), lb = cb * l2s;
    // 2^t (ca - cb (t - l2s))
    const float c0 = none ? 0.f : ca + lb, b0 = none ? 0.f : -cb;
    const float2 c2 = {c0, c0}, b2 = {b0, b0};
    float zt = 0.f;
    if (t >= 0) zt = sh_get<T>(row + t * (int)sizeof(T));
    x.each2([&](float2 q) { return __fmul2_rn(make_float2(ex2(q.x), ex2(q.y)), __ffma2_rn(b2, q, c2)); });
    if (none) {   // not 0 * NaN
#pragma unroll
      for (int e = 0; e < E; ++e) x.v[e] = 0.f;
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
// The K largest keys of a block's part of a row (unique: value, then class,
// so the result is exact whatever the ties). While it streams, each thread
// notes the largest value of each quarter of its own vectors. The K-th
// largest of these is a bound that at least K elements reach, and few more
// do, so only the quarters that reach it are read again, from L2 as a rule.
// If elements crowd above the bound (more than there are places: a row of
// equal values, for one) it is raised by bisection over them first.
constexpr int kQuarters = 4;
// Candidate places; a cluster's first block also takes in the others' lists.
__host__ __device__ inline int cand_places(int cs, int K, int threads) {
  const int n = cs * K > 4 * K ? cs * K : 4 * K;
  return n > 2 * threads ? n : 2 * threads;
}
struct TopShared {
  uint64_t* cand;     // `places` of them
  uint64_t* top;      // R4C_TOPK_MAX
  uint32_t* best;     // [kQuarters][threads]: the order of a quarter's largest value, 0: no vector
  int* active;        // [kQuarters * threads]: quarters that reach the bound
  uint32_t bound;
  int places, n_active, n_cand;
};
inline size_t top_bytes(int cs, int K, int threads) {
  return (cand_places(cs, K, threads) + R4C_TOPK_MAX) * sizeof(uint64_t) + kQuarters * threads * 2 * sizeof(uint32_t);
}
__device__ __forceinline__ uint32_t order_of(float v) { return (uint32_t)(rank_key(v, 0) >> 32); }

// Called by one warp: the largest value (up to the 13 bits that 16-bit types
// do not have) that at least K of the n orders at p reach; a slightly smaller
// one if that is quicker found, 0 with fewer than K of them.
template <typename T, int N>
__device__ __forceinline__ uint32_t warp_bound(const uint32_t* p, int K) {
  constexpr int SH = sizeof(T) == 4 ? 0 : 13;
  const int lane = threadIdx.x & 31;
  uint32_t kv[N], lo = ~0u, hi = 0;
  int reach = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    kv[i] = p[lane + 32 * i] >> SH;
    reach += kv[i] != 0;
    hi = kv[i] > hi ? kv[i] : hi;
    if (kv[i] && kv[i] < lo) lo = kv[i];
  }
  reach = __reduce_add_sync(0xffffffffu, reach);
  if (reach < K) return 0;
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi) + 1;   // none reach it
  const int enough = K + (K >> 1) + 2;
  while (reach > enough && hi - lo > 1) {
    const uint32_t mid = lo + ((hi - lo) >> 1);
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += kv[i] >= mid;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= K) {
      lo = mid;
      reach = c;
    } else {
      hi = mid;
    }
  }
  return lo << SH;
}

// (Called, not inlined: its registers would spill the streaming loop's.)
template <typename T, int NT>
__device__ __noinline__ void select_top(const uint4* p, const T* row, int off, int C, int v0, int v1, int f0, int f1,
                                        int per, int K, TopShared* shp) {
  constexpr int VE = Vec<T>::kElems, U = 4;
  TopShared& sh = *shp;
  const int tid = threadIdx.x;
  for (int j = tid; j < K; j += NT) sh.top[j] = 0;
  if (tid < 32) {
    const uint32_t b = warp_bound<T, kQuarters * NT / 32>(sh.best, K);
    if (tid == 0) {
      sh.bound = b;
      sh.n_active = sh.n_cand = 0;
    }
  }
  __syncthreads();
  uint64_t bound = (uint64_t)sh.bound << 32;
#pragma unroll
  for (int q = 0; q < kQuarters; ++q) {
    const uint32_t o = sh.best[q * NT + tid];
    if (o && o >= sh.bound) sh.active[atomicAdd(&sh.n_active, 1)] = q * NT + tid;
  }
  __syncthreads();
  const int items = sh.n_active * per, places = sh.places;
  uint64_t lo = bound, hi = ~0ull;
  bool keep = true;   // keep the elements that reach the bound, or count them
  for (;;) {
    const float low = bound >> 32 <= 0x007fffffu ? -INFINITY : key_value(bound | ((bound >> 63) || sizeof(T) == 4 ? 0ull : 0x1fffull << 32));
    int count = 0;
    auto look = [&](float z, int c) {
      const uint64_t key = rank_key(z, c);
      if (key < bound) return;
      if (keep) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < places) sh.cand[at] = key;
      } else {
        ++count;
      }
    };
    for (int i0 = tid; i0 < items; i0 += U * NT) {
      uint4 w[U];
      int v[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = i0 + j * NT;
        v[j] = f1;
        if (i < items) {
          const int g = sh.active[i / per];
          v[j] = f0 + g % NT + ((g / NT) * per + i % per) * NT;
        }
        w[j] = v[j] < f1 ? __ldg(p + v[j]) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (v[j] >= f1 || Vec<T>::top(w[j]) < low) continue;
        float y[VE];
        Vec<T>::split(w[j], y);
        unsigned hits = 0;
#pragma unroll
        for (int e = 0; e < VE; ++e) hits |= (unsigned)(y[e] >= low) << e;
        const T* at = reinterpret_cast<const T*>(p + v[j]);
        for (; hits; hits &= hits - 1) {
          const int e = __ffs(hits) - 1;
          look(Elem<T>::to_f(at[e]), v[j] * VE - off + e);
        }
      }
    }
    // the partial vectors at the row's ends
    if (f0 > v0 && tid < VE) {
      const int c = v0 * VE - off + tid;
      if (c >= 0 && c < C) look(Elem<T>::to_f(row[c]), c);
    }
    if (f1 < v1 && f1 >= f0 && tid >= NT - VE) {
      const int c = f1 * VE - off + tid - (NT - VE);
      if (c >= 0 && c < C) look(Elem<T>::to_f(row[c]), c);
    }
    if (!keep && count) atomicAdd(&sh.n_cand, count);
    __syncthreads();
    const int n = sh.n_cand;
    if (keep && n <= places) break;
    // raise the bound: at least K reach lo, fewer than K reach hi; at most 64 halvings
    if (!keep) {
      if (n < K) hi = bound;
      else lo = bound;
    }
    keep = (!keep && n >= K && n <= places) || hi - lo <= 1;
    bound = keep ? lo : lo + ((hi - lo) >> 1);
    __syncthreads();
    if (tid == 0) sh.n_cand = 0;
    __syncthreads();
  }
  // their order, by counting
  const int n = sh.n_cand;
  for (int i = tid; i < n; i += NT) {
    const uint64_t key = sh.cand[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += sh.cand[j] > key;
    if (rank < K) sh.top[rank] = key;
  }
  __syncthreads();
}

// Long rows, forward: one pass with a running maximum and sums, in batches of
// four vectors a thread that are copied ahead, across the rows' ends too. The
// memory bounds it for fp32. For 16-bit logits nothing is full (issue slots
// 0.65, the exponential unit 0.57, DRAM 0.53 at 32771 classes), and the largest
// stall is the block's barriers at the rows' ends. 4096 rows of 131072 bf16
// classes take 195 us (0.84 of copy), 4096 of 65536 fp32 174 us (0.94), 4095 of
// 32771 bf16 70 us (0.59); the first with one alternative 201 us, with twenty
// 236 us (128 threads a row; 231 and 248 us with 256). A third batch in flight changed nothing. One row of 131072 takes 16 us with
// twenty alternatives, 10 us without, on eight blocks.
constexpr int kBatch = 4, kStages = 2;
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT) fwd_block_kernel(FwdArgs a) {
  constexpr int VE = Vec<T>::kElems, U = kBatch;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ RunShared<NT> runs;
  __shared__ Run mine, joined;
  __shared__ TopShared top;
  const int tid = threadIdx.x;
  uint32_t cs = 1, cr = 0;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cs));
  if (cs > 1) cr = cluster_rank();
  if (TOP && tid == 0) {
    top.cand = reinterpret_cast<uint64_t*>(dyn + VecRing<NT, U, kStages>::kBytes);
    top.places = cand_places((int)cs, a.K, NT);
    top.top = top.cand + top.places;
    top.best = reinterpret_cast<uint32_t*>(top.top + R4C_TOPK_MAX);
    top.active = reinterpret_cast<int*>(top.best + kQuarters * NT);
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
    // batches of a quarter, and the vectors of a thread in it
    const int quarter = (f1 - f0 + kQuarters * U * NT - 1) / (kQuarters * U * NT), per = quarter * U;
    float tm = -INFINITY;
    int b = 0, q = 0;
    if (TOP) {
#pragma unroll
      for (int i = 0; i < kQuarters; ++i) top.best[i * NT + tid] = 0;
    }
    for (int left = f1 - f0; left > 0; left -= U * NT) {
      uint4 w[U];
      float vm[U];
      stream.take(w);
      if (left < U * NT) {   // the last batch: nothing past the row
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (tid + i * NT >= left)
            w[i] = make_uint4(Word<T>::kNegInf, Word<T>::kNegInf, Word<T>::kNegInf, Word<T>::kNegInf);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) vm[i] = Vec<T>::top(w[i]);
      const float bm = fmaxf(fmaxf(vm[0], vm[1]), fmaxf(vm[2], vm[3]));
      run2_raise<true>(part, bm, k);
      run2_batch<VE, U>(part, k, [&](int i, float* y) { Vec<T>::split(i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3], y); });
      if (TOP) {
        tm = fmaxf(tm, bm);
        if (++b == quarter || left <= U * NT) {
          // (a quarter counts where this thread has a vector in it)
          if (f0 + tid + q * per * NT < f1) top.best[q * NT + tid] = order_of(tm);
          tm = -INFINITY;
          b = 0;
          ++q;
        }
      }
    }
    // partial vectors: one element a thread
    auto edge = [&](int c) {
      if (c >= 0 && c < a.C) run2_one<true>(part, Elem<T>::to_f(x.row[c]), k);
    };
    if (f0 > v0 && tid < VE) edge(x.cls(v0) + tid);
    if (f1 < v1 && f1 >= f0 && tid >= NT - VE) edge(x.cls(f1) + tid - (NT - VE));
    Run run = run_block<NT>(part.join(), k, runs);   // (and the quarters' values are in place)
    if (TOP) select_top<T, NT>(x.p, x.row, x.off, a.C, v0, v1, f0, f1, per, a.K, &top);
    if (cs > 1) {
      if (tid == 0) mine = run;
      cluster_sync();
      if (cr == 0) {
        if (TOP)   // the blocks' ordered lists, side by side: a key's place is the number of larger keys in each
          for (int i = tid; i < (int)cs * a.K; i += NT)
            top.cand[i] = cluster_ld_u64(cluster_map(top.top + i % a.K, i / a.K));
        if (tid < 32) {
          run = run_cluster(&mine, (int)cs, k);
          if (tid == 0) joined = run;
        }
        __syncthreads();
        run = joined;
      }
    }
    if (cr == 0) {
      const RowOut o(run, log2f(run.s), a.inv_t);
      if (tid == 0) {
        if (a.target) {
          const int t = label_of(a.target, r, a.C, a.ignore, a.ign, a.err);
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
            for (uint32_t q0 = 0; key && q0 < cs; q0 += 4) {   // four searches at a time
              int at[4] = {0, 0, 0, 0};
              for (int step = 64; step; step >>= 1) {
                if (step > a.K) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (q0 + j < cs && at[j] + step <= a.K && top.cand[(q0 + j) * a.K + at[j] + step - 1] > key) at[j] += step;
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (q0 + j < cs && at[j] < a.K && top.cand[(q0 + j) * a.K + at[j]] > key) ++at[j];   // all of 2^n
                rank += at[j];
              }
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

// Long rows, backward: elementwise from two saved numbers a row, one block per
// piece of a row; memory bounds it. 4095 rows of 32771 bf16 classes, with the
// entropy's gradient, 90 us (0.91 of copy; 100 us with 256 threads). Pieces
// of 4 vectors a thread instead of 16 took 120 us: what a block reads before it
// starts is the same.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) bwd_block_kernel(BwdArgs a) {
  extern __shared__ __align__(16) uint8_t ring[];
  const int64_t r = blockIdx.x / a.segs;
  T* dz = static_cast<T*>(a.dz) + a.dv.base(r);
  GradPiece<T, NT> piece(static_cast<const T*>(a.z) + a.v.base(r), dz, a.C, blockIdx.x % a.segs, a.segs, ring);
  const int t = label_of(a.target, r, a.C, a.ignore, a.ign, a.err);
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
  const size_t smem = VecRing<NT, kBatch, kStages>::kBytes +
                      (a.K > 0 ? top_bytes(cs, a.K, NT) : 0);
  auto* kernel = a.K > 0 ? fwd_block_kernel<T, NT, true> : fwd_block_kernel<T, NT, false>;
  const int64_t most = (int64_t)kSMs * blocks_per_sm(kernel, NT, smem);
  int64_t grid = a.nrows * cs;
  if (cs == 1 && grid > most) grid = most;
  return launch_cluster(kernel, grid, NT, cs, smem, s, a);
}

template <typename T>
cudaError_t launch_fwd(FwdArgs& a, cudaStream_t s) {
  if (a.C <= kTileClasses) {
    int blocks;
    const TileKind kind = tile_kind(a.C, sizeof(T));
    a.tile = make_tile(a.nrows, a.C, sizeof(T), kind.g, dense_rows(a.v, a.nrows, a.C, a.z));
    return for_tile_kind<T>(kind, [&](auto c) {
      return launch_tile(fwd_tile_kernel<T, decltype(c)::G, decltype(c)::E, decltype(c)::UB>, a.tile, &blocks, s, a);
    });
  }
  if (row_threads(a.C, sizeof(T), a.K) == kWarpRow) return launch_fwd_block<T, kWarpRow>(a, s);
  if (a.K > 0 && a.nrows >= 4 * kSMs) return launch_fwd_block<T, kManyRows>(a, s);
  return launch_fwd_block<T, kLongRow>(a, s);
}

template <typename T>
cudaError_t launch_bwd(BwdArgs& a, cudaStream_t s) {
  if (a.C <= kTileClasses) {
    int blocks;
    const TileKind kind = tile_kind(a.C, sizeof(T));
    a.tile = make_tile(a.nrows, a.C, sizeof(T), kind.g,
                       dense_rows(a.v, a.nrows, a.C, a.z) && dense_rows(a.dv, a.nrows, a.C, a.dz));
    return for_tile_kind<T>(kind, [&](auto c) {
      return launch_tile(bwd_tile_kernel<T, decltype(c)::G, decltype(c)::E, decltype(c)::UB>, a.tile, &blocks, s, a);
    });
  }
  const int threads = row_threads(a.C, sizeof(T), 0) == kWarpRow ? kWarpRow : kGradRow;
  a.segs = grad_pieces(a.nrows, a.C, sizeof(T), threads);
  if (a.nrows * a.segs > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (threads == kWarpRow)
    return launch_cluster(bwd_block_kernel<T, kWarpRow>, a.nrows, kWarpRow, 1,
                          VecRing<kWarpRow, kGradBatch, kGradStages>::kBytes, s, a);
  return launch_cluster(bwd_block_kernel<T, kGradRow>, a.nrows * a.segs, kGradRow, 1,
                        VecRing<kGradRow, kGradBatch, kGradStages>::kBytes, s, a);
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
  const int ign = ignore_index >= 0 && ignore_index < d->classes ? (int)ignore_index : -1;
  const int pairs = top_k == 2 && !(((uintptr_t)top_logp | (uintptr_t)top_index) & 7);
  logp::FwdArgs a{logits, target, ignore_index, d->rows, rows::make_view(d), {}, d->classes, ign, top_k, pairs,
                  1.f / d->temperature, logp, entropy, lse, top_logp, top_index, static_cast<float2*>(stats), err};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d->dtype == R4C_BF16) e = logp::launch_fwd<__nv_bfloat16>(a, s);
  else if (d->dtype == R4C_F16) e = logp::launch_fwd<__half>(a, s);
  else e = logp::launch_fwd<float>(a, s);
  note_launches(1);
  return rows::status(e);
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
  const int ign = ignore_index >= 0 && ignore_index < d->classes ? (int)ignore_index : -1;
  logp::BwdArgs a{logits, target, ignore_index, d->rows, rows::make_view(d), rows::make_grad_view(d), {}, d->classes,
                  ign, 0, 1.f / d->temperature, entropy, static_cast<const float2*>(stats), g_logp, g_entropy, g_lse,
                  g_logp_inc, g_entropy_inc, g_lse_inc, dlogits, err};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d->dtype == R4C_BF16) e = logp::launch_bwd<__nv_bfloat16>(a, s);
  else if (d->dtype == R4C_F16) e = logp::launch_bwd<__half>(a, s);
  else e = logp::launch_bwd<float>(a, s);
  note_launches(1);
  return rows::status(e);
}
