// r4c_distill_tile.cuh — distillation for rows held in registers (up to 1024 classes).
//
// Both directions read the row once into registers; the backward computes the
// row's sums again rather than loading saved ones, which for the four classes
// of a segmentation would be more bytes than the logits (for a hundred classes
// they would be few; that form is not built). The teacher's pairs
// stay in registers as well, lane l of a row's group taking pairs l, l + G, ...
// With a rest bucket the listed classes are taken out of the staged row (their
// places set to -inf) before it is loaded, so that the loops over classes know
// nothing of the list; in the backward the pairs' lanes write the listed
// classes' gradients over the row at the end.
//
// Both directions run out of issue slots first (0.70 to 0.78 of them used,
// DRAM 0.21 to 0.31). B200, kernel alone: 4.2M rows of 4 bf16 classes, two pairs
// and a rest, 60 us forward and 65 us backward (0.25 and 0.31 of a copy's rate;
// 310 and 370 instructions a row, of which reading the pairs is 15, the loss
// 20); one pair 56 and 59 us, three (four places for them) 85 and 96 us. 369k
// rows of 105 classes with eight pairs and weights 50 and 70 us, with nine and
// a rest 67 and 82 us, with twenty (32 lanes a row) 222 and 262 us. Tests of
// the list per class instead took 171 and 203 us with eight.
#pragma once

#include "r4c_distill.cuh"

namespace r4c {
namespace distill {

constexpr int kMostSlots = 4;   // pairs of a lane; kernels hold two or four

// Blocks an SM should hold: issue-bound kernels gain from more warps as long
// as nothing spills.
constexpr int tile_blocks(int g, int e, int slots, bool bwd) {
  return g == 1 && e <= 8 && slots == 2 ? (bwd ? 6 : 8) : slots == 2 ? 4 : 3;
}

template <typename T, int G, int E, int UB, bool BWD, int kSlots, bool PLAIN>
__global__ void __launch_bounds__(kTileThreads, tile_blocks(G, E, kSlots, BWD)) tile_kernel(Args a) {
  constexpr int ES = (int)sizeof(T);
  const float k = a.inv_t * kLog2e;
  const bool rest = a.rest;
  const int K = a.K;
  auto has = [&](int s) { return s < 2 || s * G < K; };   // no test for the first two: an unused place is void
  Sum2 sum_loss, sum_w;
  const float scale1 = BWD && a.grad_inc == 0 ? grad_scale(a, 0) : 0.f;
  tile_walk<T, G, BWD>(a.tile, a.v, a.z, a.dv, a.dz, [&](int64_t r0, int r, uint32_t row, bool in) {
    const int lane = threadIdx.x & (G - 1);
    float w = a.weight ? (a.weight + r0)[r] : 1.f;
    float pv[kSlots], pz[kSlots], pq[kSlots];
    int pc[kSlots];
    const int64_t pairs0 = r0 * K;   // the tile's first pair
    const int p0 = r * K + lane;
    float qm = -INFINITY;
    bool any = false;
    if (PLAIN && G == 1 && a.even) {   // an even number of pairs, 8-byte aligned
      const float2* v2 = reinterpret_cast<const float2*>(static_cast<const float*>(a.t_logp) + pairs0 + p0);
      const int2* c2 = reinterpret_cast<const int2*>(static_cast<const int32_t*>(a.t_index) + pairs0 + p0);
#pragma unroll
      for (int s = 0; s < kSlots; s += 2) {
        pc[s] = pc[s + 1] = -1;
        pv[s] = pv[s + 1] = -INFINITY;
        if (s < K) {
          const float2 v = __ldg(v2 + s / 2);
          const int2 c = __ldg(c2 + s / 2);
          pv[s] = v.x;
          pv[s + 1] = v.y;
          pc[s] = valid_class(a, c.x, v.x);
          pc[s + 1] = valid_class(a, c.y, v.y);
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        pc[s] = -1;
        pv[s] = -INFINITY;
        if (has(s) && lane + s * G < K) {
          pv[s] = teacher_logp<PLAIN>(a, pairs0, p0 + s * G);
          pc[s] = teacher_class<PLAIN>(a, pairs0, p0 + s * G, pv[s]);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      pz[s] = -INFINITY;
      if (has(s) && pc[s] >= 0) {
        pz[s] = sh_get<T>(row + pc[s] * ES);
        qm = fmaxf(qm, pv[s]);
        any = true;
      }
    }
    if (G > 1) any = group_any<G>(any);
    if (!any) w = 0.f;

    // A class that is listed twice: its first pair stands for it (bit s of
    // `other`: pair s is not the first).
    unsigned other = 0;
    bool twice = false;
    if ((rest || BWD) && K > 1) {
      if (G == 1) {
#pragma unroll
        for (int s = 1; s < kSlots; ++s)
#pragma unroll
          for (int q = 0; q < s; ++q)
            if (pc[s] >= 0 && pc[s] == pc[q]) other |= 1u << s;
        twice = other != 0;
      } else {
        // each pair leaves its number at its class and looks whether it is still there
        __syncwarp();
#pragma unroll
        for (int s = 0; s < kSlots; ++s)
          if (has(s) && in && pc[s] >= 0) sh_put<T>(row + pc[s] * ES, (float)(lane + s * G + 1));
        __syncwarp();
#pragma unroll
        for (int s = 0; s < kSlots; ++s)
          if (has(s) && in && pc[s] >= 0) twice |= sh_get<T>(row + pc[s] * ES) != (float)(lane + s * G + 1);
        twice = group_any<G>(twice);
        if (__any_sync(0xffffffffu, twice)) {
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            if (!has(s)) continue;
            for (int i = 0; i < G; ++i) {
              const int c = __shfl_sync(0xffffffffu, pc[s], i, G);
#pragma unroll
              for (int q = 0; q < kSlots; ++q)
                if (pc[q] >= 0 && pc[q] == c && i + s * G < lane + q * G) other |= 1u << q;
            }
          }
        }
        __syncwarp();
      }
    }
    // With a rest the listed classes leave the row; else the numbers do.
    if (rest || (BWD && G > 1 && K > 1)) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (has(s) && in && pc[s] >= 0) sh_put<T>(row + pc[s] * ES, rest ? -INFINITY : pz[s]);
      if (G > 1) __syncwarp();
    }
    TileRow<T, G, E, UB> x;
    x.load(row, a.C);
    if (BWD && G > 1) __syncwarp();   // read by all before any of it is written over

    // The sums over the row as it stands and, with a rest, over the listed classes.
    const Run u = tile_exp(x, k);   // x: the exponentials from u.m
    Run l = run_empty();
    if (rest) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (has(s)) l.m = fmaxf(l.m, pz[s]);
      l.m = group_max<G>(l.m);
      const float lm = anchor(l.m);
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (has(s) && pc[s] >= 0 && !(other >> s & 1)) l.s += ex2((pz[s] - lm) * k);
      l.s = group_sum<G>(l.s);
    }
    RowSums s(u, l, rest, k);
    if (s.empty) w = 0.f;

    // The teacher's probabilities.
    const float q0 = rest ? 0.f : anchor(group_max<G>(qm));
    float sum_q = 0.f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      pq[i] = has(i) && pc[i] >= 0 ? prob(pv[i] - q0) : 0.f;
      sum_q += pq[i];
    }
    sum_q = group_sum<G>(sum_q);
    // (exact divisions where p - q may cancel)
    float noise = 0.f;
    if (!PLAIN && rest && a.t_round > 0.f) {
#pragma unroll
      for (int i = 0; i < kSlots; ++i) noise += pair_noise(pq[i], pv[i], a.t_round);
      noise = group_sum<G>(noise);
      if (s.sr != 0.f) noise = 0.f;
    }
    const float qi = rest ? 1.f : 1.f / sum_q, qr = rest ? rest_mass(sum_q, noise) : 0.f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) pq[i] *= qi;

    if constexpr (!BWD) {
      const float c0 = kLn2 * (lg2(qi) + lg2(s.s)) - q0;
      float loss = 0.f;
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
        if (has(i) && pc[i] >= 0 && !(pq[i] == 0.f)) loss += pq[i] * (pv[i] + c0 - (pz[i] - s.m) * a.inv_t);
      loss = group_sum<G>(loss) + rest_loss(qr, s, a.inv_t);
      if (in && lane == 0) {
        loss = w == 0.f ? 0.f : w * a.temp * a.temp * loss;
        if (a.row_loss) (a.row_loss + r0)[r] = loss;
        sum_loss.add(loss);
        sum_w.add(w);
      }
    } else {
      const float scale = w == 0.f ? 0.f : w * (a.grad_inc == 0 ? scale1 : grad_scale(a, r0 + r)), mass = rest ? sum_q + qr : 1.f;
      const float coef = w == 0.f ? 0.f : scale * rest_coef(rest, mass, qr, s.m, s.s, s.mr, s.sr, k);
      const float2 c2 = {coef, coef};
      x.each2([&](float2 e) { return __fmul2_rn(e, c2); });
      if (w == 0.f) {   // not 0 * NaN
#pragma unroll
        for (int e = 0; e < E; ++e) x.v[e] = 0.f;
      }
      if (in) x.store(x.v);
      if (G > 1) __syncwarp();
      // the listed classes: T w / W (Q p - q), q summed over the pairs of a class
      float q_of[kSlots];
#pragma unroll
      for (int i = 0; i < kSlots; ++i) q_of[i] = pq[i];
      if (G == 1) {
#pragma unroll
        for (int i = 1; i < kSlots; ++i)
#pragma unroll
          for (int q = 0; q < i; ++q)
            if (pc[i] >= 0 && pc[i] == pc[q]) q_of[q] += pq[i];
      } else if (__any_sync(0xffffffffu, twice)) {
#pragma unroll
        for (int i = 0; i < kSlots; ++i) q_of[i] = 0.f;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
          if (!has(i)) continue;
          for (int j = 0; j < G; ++j) {
            const int c = __shfl_sync(0xffffffffu, pc[i], j, G);
            const float q = __shfl_sync(0xffffffffu, pq[i], j, G);
#pragma unroll
            for (int h = 0; h < kSlots; ++h)
              if (pc[h] == c) q_of[h] += q;
          }
        }
      }
      const float mass_s = mass / s.s;
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
        if (has(i) && in && w != 0.f && pc[i] >= 0 && !(other >> i & 1))
          sh_put<T>(row + pc[i] * ES, scale * (mass_s * prob((pz[i] - s.m) * a.inv_t) - q_of[i]));
    }
  });
  if (!BWD && a.part) leave_part<kTileThreads>(sum_loss.value(), sum_w.value(), a);
}

// As for other tiles, with lanes enough for the pairs.
inline TileKind pairs_kind(int C, int K, int es) {
  TileKind kind = tile_kind(C, es);
  if (K <= kind.g * kMostSlots) return kind;
  const int ub = kind.ub == 16 ? 16 : 4;
  if (C <= 64 && K <= 8 * kMostSlots) return {8, 8, ub};
  if (C <= 256) return {32, 8, ub};
  return {32, 32, ub};
}

template <typename T>
cudaError_t launch_tiles(Args& a, bool bwd, int* blocks, cudaStream_t s) {
  const TileKind kind = pairs_kind(a.C, a.K, sizeof(T));
  a.tile = make_tile(a.nrows, a.C, sizeof(T), kind.g,
                     dense_rows(a.v, a.nrows, a.C, a.z) && (!bwd || dense_rows(a.dv, a.nrows, a.C, a.dz)));
  a.even = a.K % 2 == 0 && !(((uintptr_t)a.t_logp | (uintptr_t)a.t_index) & 7);
  const bool plain = a.t_dtype == R4C_F32 && !a.t_wide;
  auto launch = [&](auto c) {
    constexpr int G = decltype(c)::G, E = decltype(c)::E;
    constexpr int UB = decltype(c)::UB;
    if (plain && a.K <= 2 * G) {
      if (bwd) return launch_tile(tile_kernel<T, G, E, UB, true, 2, true>, a.tile, blocks, s, a);
      return launch_tile(tile_kernel<T, G, E, UB, false, 2, true>, a.tile, blocks, s, a);
    }
    if (plain && bwd) return launch_tile(tile_kernel<T, G, E, UB, true, 4, true>, a.tile, blocks, s, a);
    if (plain) return launch_tile(tile_kernel<T, G, E, UB, false, 4, true>, a.tile, blocks, s, a);
    if (bwd) return launch_tile(tile_kernel<T, G, E, UB, true, 4, false>, a.tile, blocks, s, a);
    return launch_tile(tile_kernel<T, G, E, UB, false, 4, false>, a.tile, blocks, s, a);
  };
  if (kind.g == 8 && kind.e == 8) return kind.ub == 16 ? launch(TileConst<8, 8, 16>{}) : launch(TileConst<8, 8, 4>{});
  if (kind.g == 32 && kind.e == 8) return kind.ub == 16 ? launch(TileConst<32, 8, 16>{}) : launch(TileConst<32, 8, 4>{});
  return for_tile_kind<T>(kind, launch);
}

}  // namespace distill
}  // namespace r4c
