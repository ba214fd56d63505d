// r4c_gn.cu — group normalisation with an activation: plans and entry points (r4c_gn_*).
#include <algorithm>
#include <cmath>
#include <numeric>

#include "r4c_gn.cuh"

namespace r4c {
namespace gn {
namespace {

struct Plan {
  Geo g;
  int V, threads;
  int sums_nb;       // blocks a sample of the sums
};

bool ok_desc(const r4c_gn_desc* d) {
  return d && d->samples >= 0 && d->inner >= 0 && d->channels > 0 && d->groups > 0 && d->channels % d->groups == 0 &&
         (d->dtype == R4C_BF16 || d->dtype == R4C_F16 || d->dtype == R4C_F32) &&
         (d->param_dtype == R4C_BF16 || d->param_dtype == R4C_F16 || d->param_dtype == R4C_F32) &&
         d->activation >= R4C_ACT_NONE && d->activation <= R4C_ACT_GELU && d->eps >= 0.f;
}

// A cluster for each sample and channel tile of whole groups, if one can keep its share on chip and is expected to be
// faster than two passes. Narrower tiles and larger clusters bring more SMs to few samples; tiles below 48 bytes a
// voxel would read sectors twice. The modelled times (us) follow these measurements, forward / backward: [1,192,4,8,8]
// bf16 silu, 1 block of 6 vectors a thread 5.9, 8 blocks of 1 vector 4.4, two passes 5.7; [64,96,6,6,6] 96 groups, 6
// vectors 5.5 / 8.4, two passes 9.7 / 10.5, 512 blocks in clusters of 4 11.4 / 17.4; [4,192,8,16,16] 6 vectors in 128
// blocks in clusters of 4 7.5 / 12.8, two passes 7.9 / 11.6. (The small backward's parameters take a launch of their own.)
void plan_small(const r4c_gn_desc* d, bool backward, int V, Geo& g, int* threads) {
  const int most = backward ? kSmallBwd : kSmallFwd, elem = (int)dtype_bytes(d->dtype);
  const double each = backward ? 0.5 : 0.35, mb = (double)d->samples * (double)g.sample * elem * 1e-6;
  double best = (backward ? 9.0 : 5.6) + 0.65 * mb + (double)d->samples / 300.0;
  for (int k = g.G;; k = (k + 1) / 2) {
    const bool whole = k == g.G;
    const int64_t width = whole ? g.L : (int64_t)k * g.Cg;
    const bool ok = whole || (g.L == g.C && width % V == 0 && width * elem >= 48);
    if (ok && width / V <= kThreads && k <= kSmallGroups) {
      const int lanes = (int)(width / V), tiles = whole ? 1 : cdiv(g.G, k);
      if (tiles > 65535) break;
      for (int cl = 1; cl <= 8; cl *= 2) {
        const int64_t per = std::max<int64_t>(1, (g.rows + cl - 1) / cl);
        int R = (int)std::min<int64_t>(std::max(1, kThreads / lanes), per);
        if (R > 4) R = R / 4 * 4;
        const int64_t nv = (per + R - 1) / R;
        if (nv > most || (cl > 1 && per < 4)) continue;
        const double blocks = (double)d->samples * tiles * cl;
        const double waves = std::ceil(blocks / (148.0 * 2));
        const double cost = (backward ? 5.5 : 3.5) + each * nv + (cl > 1 ? 0.2 + (backward ? 0.025 : 0.015) * blocks : 0.0) +
                            (waves - 1.0) * (1.5 + each * nv);
        if (cost < best - 1e-9) {
          best = cost;
          g.small = (int)nv;
          g.lanes = lanes;
          g.tiles = tiles;
          g.R = R;
          g.nb = cl;
          g.chunk = nv * R;
          *threads = cdiv((int64_t)R * lanes, 32) * 32;
        }
      }
    }
    if (k == 1) break;
  }
}

// Blocks a sample so that all fill the SMs once, `fit` on each, and a thread has four rows or more.
int blocks_for(const Geo& g, int64_t samples, int fit) {
  const int64_t want = std::max<int64_t>(1, 148 * fit / std::max<int64_t>(1, samples * g.tiles));
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (g.rows + 4 * g.R - 1) / (4 * g.R)));
}

// How the blocks share the data; false where a count passes a launch's limits.
bool make_plan(const r4c_gn_desc* d, bool backward, Plan* pl) {
  Geo& g = pl->g;
  const int64_t C = d->channels;
  if (d->inner > INT64_MAX / 8 / C || (d->samples && d->inner * C > INT64_MAX / 8 / d->samples)) return false;
  g.sample = d->inner * C;
  g.samples = d->samples;
  g.C = d->channels;
  g.G = d->groups;
  g.Cg = g.C / g.G;
  g.inv_m = 1.0 / ((double)g.Cg * (double)std::max<int64_t>(1, d->inner));
  g.eps = d->eps;
  g.slope = d->slope;
  g.act = d->activation;
  g.pdtype = d->param_dtype;
  g.format = g.pack = g.wide_params = 0;
  pl->sums_nb = 1;
  // the widest vector that parts a voxel's channels, or whose rows of lcm(C, V) elements (several voxels) fit a block's
  // threads
  int V = 16 / (int)dtype_bytes(d->dtype);
  while (C % V != 0 && std::lcm(C, (int64_t)V) > kThreads * V) V /= 2;
  pl->V = V;
  g.L = (int)std::lcm(C, (int64_t)V);
  g.rows = g.sample / g.L;
  g.edges = g.sample % g.L != 0;
  g.small = 0;
  if (g.rows > 0 || g.edges) plan_small(d, backward, V, g, &pl->threads);
  if (g.small) {
    g.blocks = d->samples * g.nb;
    g.chunk_tiles = g.small;
    g.np = g.nb * g.tiles;
    pl->sums_nb = g.nb;
    return g.blocks + g.C <= INT32_MAX;
  }
  const int lanes = g.L / V;
  g.tiles = cdiv(lanes, kThreads);
  g.lanes = cdiv(lanes, g.tiles);
  g.R = std::max(1, kThreads / g.lanes);
  if (g.R > 4) g.R = g.R / 4 * 4;       // a tile of rows starts at a block of 32 elements (fused packing)
  pl->threads = cdiv(g.R * g.lanes, 32) * 32;
  // one wave of blocks, none with less than four rows for each thread
  const double each_sm = (double)d->samples * g.tiles * (double)((g.rows + g.R - 1) / g.R) / 148.0;
  const int sums_fit = each_sm < kShortSums ? 1 : backward ? kBwdSumsFit : kStatsFit;
  const Geo sums = split(g, blocks_for(g, d->samples, sums_fit));
  pl->sums_nb = sums.nb;
  g = split(g, blocks_for(g, d->samples, backward ? kBwdFit : kApplyFit));
  g.np = sums.nb * g.tiles;
  const int64_t most = std::max(g.blocks, sums.blocks);
  return most + g.C <= INT32_MAX && g.tiles <= 65535 && g.rows / g.R < INT32_MAX;
}

// Whether a block of 32 elements is 32 / V neighbouring threads' in every tile of rows, so that the forward can write
// the 8 bits in its own pass over x.
bool fused_pack(const Plan& pl, size_t elem) {
  const Geo& g = pl.g;
  if (pl.V * elem != 16 || g.edges || g.sample % r4c::q8::kBlock) return false;
  if (g.tiles == 1) return (int64_t)g.R * g.L % r4c::q8::kBlock == 0;
  return g.C % r4c::q8::kBlock == 0 && g.lanes * pl.V % r4c::q8::kBlock == 0;
}

size_t fwd_bytes(const Plan& pl) {
  return align_up((size_t)pl.g.samples * pl.sums_nb * pl.g.tiles * pl.g.G * sizeof(double2), 256);
}
size_t cpart_bytes(const Plan& pl) { return align_up((size_t)pl.g.samples * pl.sums_nb * pl.g.C * sizeof(double2), 256); }
size_t bwd_bytes(const Plan& pl) {
  return cpart_bytes(pl) + align_up((size_t)pl.g.samples * pl.sums_nb * pl.g.tiles * pl.g.G * sizeof(double2), 256);
}

// Parameters as fp32 words of four: a thread's channels follow each other where a row is one voxel.
int wide_params(const Geo& g, const void* gamma, const void* beta) {
  return g.pdtype == R4C_F32 && g.L == g.C && ((reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(beta)) & 15) == 0;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int status(cudaError_t e) {
  if (e == cudaSuccess) return R4C_OK;
  (void)cudaGetLastError();             // a failed launch leaves no error behind for the next call
  return R4C_ERR_CUDA;
}

}  // namespace
}  // namespace gn
}  // namespace r4c

using namespace r4c::gn;

extern "C" {

size_t r4c_gn_workspace_size(const r4c_gn_desc* desc, int backward) {
  Plan pl;
  if (!ok_desc(desc) || !make_plan(desc, backward != 0, &pl)) return 0;
  if (backward) return bwd_bytes(pl);
  return pl.g.small ? 0 : fwd_bytes(pl);
}

int r4c_gn_fwd(const r4c_gn_desc* desc, const void* x, const void* gamma, const void* beta, void* y, float* mean_rstd,
               int format, void* codes, void* exponents, void* ws, size_t ws_bytes, r4c_stream_t stream) {
  if (!ok_desc(desc)) return R4C_ERR_INVALID;
  if (desc->samples == 0 || desc->inner == 0) return R4C_OK;
  Plan pl;
  if (!make_plan(desc, false, &pl)) return R4C_ERR_TOO_LARGE;
  if (!x || !y || !mean_rstd || (codes == nullptr) != (exponents == nullptr)) return R4C_ERR_INVALID;
  if (codes && format != R4C_Q8_INT8 && format != R4C_Q8_E4M3) return R4C_ERR_INVALID;
  if (!aligned(x) || !aligned(y) || !aligned(codes) || !aligned(ws)) return R4C_ERR_ALIGN;
  if (!pl.g.small && (!ws || ws_bytes < fwd_bytes(pl))) return R4C_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  FwdArgs a;
  a.x = x;
  a.gamma = gamma;
  a.beta = beta;
  a.y = y;
  a.mean_rstd = reinterpret_cast<float2*>(mean_rstd);
  a.part = static_cast<double2*>(ws);
  a.sums_nb = pl.sums_nb;
  pl.g.wide_params = wide_params(pl.g, gamma, beta);
  a.codes = static_cast<uint8_t*>(codes);
  a.exps = static_cast<uint8_t*>(exponents);
  pl.g.format = format;
  pl.g.pack = codes && fused_pack(pl, r4c::dtype_bytes(desc->dtype));
  cudaError_t e;
  if (desc->dtype == R4C_BF16) e = launch_fwd<__nv_bfloat16>(a, pl.g, pl.V, pl.threads, s);
  else if (desc->dtype == R4C_F16) e = launch_fwd<__half>(a, pl.g, pl.V, pl.threads, s);
  else e = launch_fwd<float>(a, pl.g, pl.V, pl.threads, s);
  if (e != cudaSuccess) return status(e);
  if (codes && !pl.g.pack) return r4c_pack8(x, desc->samples * pl.g.sample, desc->dtype, format, codes, exponents, stream);
  return R4C_OK;
}

int r4c_gn_bwd(const r4c_gn_desc* desc, const void* dy, const void* x, int format, const void* exponents,
               const float* mean_rstd, const void* gamma, const void* beta, void* dx, float* dgamma, float* dbeta,
               void* ws, size_t ws_bytes, r4c_stream_t stream) {
  if (!ok_desc(desc)) return R4C_ERR_INVALID;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (desc->samples == 0 || desc->inner == 0) {
    const size_t bytes = sizeof(float) * (size_t)desc->channels;
    if (dgamma && cudaMemsetAsync(dgamma, 0, bytes, s) != cudaSuccess) return R4C_ERR_CUDA;
    if (dbeta && cudaMemsetAsync(dbeta, 0, bytes, s) != cudaSuccess) return R4C_ERR_CUDA;
    return R4C_OK;
  }
  Plan pl;
  if (!make_plan(desc, true, &pl)) return R4C_ERR_TOO_LARGE;
  if (!dy || !x || !mean_rstd) return R4C_ERR_INVALID;
  if (exponents && format != R4C_Q8_INT8 && format != R4C_Q8_E4M3) return R4C_ERR_INVALID;
  if (!aligned(dy) || !aligned(x) || !aligned(exponents) || !aligned(dx) || !aligned(ws)) return R4C_ERR_ALIGN;
  if (!ws || ws_bytes < bwd_bytes(pl)) return R4C_ERR_WORKSPACE;
  if (!dx && !dgamma && !dbeta) return R4C_OK;
  BwdArgs a;
  a.dy = dy;
  a.x = x;
  a.gamma = gamma;
  a.beta = beta;
  a.exps = static_cast<const uint8_t*>(exponents);
  a.mean_rstd = reinterpret_cast<const float2*>(mean_rstd);
  a.dx = dx;
  a.dgamma = dgamma;
  a.dbeta = dbeta;
  a.cpart = static_cast<double2*>(ws);
  a.gpart = reinterpret_cast<double2*>(static_cast<uint8_t*>(ws) + cpart_bytes(pl));
  a.sums_nb = pl.sums_nb;
  pl.g.format = format;
  pl.g.wide_params = wide_params(pl.g, gamma, beta);
  if (desc->dtype == R4C_BF16) return status(launch_bwd<__nv_bfloat16>(a, pl.g, pl.V, pl.threads, s));
  if (desc->dtype == R4C_F16) return status(launch_bwd<__half>(a, pl.g, pl.V, pl.threads, s));
  return status(launch_bwd<float>(a, pl.g, pl.V, pl.threads, s));
}

}  // extern "C"
