// The step between two blocks of a Transformer in one pass over its rows: the norm behind a block, its gate, the scaled
// residual sum and the norm in front of the next block,
//
//   u = post(h) ;  r = a x + b gate * u ;  y = norm(r) ,      norm(t) = (t - mean) rstd gamma + beta   (LayerNorm)
//                                                                       t rstd gamma + beta            (RMSNorm)
//
// and its backward pass.  With g = dy gamma, xhat = (r - mean) rstd and D the row's width:
//   dR = dr + rstd (g - [sum g / D] - xhat sum(g xhat) / D)          ([..]: LayerNorm)
//   dx = a dR ;  du = b gate * dR ;  dgate = sum b dR * u ;  dh = post'(du), by the same formula with du post_gamma
//   dgamma = sum dy xhat, dbeta = sum dy, dpost_gamma = sum du hhat, dpost_beta = sum du, over the rows.
#pragma once
#include "elementwise.cuh"

namespace snb {

enum NormKind : int { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };
// column sums of the backward pass over all rows, in the order in which the scratch memory holds them
enum NormSum : int { SUM_GAMMA = 0, SUM_BETA = 1, SUM_POST_GAMMA = 2, SUM_POST_BETA = 3, SUM_COUNT = 4 };

struct NormArgs {
  long long rows;
  int dim, norm, post;
  int gate_rows;                 // 0: no gate
  long long rows_per_gate;       // consecutive rows that share a row of the gate
  float a, b, eps;
  const float *gamma, *beta, *post_gamma, *post_beta, *gate;
  const float *x, *h;
  float *r, *y, *stats, *post_stats;          // stats: [rows][2] mean, 1 / standard deviation (or root mean square)
};
struct NormGradArgs {
  long long rows;
  int dim, norm, post, gate_rows;
  long long rows_per_gate;
  float a, b;
  const float *gamma, *post_gamma, *post_beta, *gate;
  const float *r, *h, *dy, *dr, *stats, *post_stats;
  float *dx, *dh;
  int slot[SUM_COUNT], sums;     // slot[k] is the place of NormSum k among the `sums` vectors that are wanted, or -1
  int pieces, units;             // pieces that the rows of one gate row are cut into; work units: all pieces
  float* partial;                // [teams][sums][dim]
  float* dgate;                  // NULL where it is not wanted
  float* gate_partial;           // [units][dim]: the gate's sums where pieces > 1
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sums over the threads of a block, in a fixed order; every thread gets them.  `red` holds 2 x 32 floats, used in
// turn by `flip`, so that one barrier a sum is enough.
__device__ __forceinline__ float2 block_sum2(float2 v, float2 (*red)[32], int& flip) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v.x = warp_sum(v.x); v.y = warp_sum(v.y);
  if (lane == 0) red[flip][warp] = v;
  __syncthreads();
  float2 t = lane < warps ? red[flip][lane] : make_float2(0.0f, 0.0f);
  flip ^= 1;
  t.x = warp_sum(t.x); t.y = warp_sum(t.y);
  return t;
}

__device__ __forceinline__ float affine(float v, const float* gamma, const float* beta, int c) {
  if (gamma) v *= __ldg(gamma + c);
  if (beta) v += __ldg(beta + c);
  return v;
}

// ---------------------------------------------------------------- rows of any width: a block per row, read again for every sum
static __global__ void __launch_bounds__(256)
residual_norm_fwd_wide_kernel(const NormArgs p) {
  pdl_prologue();
  __shared__ float2 red[2][32];
  int flip = 0;
  const float inv_dim = 1.0f / p.dim;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const long long at = row * p.dim;
    const float* gate = p.gate_rows ? p.gate + (row / p.rows_per_gate) * p.dim : nullptr;
    float pm = 0.0f, pr = 1.0f;
    if (p.post != NORM_NONE) {
      float s = 0.0f, q = 0.0f;
      if (p.post == NORM_LAYER) {
        for (int c = threadIdx.x; c < p.dim; c += blockDim.x) s += p.h[at + c];
        pm = block_sum2(make_float2(s, 0.0f), red, flip).x * inv_dim;
      }
      for (int c = threadIdx.x; c < p.dim; c += blockDim.x) { const float d = p.h[at + c] - pm; q = fmaf(d, d, q); }
      pr = 1.0f / sqrtf(block_sum2(make_float2(q, 0.0f), red, flip).x * inv_dim + p.eps);
      if (p.post_stats && threadIdx.x == 0) { p.post_stats[2 * row] = pm; p.post_stats[2 * row + 1] = pr; }
    }
    // r is stored where the caller wants it; each thread reads back only what it wrote itself
    float s = 0.0f;
    for (int c = threadIdx.x; c < p.dim; c += blockDim.x) {
      float v = p.a * p.x[at + c];
      if (p.h) {
        float u = p.h[at + c];
        if (p.post != NORM_NONE) u = affine((u - pm) * pr, p.post_gamma, p.post_beta, c);
        v = fmaf(gate ? p.b * __ldg(gate + c) : p.b, u, v);
      }
      if (p.r) p.r[at + c] = v;
      s += v;
    }
    if (p.norm == NORM_NONE) continue;
    float m = 0.0f, q = 0.0f;
    if (p.norm == NORM_LAYER) m = block_sum2(make_float2(s, 0.0f), red, flip).x * inv_dim;
    const float* src = p.r ? p.r : p.x;
    const float f = p.r ? 1.0f : p.a;
    for (int c = threadIdx.x; c < p.dim; c += blockDim.x) { const float d = f * src[at + c] - m; q = fmaf(d, d, q); }
    const float rstd = 1.0f / sqrtf(block_sum2(make_float2(q, 0.0f), red, flip).x * inv_dim + p.eps);
    if (p.stats && threadIdx.x == 0) { p.stats[2 * row] = m; p.stats[2 * row + 1] = rstd; }
    for (int c = threadIdx.x; c < p.dim; c += blockDim.x)
      p.y[at + c] = affine((f * src[at + c] - m) * rstd, p.gamma, p.beta, c);
  }
}

// dR of one element: c1 = sum g / D (LayerNorm), c2 = sum g xhat / D
__device__ __forceinline__ float norm_dr(const NormGradArgs& p, long long i, int c, float m, float rstd, float c1, float c2, float* xhat, float* dyv) {
  float d = p.dr ? p.dr[i] : 0.0f;
  if (p.norm == NORM_NONE) return d;
  *dyv = p.dy[i];
  *xhat = (p.r[i] - m) * rstd;
  const float g = p.gamma ? *dyv * __ldg(p.gamma + c) : *dyv;
  return d + rstd * (g - c1 - *xhat * c2);
}

// The rows [begin, end) of a work unit: a piece of the rows that share a row of the gate.
__device__ __forceinline__ void norm_unit_rows(const NormGradArgs& p, int unit, long long* begin, long long* end) {
  const long long group = unit / p.pieces, piece = unit % p.pieces;
  *begin = group * p.rows_per_gate + p.rows_per_gate * piece / p.pieces;
  *end = group * p.rows_per_gate + p.rows_per_gate * (piece + 1) / p.pieces;
}

// The column sums live in the block's own part of the scratch memory; each thread touches its own columns only.
static __global__ void __launch_bounds__(256)
residual_norm_bwd_wide_kernel(const NormGradArgs p) {
  pdl_prologue();
  __shared__ float2 red[2][32];
  int flip = 0;
  const float inv_dim = 1.0f / p.dim;
  float* sums = p.partial + static_cast<long long>(blockIdx.x) * p.sums * p.dim;
  for (int k = 0; k < p.sums; ++k)
    for (int c = threadIdx.x; c < p.dim; c += blockDim.x) sums[static_cast<long long>(k) * p.dim + c] = 0.0f;
  for (int unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
    long long row, end;
    norm_unit_rows(p, unit, &row, &end);
    const float* gate = p.gate_rows ? p.gate + static_cast<long long>(unit / p.pieces) * p.dim : nullptr;
    float* gate_sum = p.dgate ? (p.pieces == 1 ? p.dgate : p.gate_partial) + static_cast<long long>(unit) * p.dim : nullptr;
    if (gate_sum)
      for (int c = threadIdx.x; c < p.dim; c += blockDim.x) gate_sum[c] = 0.0f;
    for (; row < end; ++row) {
      const long long at = row * p.dim;
      float m = 0.0f, rstd = 1.0f, pm = 0.0f, pr = 1.0f, c1 = 0.0f, c2 = 0.0f, p1 = 0.0f, p2 = 0.0f, xhat = 0.0f, dyv = 0.0f;
      if (p.norm != NORM_NONE) {
        m = p.stats[2 * row]; rstd = p.stats[2 * row + 1];
        float2 s = make_float2(0.0f, 0.0f);
        for (int c = threadIdx.x; c < p.dim; c += blockDim.x) {
          const float g = p.gamma ? p.dy[at + c] * __ldg(p.gamma + c) : p.dy[at + c];
          s.x += g;
          s.y = fmaf(g, (p.r[at + c] - m) * rstd, s.y);
        }
        s = block_sum2(s, red, flip);
        c1 = p.norm == NORM_LAYER ? s.x * inv_dim : 0.0f;
        c2 = s.y * inv_dim;
      }
      if (p.post != NORM_NONE) {
        pm = p.post_stats[2 * row]; pr = p.post_stats[2 * row + 1];
        float2 s = make_float2(0.0f, 0.0f);
        for (int c = threadIdx.x; c < p.dim; c += blockDim.x) {
          const float d = norm_dr(p, at + c, c, m, rstd, c1, c2, &xhat, &dyv);
          float g = (gate ? p.b * __ldg(gate + c) : p.b) * d;
          if (p.post_gamma) g *= __ldg(p.post_gamma + c);
          s.x += g;
          s.y = fmaf(g, (p.h[at + c] - pm) * pr, s.y);
        }
        s = block_sum2(s, red, flip);
        p1 = p.post == NORM_LAYER ? s.x * inv_dim : 0.0f;
        p2 = s.y * inv_dim;
      }
      for (int c = threadIdx.x; c < p.dim; c += blockDim.x) {
        const float d = norm_dr(p, at + c, c, m, rstd, c1, c2, &xhat, &dyv);
        if (p.slot[SUM_GAMMA] >= 0) sums[static_cast<long long>(p.slot[SUM_GAMMA]) * p.dim + c] += dyv * xhat;
        if (p.slot[SUM_BETA] >= 0) sums[static_cast<long long>(p.slot[SUM_BETA]) * p.dim + c] += dyv;
        if (p.h || p.dh) {
          const float du = (gate ? p.b * __ldg(gate + c) : p.b) * d;
          const float hv = p.h ? p.h[at + c] : 0.0f;
          const float hhat = p.post != NORM_NONE ? (hv - pm) * pr : hv;
          if (p.slot[SUM_POST_GAMMA] >= 0) sums[static_cast<long long>(p.slot[SUM_POST_GAMMA]) * p.dim + c] += du * hhat;
          if (p.slot[SUM_POST_BETA] >= 0) sums[static_cast<long long>(p.slot[SUM_POST_BETA]) * p.dim + c] += du;
          if (gate_sum) gate_sum[c] += p.b * d * (p.post != NORM_NONE ? affine(hhat, p.post_gamma, p.post_beta, c) : hv);
          if (p.dh) {
            const float g = p.post_gamma ? du * __ldg(p.post_gamma + c) : du;
            p.dh[at + c] = p.post != NORM_NONE ? pr * (g - p1 - hhat * p2) : du;
          }
        }
        if (p.dx) p.dx[at + c] = p.a * d;
      }
    }
  }
}

// ---------------------------------------------------------------- rows that stay in registers
// A team of WARPS warps holds a row: VPT groups of four elements a thread, one 16-byte vector (VEC = 4) or four elements
// TEAM apart (VEC = 1, for widths and pointers that allow no vectors).  A warp alone needs no barrier (8 teams a block);
// wider rows take a block each.
template <int TEAM, int VEC>
__device__ __forceinline__ float4 row_load(const float* row, int j, int t, int dim) {
  if (VEC == 4) {
    const int c = 4 * (j * TEAM + t);
    return c < dim ? __ldcs(reinterpret_cast<const float4*>(row + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  float4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = (4 * j + k) * TEAM + t;
    lane_set(v, k, c < dim ? __ldcs(row + c) : 0.0f);
  }
  return v;
}
// The same for a parameter vector, which every row reads: kept in the caches; `fill` where there is none.
template <int TEAM, int VEC>
__device__ __forceinline__ float4 param_load(const float* p, int j, int t, int dim, float fill) {
  float4 v = make_float4(fill, fill, fill, fill);
  if (!p) return v;
  if (VEC == 4) {
    const int c = 4 * (j * TEAM + t);
    return c < dim ? __ldg(reinterpret_cast<const float4*>(p + c)) : v;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = (4 * j + k) * TEAM + t;
    if (c < dim) lane_set(v, k, __ldg(p + c));
  }
  return v;
}
template <int TEAM, int VEC>
__device__ __forceinline__ void row_store(float* row, int j, int t, int dim, const float4& v) {
  if (VEC == 4) {
    const int c = 4 * (j * TEAM + t);
    if (c < dim) __stcs(reinterpret_cast<float4*>(row + c), v);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = (4 * j + k) * TEAM + t;
    if (c < dim) __stcs(row + c, lane_get(v, k));
  }
}
// Whether element k of group j lies in the row (the groups behind its end hold zeros, which a centred sum must not see).
template <int TEAM, int VEC>
__device__ __forceinline__ bool row_has(int j, int k, int t, int dim) {
  return (VEC == 4 ? 4 * (j * TEAM + t) : (4 * j + k) * TEAM + t) < dim;
}
template <int WARPS>
__device__ __forceinline__ float2 team_sum2(float2 v, float2 (*red)[32], int& flip) {
  if (WARPS == 1) return make_float2(warp_sum(v.x), warp_sum(v.y));
  return block_sum2(v, red, flip);
}
// Mean (LayerNorm; 0 for RMSNorm) and 1 / deviation of a row: the deviations are taken from the mean, so a mean that is
// large against them costs no digits.
template <int WARPS, int VPT, int VEC>
__device__ __forceinline__ float2 row_statistics(const float4 (&v)[VPT], int kind, int t, int dim, float inv_dim, float eps,
                                                 float2 (*red)[32], int& flip) {
  constexpr int TEAM = 32 * WARPS;
  float m = 0.0f;
  if (kind == NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) s += (v[j].x + v[j].y) + (v[j].z + v[j].w);
    m = team_sum2<WARPS>(make_float2(s, 0.0f), red, flip).x * inv_dim;
  }
  float q = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float d = row_has<TEAM, VEC>(j, k, t, dim) ? lane_get(v[j], k) - m : 0.0f;
      q = fmaf(d, d, q);
    }
  }
  q = team_sum2<WARPS>(make_float2(q, 0.0f), red, flip).x;
  return make_float2(m, 1.0f / sqrtf(q * inv_dim + eps));
}

template <int WARPS, int VPT, int VEC>
static __global__ void __launch_bounds__(WARPS == 1 ? 256 : 32 * WARPS)
residual_norm_fwd_kernel(const NormArgs p) {
  pdl_prologue();
  constexpr int TEAM = 32 * WARPS, TEAMS = WARPS == 1 ? 8 : 1;
  __shared__ float2 red[2][32];
  int flip = 0;
  const int t = threadIdx.x % TEAM;
  const float inv_dim = 1.0f / p.dim;
  for (long long row = blockIdx.x * static_cast<long long>(TEAMS) + threadIdx.x / TEAM; row < p.rows;
       row += static_cast<long long>(gridDim.x) * TEAMS) {
    const long long at = row * p.dim;
    float4 r[VPT], h[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      r[j] = row_load<TEAM, VEC>(p.x + at, j, t, p.dim);
      if (p.h) h[j] = row_load<TEAM, VEC>(p.h + at, j, t, p.dim);
    }
    float2 ps = make_float2(0.0f, 1.0f);
    if (p.post != NORM_NONE) {
      ps = row_statistics<WARPS, VPT, VEC>(h, p.post, t, p.dim, inv_dim, p.eps, red, flip);
      if (p.post_stats && t == 0) { p.post_stats[2 * row] = ps.x; p.post_stats[2 * row + 1] = ps.y; }
    }
    const float* gate = p.gate_rows ? p.gate + (row / p.rows_per_gate) * p.dim : nullptr;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (p.h) {
        const float4 pg = param_load<TEAM, VEC>(p.post_gamma, j, t, p.dim, 1.0f), pb = param_load<TEAM, VEC>(p.post_beta, j, t, p.dim, 0.0f);
        const float4 gt = param_load<TEAM, VEC>(gate, j, t, p.dim, 1.0f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float u = lane_get(h[j], k);
          if (p.post != NORM_NONE) u = fmaf((u - ps.x) * ps.y, lane_get(pg, k), lane_get(pb, k));
          const float v = fmaf(p.b * lane_get(gt, k), u, p.a * lane_get(r[j], k));
          lane_set(r[j], k, row_has<TEAM, VEC>(j, k, t, p.dim) ? v : 0.0f);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) lane_set(r[j], k, p.a * lane_get(r[j], k));
      }
      if (p.r) row_store<TEAM, VEC>(p.r + at, j, t, p.dim, r[j]);
    }
    if (p.norm == NORM_NONE) continue;
    const float2 st = row_statistics<WARPS, VPT, VEC>(r, p.norm, t, p.dim, inv_dim, p.eps, red, flip);
    if (p.stats && t == 0) { p.stats[2 * row] = st.x; p.stats[2 * row + 1] = st.y; }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const float4 ga = param_load<TEAM, VEC>(p.gamma, j, t, p.dim, 1.0f), be = param_load<TEAM, VEC>(p.beta, j, t, p.dim, 0.0f);
      float4 y;
#pragma unroll
      for (int k = 0; k < 4; ++k) lane_set(y, k, fmaf((lane_get(r[j], k) - st.x) * st.y, lane_get(ga, k), lane_get(be, k)));
      row_store<TEAM, VEC>(p.y + at, j, t, p.dim, y);
    }
  }
}

// The backward pass.  The column sums are added up in shared memory, where each thread keeps its own columns (five
// vectors of a wide row do not fit beside the row in registers, and a second pass over the batch for them would double
// the traffic); a block writes its sums once, when its rows are done.
__device__ __forceinline__ void add_to(float4* sum, const float4& v) {
  float4 s = *sum;
  s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  *sum = s;
}
template <int WARPS, int VPT, int VEC>
static __global__ void __launch_bounds__(WARPS == 1 ? 256 : 32 * WARPS)
residual_norm_bwd_kernel(const NormGradArgs p) {
  pdl_prologue();
  constexpr int TEAM = 32 * WARPS, TEAMS = WARPS == 1 ? 8 : 1, VECTOR = VPT * TEAM;     // float4s of one column sum
  extern __shared__ float4 norm_smem[];                // [TEAMS][sums (+ 1 for the gate)][VECTOR]
  __shared__ float2 red[2][32];
  int flip = 0;
  const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv_dim = 1.0f / p.dim;
  const int vectors = p.sums + (p.dgate != nullptr);
  float4* const mine = norm_smem + team * vectors * VECTOR + t;
  float4* const gate_sum = mine + p.sums * VECTOR;
  for (int k = 0; k < vectors; ++k)
#pragma unroll
    for (int j = 0; j < VPT; ++j) mine[k * VECTOR + j * TEAM] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int unit = blockIdx.x * TEAMS + team; unit < p.units; unit += gridDim.x * TEAMS) {
    long long row, end;
    norm_unit_rows(p, unit, &row, &end);
    const float* gate = p.gate_rows ? p.gate + static_cast<long long>(unit / p.pieces) * p.dim : nullptr;
    for (; row < end; ++row) {
      const long long at = row * p.dim;
      float4 d[VPT], xh[VPT], g[VPT], h[VPT];
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (p.norm != NORM_NONE) {
          xh[j] = row_load<TEAM, VEC>(p.r + at, j, t, p.dim);
          g[j] = row_load<TEAM, VEC>(p.dy + at, j, t, p.dim);
        }
        d[j] = p.dr ? row_load<TEAM, VEC>(p.dr + at, j, t, p.dim) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p.h) h[j] = row_load<TEAM, VEC>(p.h + at, j, t, p.dim);
      }
      if (p.norm != NORM_NONE) {
        const float m = __ldg(p.stats + 2 * row), rstd = __ldg(p.stats + 2 * row + 1);
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
          const float4 ga = param_load<TEAM, VEC>(p.gamma, j, t, p.dim, 1.0f);
          float4 w;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            lane_set(xh[j], k, (lane_get(xh[j], k) - m) * rstd);
            lane_set(w, k, lane_get(g[j], k) * lane_get(xh[j], k));
          }
          if (p.slot[SUM_GAMMA] >= 0) add_to(mine + p.slot[SUM_GAMMA] * VECTOR + j * TEAM, w);
          if (p.slot[SUM_BETA] >= 0) add_to(mine + p.slot[SUM_BETA] * VECTOR + j * TEAM, g[j]);
#pragma unroll
          for (int k = 0; k < 4; ++k) {      // behind the row's end g is zero
            const float v = lane_get(g[j], k) * lane_get(ga, k);
            lane_set(g[j], k, v);
            s.x += v;
            s.y = fmaf(v, lane_get(xh[j], k), s.y);
          }
        }
        s = team_sum2<WARPS>(s, red, flip);
        const float c1 = p.norm == NORM_LAYER ? s.x * inv_dim : 0.0f, c2 = s.y * inv_dim;
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            lane_set(d[j], k, fmaf(rstd, lane_get(g[j], k) - c1 - lane_get(xh[j], k) * c2, lane_get(d[j], k)));
      }
      if (p.dx) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
          row_store<TEAM, VEC>(p.dx + at, j, t, p.dim, make_float4(p.a * d[j].x, p.a * d[j].y, p.a * d[j].z, p.a * d[j].w));
      }
      if (!p.h && !p.dh) continue;
      float pm = 0.0f, pr = 1.0f;
      if (p.post != NORM_NONE) { pm = __ldg(p.post_stats + 2 * row); pr = __ldg(p.post_stats + 2 * row + 1); }
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const float4 gt = param_load<TEAM, VEC>(gate, j, t, p.dim, 1.0f), pg = param_load<TEAM, VEC>(p.post_gamma, j, t, p.dim, 1.0f);
        if (p.h) {
#pragma unroll
          for (int k = 0; k < 4; ++k) if (p.post != NORM_NONE) lane_set(h[j], k, (lane_get(h[j], k) - pm) * pr);
          if (p.dgate) {
            const float4 pb = param_load<TEAM, VEC>(p.post_beta, j, t, p.dim, 0.0f);
            float4 w;
#pragma unroll
            for (int k = 0; k < 4; ++k) lane_set(w, k, p.b * lane_get(d[j], k) * fmaf(lane_get(h[j], k), lane_get(pg, k), lane_get(pb, k)));
            add_to(gate_sum + j * TEAM, w);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) lane_set(d[j], k, p.b * lane_get(gt, k) * lane_get(d[j], k));       // du
        if (p.slot[SUM_POST_BETA] >= 0) add_to(mine + p.slot[SUM_POST_BETA] * VECTOR + j * TEAM, d[j]);
        if (p.post != NORM_NONE) {
          float4 w;
#pragma unroll
          for (int k = 0; k < 4; ++k) lane_set(w, k, lane_get(d[j], k) * lane_get(h[j], k));
          if (p.slot[SUM_POST_GAMMA] >= 0) add_to(mine + p.slot[SUM_POST_GAMMA] * VECTOR + j * TEAM, w);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float v = row_has<TEAM, VEC>(j, k, t, p.dim) ? lane_get(d[j], k) * lane_get(pg, k) : 0.0f;
            lane_set(d[j], k, v);
            s.x += v;
            s.y = fmaf(v, lane_get(h[j], k), s.y);
          }
        }
      }
      if (!p.dh) continue;
      if (p.post != NORM_NONE) {
        s = team_sum2<WARPS>(s, red, flip);
        const float p1 = p.post == NORM_LAYER ? s.x * inv_dim : 0.0f, p2 = s.y * inv_dim;
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) lane_set(d[j], k, pr * (lane_get(d[j], k) - p1 - lane_get(h[j], k) * p2));
      }
#pragma unroll
      for (int j = 0; j < VPT; ++j) row_store<TEAM, VEC>(p.dh + at, j, t, p.dim, d[j]);
    }
    if (p.dgate) {
      float* to = (p.pieces == 1 ? p.dgate : p.gate_partial) + static_cast<long long>(unit) * p.dim;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        row_store<TEAM, VEC>(to, j, t, p.dim, gate_sum[j * TEAM]);
        gate_sum[j * TEAM] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    }
  }
  if (TEAMS > 1) __syncthreads();
  // the teams' sums in order; each thread adds what lies at its own places
  if (team == 0) {
    for (int k = 0; k < p.sums; ++k) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        float4 s = mine[k * VECTOR + j * TEAM];
        for (int o = 1; o < TEAMS; ++o) {
          const float4 v = mine[(o * vectors + k) * VECTOR + j * TEAM];
          s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        row_store<TEAM, VEC>(p.partial + (static_cast<long long>(blockIdx.x) * p.sums + k) * p.dim, j, t, p.dim, s);
      }
    }
  }
}

// The column sums of all blocks, one launch for every vector: row y < sums of the grid adds vector y over the blocks'
// parts, the others a row of the gate over its pieces.  32 warps each take every 32nd part, and their sums are added in
// order.
struct NormSums {
  const float *partial, *gate_partial;
  int parts, pieces, sums, dim;
  float* out[SUM_COUNT];
  float* gate;
};
static __global__ void __launch_bounds__(1024)
norm_sums_kernel(const NormSums p) {
  pdl_prologue();
  __shared__ float red[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, y = blockIdx.y;
  const int c = blockIdx.x * 32 + lane;
  const bool gate = y >= p.sums;
  const int parts = gate ? p.pieces : p.parts;
  const long long pitch = gate ? p.dim : static_cast<long long>(p.sums) * p.dim;
  const float* src = gate ? p.gate_partial + static_cast<long long>(y - p.sums) * parts * p.dim : p.partial + static_cast<long long>(y) * p.dim;
  float s = 0.0f;
  if (c < p.dim) {
#pragma unroll 4
    for (int k = warp; k < parts; k += 32) s += src[k * pitch + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  // transposed: warp w adds the 32 sums of column w
  s = warp_sum(red[lane][warp]);
  const int col = blockIdx.x * 32 + warp;
  if (lane == 0 && col < p.dim) (gate ? p.gate + static_cast<long long>(y - p.sums) * p.dim : p.out[y])[col] = s;
}

}  // namespace snb
