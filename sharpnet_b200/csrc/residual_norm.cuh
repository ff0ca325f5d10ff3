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

// out[g, :] = sum over k < parts of partial[g * parts + k] (rows of `pitch` floats), in a fixed order: eight warps each
// take every eighth part, and their sums are added in order.
static __global__ void __launch_bounds__(256)
norm_sums_kernel(const float* __restrict__ partial, long long pitch, int parts, int dim, float* __restrict__ out) {
  pdl_prologue();
  __shared__ float red[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x * 32 + lane;
  const float* src = partial + static_cast<long long>(blockIdx.y) * parts * pitch;
  float s = 0.0f;
  if (c < dim)
    for (int k = warp; k < parts; k += 8) s += src[k * pitch + c];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < dim) {
    float t = red[0][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += red[k][lane];
    out[static_cast<long long>(blockIdx.y) * dim + c] = t;
  }
}

}  // namespace snb
