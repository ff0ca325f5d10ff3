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
#include "ptx.cuh"

namespace snb {

enum NormKind : int { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };
// column sums of the backward pass over all rows, in the order in which the scratch memory holds them
// (the gate's is one of them where one gate serves all rows)
enum NormSum : int { SUM_GAMMA = 0, SUM_BETA = 1, SUM_POST_GAMMA = 2, SUM_POST_BETA = 3, SUM_GATE = 4, SUM_COUNT = 5 };

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
  float* dgate;                  // of a gate that changes with the rows; NULL where it is not wanted
  float* gate_partial;           // [units][dim]: the gate's sums where pieces > 1
  int* error_word;
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
          if (p.slot[SUM_GATE] >= 0)
            sums[static_cast<long long>(p.slot[SUM_GATE]) * p.dim + c] += p.b * d * (p.post != NORM_NONE ? affine(hhat, p.post_gamma, p.post_beta, c) : hv);
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
// wider rows take a block each.  Bound by memory: 16384 x 4096 forward takes 165 us (6.5 TB/s; 358 with rows read again for
// every sum), one row of 4096 3.0 us.
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

// The backward pass of rows of up to 4096 elements: blocks of 16 warps, one a SM, cut into teams of WARPS warps with a row
// each.  A warp owns VPT * 128 consecutive columns.  It has its part of the row's r, dy, dr and h (and of the gate where
// its rows change) copied into shared memory by bulk copies of its own, two rows ahead, on barriers of its own, so that
// the memory pipe is busy while rows go through their two reductions and no warp waits for another's data; the thread's
// share of the five column sums stays in registers.  What all rows read (gamma, post_gamma, post_beta, a gate for all)
// lies in shared memory.
// Bound by memory: 16384 x 4096 with everything on takes 260 us (6.2 TB/s); with the sums in shared memory and no copies
// ahead it took 385, with every thread copying its own elements 371 (the shared-memory pipe full).
// Bulk copies begin and end on 16-byte borders: a part that does not (VEC = 1) is fetched with the few bytes around it,
// which lie in the same 16-byte granules.
constexpr int kNormThreads = 512;
constexpr int kNormWarps = kNormThreads / 32;
constexpr int kNormStages = 2;
template <int VPT> __host__ __device__ constexpr int norm_part() { return VPT * 512 + 16; }       // bytes of a warp's part of a row, as fetched

__device__ __forceinline__ void bulk_copy(void* smem, const void* global, unsigned bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(smem)), "l"(global), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy_async4(void* smem, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}

// The rows that a team takes, in order.
struct NormRows {
  int unit;
  long long row, end;
  __device__ __forceinline__ void start(const NormGradArgs& p, int first) {
    unit = first;
    if (unit < p.units) norm_unit_rows(p, unit, &row, &end);
  }
  __device__ __forceinline__ void next(const NormGradArgs& p, int stride) {
    if (++row < end) return;
    unit += stride;
    if (unit < p.units) norm_unit_rows(p, unit, &row, &end);
  }
};

// Two sums over a team of WARPS warps, in a fixed order.  The lower half of a warp adds up x and the upper half y, which
// takes one exchange instead of a second chain of five; barrier 1 + team is the team's own, `red` is used in turn by
// `flip` so that one barrier a sum is enough.
template <int WARPS>
__device__ __forceinline__ float2 team_sum_pair(float2 v, float (*red)[2][kNormWarps], int team, int& flip) {
  const int lane = threadIdx.x & 31, half = lane >> 4;
  float s = half ? v.y : v.x;
  s += __shfl_xor_sync(0xffffffffu, half ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (WARPS > 1) {
    const int warp = threadIdx.x >> 5;
    if ((lane & 15) == 0) red[flip][half][warp] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * WARPS) : "memory");
    s = (lane & 15) < WARPS ? red[flip][half][team * WARPS + (lane & 15)] : 0.0f;
    flip ^= 1;
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  return make_float2(__shfl_sync(0xffffffffu, s, 0), __shfl_sync(0xffffffffu, s, 16));
}

// Elements of group j of a warp's part, in pairs: one 16-byte vector a lane (VEC = 4), or four elements 32 apart (VEC = 1);
// zeros behind the row's end (`left`: columns from the lane's first to the row's end).
struct Pairs { float2 a, b; };
template <int VEC>
__device__ __forceinline__ Pairs part_load(const float* part, int j, int lane, int left) {
  if (VEC == 4) {
    const float4 v = 128 * j < left ? *reinterpret_cast<const float4*>(part + 128 * j + 4 * lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return Pairs{make_float2(v.x, v.y), make_float2(v.z, v.w)};
  }
  const float* e = part + 128 * j + lane;
  float v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = 128 * j + 32 * k < left ? e[32 * k] : 0.0f;
  return Pairs{make_float2(v[0], v[1]), make_float2(v[2], v[3])};
}
// The same of a parameter vector in global memory; `fill` where there is none.
template <int VEC>
__device__ __forceinline__ Pairs param_pairs(const float* v, int mine, int j, int left, float fill) {
  float e[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = 128 * j + (VEC == 4 ? k : 32 * k);
    e[k] = !v ? fill : c < left ? __ldg(v + mine + c) : 0.0f;
  }
  return Pairs{make_float2(e[0], e[1]), make_float2(e[2], e[3])};
}
// `row`: at the lane's first column.
template <int VEC>
__device__ __forceinline__ void part_store(float* row, int j, int left, const Pairs& v) {
  if (VEC == 4) {
    if (128 * j < left) __stcs(reinterpret_cast<float4*>(row + 128 * j), make_float4(v.a.x, v.a.y, v.b.x, v.b.y));
    return;
  }
  const float e[4] = {v.a.x, v.a.y, v.b.x, v.b.y};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (128 * j + 32 * k < left) __stcs(row + 128 * j + 32 * k, e[k]);
}

// Per row, with e = b dR:  A += e hhat and B += e.  A gate's gradient is post_gamma A + post_beta B over its rows, those of
// post_gamma and post_beta are gate A and gate B summed over the gates, so the loop over rows needs neither parameter by
// itself: only b gate post_gamma, which is one vector unless the gate changes with the rows (GATES: it does; its rows come
// as a fifth stream).
template <int WARPS, int VPT, int VEC, bool GATES>
static __global__ void __launch_bounds__(kNormThreads, 1)
residual_norm_bwd_kernel(NormGradArgs p) {
  pdl_prologue();
  constexpr int TEAMS = kNormWarps / WARPS, COLUMNS = WARPS * VPT * 128, PART = norm_part<VPT>();
  extern __shared__ float4 norm_smem[];   // [warps][stages][streams][PART bytes], [2][COLUMNS]
  __shared__ float red[2][2][kNormWarps];
  __shared__ float stat_slots[kNormWarps][kNormStages][4];
  __shared__ uint64_t bars[kNormWarps][kNormStages];
  __shared__ int abort_flag;
  int flip = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, team = warp / WARPS, stride = gridDim.x * TEAMS;
  const int first = (warp % WARPS) * VPT * 128;                        // the warp's first column
  const int columns = min(VPT * 128, p.dim - first);                   // and how many of its columns there are (<= 0: none)
  const int mine = first + (VEC == 4 ? 4 * lane : lane), left = p.dim - mine;
  const float inv_dim = 1.0f / p.dim;
  const bool norm = p.norm != NORM_NONE, post = p.post != NORM_NONE;
  const int at_dr = norm ? 2 : 0, at_h = at_dr + (p.dr != nullptr), at_gate = at_h + (p.h != nullptr);
  const int streams = at_gate + GATES;
  char* const parts = reinterpret_cast<char*>(norm_smem) + warp * kNormStages * streams * PART;
  float* const gamma = reinterpret_cast<float*>(reinterpret_cast<char*>(norm_smem) + kNormWarps * kNormStages * streams * PART);
  float* const back = gamma + COLUMNS;                                 // b gate post_gamma, or b post_gamma where the gates change
  if (lane < kNormStages) mbar_init(&bars[warp][lane], 1);          // a warp's barriers are its own
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  __syncwarp();

  // lane k < streams has the warp's part of stream k copied
  const float* source = nullptr;
  if (norm && lane < 2) source = lane == 0 ? p.r : p.dy;
  if (p.dr && lane == at_dr) source = p.dr;
  if (p.h && lane == at_h) source = p.h;
  if (GATES && lane == at_gate) source = p.gate;
  const float* const stat_source = lane < 2 ? p.stats : p.post_stats;
  auto fetch = [&](const NormRows& it, int stage) {
    if (it.unit < p.units) {
      uint64_t* const bar = &bars[warp][stage];
      const float* from = source + (GATES && lane == at_gate ? static_cast<long long>(it.unit / p.pieces) : it.row) * p.dim + first;
      unsigned over = 0, bytes = 4 * columns;
      if (VEC == 1) {
        over = static_cast<unsigned>(reinterpret_cast<uintptr_t>(from) & 15);
        bytes = (over + bytes + 15) & ~15u;
      }
      if (columns > 0) {
        if (VEC == 4) {
          if (lane == 0) mbar_arrive_expect_tx(bar, streams * bytes);
        } else {
          const unsigned total = __reduce_add_sync(0xffffffffu, lane < streams ? bytes : 0);
          if (lane == 0) mbar_arrive_expect_tx(bar, total);
        }
        __syncwarp();
        if (lane < streams) bulk_copy(parts + (stage * streams + lane) * PART, reinterpret_cast<const char*>(from) - over, bytes, bar);
      } else if (lane == 0) {
        mbar_arrive(bar);
      }
      if (lane < 4 && (lane < 2 ? norm : post)) copy_async4(&stat_slots[warp][stage][lane], stat_source + 2 * it.row + (lane & 1));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");       // a group a row, an empty one behind the last
  };
  // the warp's part of stream k, past the bytes in front of it
  auto part_of = [&](int stage, int k, const float* row) {
    const float* part = reinterpret_cast<const float*>(parts + (stage * streams + k) * PART);
    return VEC == 4 ? part : part + ((reinterpret_cast<uintptr_t>(row + first) & 15) >> 2);
  };
  const Pairs zero = {both(0.0f), both(0.0f)};
  Pairs sum_gamma[VPT], sum_beta[VPT], A[VPT], B[VPT], sum_post_gamma[GATES ? VPT : 1], sum_post_beta[GATES ? VPT : 1];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    sum_gamma[j] = sum_beta[j] = A[j] = B[j] = zero;
    if (GATES) sum_post_gamma[j] = sum_post_beta[j] = zero;
  }

  NormRows now, ahead;
  now.start(p, blockIdx.x * TEAMS + team);
  ahead.start(p, now.unit);
  for (int s = 0; s < kNormStages; ++s) {
    fetch(ahead, s);
    if (ahead.unit < p.units) ahead.next(p, stride);
  }
  // the parameters, while the first rows are on their way
  for (int i = threadIdx.x; i < COLUMNS; i += kNormThreads) {
    const bool in = i < p.dim;
    gamma[i] = !in ? 0.0f : p.gamma ? __ldg(p.gamma + i) : 1.0f;
    const float g = !in ? 0.0f : !GATES && p.gate_rows ? p.b * __ldg(p.gate + i) : p.b;
    back[i] = in && p.post_gamma ? g * __ldg(p.post_gamma + i) : g;
  }
  __syncthreads();
  int stage = 0;
  unsigned parity = 0;
  while (now.unit < p.units) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kNormStages - 1) : "memory");
    __syncwarp();
    mbar_wait(&bars[warp][stage], parity, &abort_flag);
    const long long out = now.row * p.dim;
    const float* const st = stat_slots[warp][stage];
    Pairs d[VPT], x[VPT], g[VPT];
    const float* const part_d = part_of(stage, at_dr, p.dr + out);
#pragma unroll
    for (int j = 0; j < VPT; ++j) d[j] = p.dr ? part_load<VEC>(part_d, j, lane, left) : zero;
    if (norm) {
      const float2 m = both(-st[0]), rstd = both(st[1]);
      const float* const part_r = part_of(stage, 0, p.r + out);
      const float* const part_g = part_of(stage, 1, p.dy + out);
      float2 s = both(0.0f), q = both(0.0f);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const Pairs r = part_load<VEC>(part_r, j, lane, left), v = part_load<VEC>(part_g, j, lane, left);
        const Pairs ga = part_load<VEC>(gamma + first, j, lane, 1 << 20);
        x[j].a = mul2(add2(r.a, m), rstd); x[j].b = mul2(add2(r.b, m), rstd);
        sum_gamma[j].a = fma2(v.a, x[j].a, sum_gamma[j].a); sum_gamma[j].b = fma2(v.b, x[j].b, sum_gamma[j].b);
        sum_beta[j].a = add2(sum_beta[j].a, v.a); sum_beta[j].b = add2(sum_beta[j].b, v.b);
        g[j].a = mul2(v.a, ga.a); g[j].b = mul2(v.b, ga.b);
        s = add2(s, add2(g[j].a, g[j].b));
        q = fma2(g[j].a, x[j].a, q); q = fma2(g[j].b, x[j].b, q);
      }
      const float2 c = team_sum_pair<WARPS>(make_float2(s.x + s.y, q.x + q.y), red, team, flip);
      const float2 c1 = both(p.norm == NORM_LAYER ? -c.x * inv_dim : 0.0f), c2 = both(-c.y * inv_dim);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        d[j].a = fma2(rstd, add2(fma2(x[j].a, c2, g[j].a), c1), d[j].a);
        d[j].b = fma2(rstd, add2(fma2(x[j].b, c2, g[j].b), c1), d[j].b);
      }
    }
    if (p.dx) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) part_store<VEC>(p.dx + out + mine, j, left, Pairs{mul2(both(p.a), d[j].a), mul2(both(p.a), d[j].b)});
    }
    float2 s = both(0.0f), q = both(0.0f);
    float2 pr = both(1.0f);
    if (p.h || p.dh) {
      const float2 pm = both(post ? -st[2] : 0.0f);
      if (post) pr = both(st[3]);
      const float* const part_h = part_of(stage, at_h, p.h + out);
      const float* const part_gate = part_of(stage, at_gate, GATES ? p.gate + static_cast<long long>(now.unit / p.pieces) * p.dim : nullptr);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const Pairs h = p.h ? part_load<VEC>(part_h, j, lane, left) : zero;
        Pairs bk = part_load<VEC>(back + first, j, lane, 1 << 20);
        if (GATES) {
          const Pairs gt = part_load<VEC>(part_gate, j, lane, left);
          bk.a = mul2(bk.a, gt.a); bk.b = mul2(bk.b, gt.b);
        }
        const Pairs e = {mul2(both(p.b), d[j].a), mul2(both(p.b), d[j].b)};
        x[j].a = mul2(add2(h.a, pm), pr); x[j].b = mul2(add2(h.b, pm), pr);
        A[j].a = fma2(e.a, x[j].a, A[j].a); A[j].b = fma2(e.b, x[j].b, A[j].b);
        B[j].a = add2(B[j].a, e.a); B[j].b = add2(B[j].b, e.b);
        d[j].a = mul2(d[j].a, bk.a); d[j].b = mul2(d[j].b, bk.b);
        s = add2(s, add2(d[j].a, d[j].b));
        q = fma2(d[j].a, x[j].a, q); q = fma2(d[j].b, x[j].b, q);
      }
    }
    __syncwarp();                            // every lane has read its part: it takes the row after the next
    fetch(ahead, stage);
    if (ahead.unit < p.units) ahead.next(p, stride);
    if (p.dh) {
      if (post) {
        const float2 c = team_sum_pair<WARPS>(make_float2(s.x + s.y, q.x + q.y), red, team, flip);
        const float2 c1 = both(p.post == NORM_LAYER ? -c.x * inv_dim : 0.0f), c2 = both(-c.y * inv_dim);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
          d[j].a = mul2(pr, add2(fma2(x[j].a, c2, d[j].a), c1));
          d[j].b = mul2(pr, add2(fma2(x[j].b, c2, d[j].b), c1));
        }
      }
#pragma unroll
      for (int j = 0; j < VPT; ++j) part_store<VEC>(p.dh + out + mine, j, left, d[j]);
    }
    const int unit = now.unit;
    now.next(p, stride);
    if (GATES && now.unit != unit) {         // the last row of a piece: what its gate gathered
      const float* gate = p.gate + static_cast<long long>(unit / p.pieces) * p.dim;
      float* to = (p.pieces == 1 ? p.dgate : p.gate_partial) + static_cast<long long>(unit) * p.dim + mine;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const Pairs gt = param_pairs<VEC>(gate, mine, j, left, 1.0f);
        if (p.dgate) {
          const Pairs pg = param_pairs<VEC>(p.post_gamma, mine, j, left, 1.0f), pb = param_pairs<VEC>(p.post_beta, mine, j, left, 0.0f);
          part_store<VEC>(to, j, left, Pairs{fma2(pg.a, A[j].a, mul2(pb.a, B[j].a)), fma2(pg.b, A[j].b, mul2(pb.b, B[j].b))});
        }
        sum_post_gamma[j].a = fma2(gt.a, A[j].a, sum_post_gamma[j].a); sum_post_gamma[j].b = fma2(gt.b, A[j].b, sum_post_gamma[j].b);
        sum_post_beta[j].a = fma2(gt.a, B[j].a, sum_post_beta[j].a); sum_post_beta[j].b = fma2(gt.b, B[j].b, sum_post_beta[j].b);
        A[j] = B[j] = zero;
      }
    }
    if (++stage == kNormStages) { stage = 0; parity ^= 1; }
  }
  // the block's sums: the teams' in order, through shared memory
  auto finish = [&](int slot, const Pairs (&sum)[VPT]) {
    if (slot < 0) return;
    float* to = p.partial + (static_cast<long long>(blockIdx.x) * p.sums + slot) * p.dim + mine;
    if (TEAMS > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VPT; ++j) norm_smem[(warp * VPT + j) * 32 + lane] = make_float4(sum[j].a.x, sum[j].a.y, sum[j].b.x, sum[j].b.y);
      __syncthreads();
      if (team > 0) return;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      Pairs s = sum[j];
      for (int o = 1; o < TEAMS; ++o) {
        const float4 v = norm_smem[((o * WARPS + warp) * VPT + j) * 32 + lane];
        s.a = add2(s.a, make_float2(v.x, v.y)); s.b = add2(s.b, make_float2(v.z, v.w));
      }
      part_store<VEC>(to, j, left, s);
    }
  };
  finish(p.slot[SUM_GAMMA], sum_gamma);
  finish(p.slot[SUM_BETA], sum_beta);
  if constexpr (GATES) {
    finish(p.slot[SUM_POST_GAMMA], sum_post_gamma);
    finish(p.slot[SUM_POST_BETA], sum_post_beta);
  } else {
    Pairs s[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const Pairs pg = param_pairs<VEC>(p.post_gamma, mine, j, left, 1.0f), pb = param_pairs<VEC>(p.post_beta, mine, j, left, 0.0f);
      s[j] = Pairs{fma2(pg.a, A[j].a, mul2(pb.a, B[j].a)), fma2(pg.b, A[j].b, mul2(pb.b, B[j].b))};
    }
    finish(p.slot[SUM_GATE], s);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const Pairs gt = param_pairs<VEC>(p.gate, mine, j, left, 1.0f);
      A[j] = Pairs{mul2(gt.a, A[j].a), mul2(gt.b, A[j].b)};
      B[j] = Pairs{mul2(gt.a, B[j].a), mul2(gt.b, B[j].b)};
    }
    finish(p.slot[SUM_POST_GAMMA], A);
    finish(p.slot[SUM_POST_BETA], B);
  }
  if (threadIdx.x == 0 && abort_flag) atomicExch(p.error_word, 1);
}

// The backward pass of rows of 4097 to 8192 elements: a block of 16 warps a row.  The column sums are added up in shared
// memory, where each thread keeps its own columns (five vectors of such a row do not fit beside it in registers, and a
// second pass over the batch for them would double the traffic).
__device__ __forceinline__ void add_to(float4* sum, const float4& v) {
  float4 s = *sum;
  s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  *sum = s;
}
template <int VEC>
static __global__ void __launch_bounds__(512)
residual_norm_bwd_long_kernel(NormGradArgs p) {
  pdl_prologue();
  constexpr int WARPS = 16, VPT = 4, TEAM = 32 * WARPS, VECTOR = VPT * TEAM;     // float4s of one column sum
  extern __shared__ float4 norm_smem[];                // [sums (+ 1 for the gate)][VECTOR]
  __shared__ float2 red[2][32];
  int flip = 0;
  const int t = threadIdx.x;
  const float inv_dim = 1.0f / p.dim;
  const int vectors = p.sums + (p.dgate != nullptr);
  float4* const mine = norm_smem + t;
  float4* const gate_sum = mine + p.sums * VECTOR;
  for (int k = 0; k < vectors; ++k)
#pragma unroll
    for (int j = 0; j < VPT; ++j) mine[k * VECTOR + j * TEAM] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
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
          if (p.dgate || p.slot[SUM_GATE] >= 0) {
            const float4 pb = param_load<TEAM, VEC>(p.post_beta, j, t, p.dim, 0.0f);
            float4 w;
#pragma unroll
            for (int k = 0; k < 4; ++k) lane_set(w, k, p.b * lane_get(d[j], k) * fmaf(lane_get(h[j], k), lane_get(pg, k), lane_get(pb, k)));
            add_to((p.dgate ? gate_sum : mine + p.slot[SUM_GATE] * VECTOR) + j * TEAM, w);
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
  for (int k = 0; k < p.sums; ++k)
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      row_store<TEAM, VEC>(p.partial + (static_cast<long long>(blockIdx.x) * p.sums + k) * p.dim, j, t, p.dim, mine[k * VECTOR + j * TEAM]);
}

// The column sums of all blocks, one launch for every vector: row y < sums of the grid adds vector y over the blocks'
// parts, the others a row of the gate over its pieces.  32 warps each take every 32nd part, and their sums are added in
// order.
struct NormSums {
  const float *partial, *gate_partial;
  int parts, pieces, sums, dim;
  float* out[SUM_COUNT];
  float* gate;                   // of a gate that changes with the rows
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
