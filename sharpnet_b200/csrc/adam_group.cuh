// One Adam / AdamW step over many parameter tensors as one launch, with the moments in 32 bits or in 8.
//
//   v = beta1 v + (1 - beta1) dW ; s = beta2 s + (1 - beta2) dW^2 ;
//   W -= factor v / (sqrt(s) + eps) + weight_decay W ,  factor = lr sqrt(1 - beta2^t) / (1 - beta1^t)
//
// the formula of adam_update_kernel (elementwise.cuh).  The tensors are described by a table that
// travels as a kernel parameter: no copy, no workspace, and a captured launch keeps its own.
#pragma once
#include <cuda_fp8.h>

#include "elementwise.cuh"

namespace snb {

constexpr int kAdamThreads = 256;
constexpr int kAdamChunk32 = 4096;    // elements of one work item, moments in 32 bits
constexpr int kAdamBlock8 = 256;      // elements that share a scale, moments in 8 bits: one warp's work
constexpr int kAdamChunk8 = 4096;     // elements of one work item, moments in 8 bits: two blocks per warp

struct AdamTensor {
  const float* g;
  float* w;
  void* v;
  void* s;
  float* v_scale;
  float* s_scale;
  long long count;
  float weight_decay;
  unsigned ordinal_vec;   // the tensor's place in the caller's list << 1, and whether its pointers allow vector accesses
};
// N tensors and the number of the first work item of each.  A kernel takes at most 32764 bytes of parameters: 448
// tensors fill 30472.  Up to 32 tensors take a small one: the launch copies the whole parameter, and a step of 16 tensors
// costs the host 5.8 us instead of 8.6 (the device the same 4.5).
constexpr int kAdamMaxTensors = 448;
template <int N> struct AdamTable {
  int n;
  unsigned total;          // work items of all tensors
  unsigned first[N + 1];   // and behind the last tensor
  AdamTensor t[N];
};
struct AdamCoefficients { float beta1, beta2, eps, factor, minus_zero; };

// The tensor whose work items include `item`: the last one whose first item is not above it, searched from `which` on (a
// block's items come in ascending order).
template <int N>
__device__ __forceinline__ int adam_find(const AdamTable<N>& table, unsigned item, int which) {
  while (item >= table.first[which + 1]) ++which;
  return which;
}

// The update of adam_one (elementwise.cuh) with its roundings written out, so that an element's result does not depend
// on the access width that its tensor's alignment allows (the compiler contracts the two forms of adam_one differently).
__device__ __forceinline__ void adam32_one(const AdamCoefficients& c, float wd, float g, float& w, float& v, float& s) {
  v = __fmaf_rn(c.beta1, v, __fmul_rn(1.0f - c.beta1, g));
  s = __fmaf_rn(c.beta2, s, __fmul_rn(__fmul_rn(1.0f - c.beta2, g), g));
  w = __fsub_rn(w, __fmaf_rn(wd, w, __fdiv_rn(__fmul_rn(c.factor, v), __fadd_rn(__fsqrt_rn(s), c.eps))));
}

// Bound by memory: 28 bytes an element, 57.7 us for 12.6 M of them (6.1 TB/s).
template <int N>
static __global__ void __launch_bounds__(kAdamThreads)
adam_group32_kernel(const __grid_constant__ AdamTable<N> table, const AdamCoefficients c) {
  pdl_prologue();
  int which = 0;
  for (unsigned item = blockIdx.x; item < table.total; item += gridDim.x) {
    which = adam_find(table, item, which);
    const AdamTensor& t = table.t[which];
    const long long base = static_cast<long long>(item - table.first[which]) * kAdamChunk32;
    const int count = static_cast<int>(min(static_cast<long long>(kAdamChunk32), t.count - base));
    const float* __restrict__ g = t.g + base;
    float* __restrict__ w = t.w + base;
    float* __restrict__ v = static_cast<float*>(t.v) + base;
    float* __restrict__ s = static_cast<float*>(t.s) + base;
    const float wd = t.weight_decay;
    int done = 0;
    if (t.ordinal_vec & 1) {
      const int quads = count >> 2;
      for (int i = threadIdx.x; i < quads; i += kAdamThreads) {
        const float4 gv = reinterpret_cast<const float4*>(g)[i];
        float4 wv = reinterpret_cast<float4*>(w)[i], vv = reinterpret_cast<float4*>(v)[i], sv = reinterpret_cast<float4*>(s)[i];
        adam32_one(c, wd, gv.x, wv.x, vv.x, sv.x);
        adam32_one(c, wd, gv.y, wv.y, vv.y, sv.y);
        adam32_one(c, wd, gv.z, wv.z, vv.z, sv.z);
        adam32_one(c, wd, gv.w, wv.w, vv.w, sv.w);
        reinterpret_cast<float4*>(w)[i] = wv;
        reinterpret_cast<float4*>(v)[i] = vv;
        reinterpret_cast<float4*>(s)[i] = sv;
      }
      done = quads << 2;
    }
    for (int i = done + threadIdx.x; i < count; i += kAdamThreads) {
      float wv = w[i], vv = v[i], sv = s[i];
      adam32_one(c, wd, g[i], wv, vv, sv);
      w[i] = wv; v[i] = vv; s[i] = sv;
    }
  }
}

// ---------------------------------------------------------------- moments in 8 bits
// A block of 256 elements holds v as e4m3 codes times a power of two, and the root r of s the same way (e4m3 spans 17
// binades, so r spans 34 binades of s; s itself would not fit).  The scale brings the largest magnitude of the block
// to [128, 256) and is a power of two, so scaling never rounds.
//   v: nearest, ties to even.
//   r: up or down at random, in proportion (hash of the caller's seed and the element's place).  With 1 - beta2 = 1e-3
//      s moves by a thousandth a step and three bits of mantissa would never see it under nearest rounding: r would
//      stay where it was after the first few steps.  It is rounded to zero only where it is zero, so that the
//      denominator of an element with a history never collapses to eps.
// The state is a function of the inputs bit for bit: every operation on the way to it is one rounded 32-bit operation
// in the order written here (no contraction).
__device__ __forceinline__ float adam8_scale(unsigned largest_bits) {   // bits of the largest magnitude
  if (largest_bits < (27u << 23)) return 0.0f;                          // below 2^-100: the block counts as zero
  if (largest_bits >= 0x7f800000u) return __int_as_float(0x7fffffff);   // infinity or NaN: the whole block is NaN from here on
  return __uint_as_float((largest_bits & 0x7f800000u) - (7u << 23));
}
__device__ __forceinline__ float adam8_inverse(float scale) {
  return scale > 0.0f ? __uint_as_float((254u << 23) - __float_as_uint(scale)) : 0.0f;
}
__device__ __forceinline__ unsigned adam8_hash(unsigned x) {
  x = (x ^ (x >> 16)) * 0x6C8E9CF5u;
  x = (x ^ (x >> 12)) * 0xB5297A4Du;
  return x ^ (x >> 15);
}
// r * inverse(scale) > 0, rounded at random to an e4m3 value; rnd: 20 random bits.  Below 2^-6 the values lie 2^-9 apart.
__device__ __forceinline__ float adam8_round_low(float x, unsigned rnd) {
  return fmaxf(floorf(__fadd_rn(x * 512.0f, static_cast<float>(rnd) * 0x1p-20f)), 1.0f) * 0x1p-9f;
}
__device__ __forceinline__ float adam8_round(float x, unsigned rnd) { return __uint_as_float((__float_as_uint(x) + rnd) & ~0xFFFFFu); }
__device__ __forceinline__ float2 adam8_decode2(unsigned short codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ unsigned adam8_encode2(float2 v) { return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3); }

// A warp's block of 256 elements, and whether it can be fetched in vectors.  A warp has two blocks of an item, one after
// the other.
struct AdamBlock {
  unsigned item;
  int which;
  long long block;
  bool live, whole;
  template <int N> __device__ __forceinline__ void set(const AdamTable<N>& table) {      // live and whole, from the others
    const AdamTensor& t = table.t[which];
    live = block * kAdamBlock8 < t.count;              // the same for the whole warp
    whole = (t.ordinal_vec & 1) && (block + 1) * kAdamBlock8 <= t.count;
  }
  template <int N> __device__ __forceinline__ void start(const AdamTable<N>& table, unsigned first) {
    item = first;
    live = whole = false;
    if (item >= table.total) return;
    which = adam_find(table, item, which);
    block = static_cast<long long>(item - table.first[which]) * (kAdamChunk8 / kAdamBlock8) + 2 * (threadIdx.x >> 5);
    set(table);
  }
  template <int N> __device__ __forceinline__ void next(const AdamTable<N>& table) {
    if (block & 1) { start(table, item + gridDim.x); return; }
    ++block;
    set(table);
  }
};
__device__ __forceinline__ void copy_async_16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(smem))), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_async_4(void* smem, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(smem))), "l"(global) : "memory");
}

// Bound by instructions nearly as much as by memory (the 16 bytes of an element are 73 instructions' time): pairs of
// elements go through the packed 32-bit arithmetic; the quotient of the weight's step, which no state depends on, is a
// product with the approximate reciprocal (2 ulp); the rounding below 2^-6, which few elements need, sits behind a branch.
// A block's elements are copied into shared memory slots of the thread that updates them while the block before them is
// updated (185 M parameters: 617 us without, 498 with two blocks an item; 6.0 TB/s).
template <int N>
static __global__ void __launch_bounds__(kAdamThreads, 4)
adam_group8_kernel(const __grid_constant__ AdamTable<N> table, const AdamCoefficients c, const unsigned seed) {
  pdl_prologue();
  __shared__ float4 slots4[2][4][kAdamThreads];        // g, g, w, w
  __shared__ unsigned slots1[2][4][kAdamThreads];      // codes of v, v, s, s
  const int lane = threadIdx.x & 31;
  // products that are added take a minus zero that the compiler does not know: it contracts packed products and sums into
  // one operation, which would round the state once where it is defined to round twice
  const float2 nothing = both(c.minus_zero);
  const float2 b1 = both(c.beta1), b2 = both(c.beta2), c1 = both(1.0f - c.beta1), c2 = both(1.0f - c.beta2);
  float scale_v = 0.0f, scale_s = 0.0f;
  auto fetch = [&](const AdamBlock& b, int stage) {
    if (b.live) {
      const AdamTensor& t = table.t[b.which];
      scale_v = t.v_scale[b.block];
      scale_s = t.s_scale[b.block];
      if (b.whole) {
        const long long base = b.block * kAdamBlock8 + 4 * lane;
        const unsigned char *v = static_cast<const unsigned char*>(t.v) + base, *s = static_cast<const unsigned char*>(t.s) + base;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          copy_async_16(&slots4[stage][j][threadIdx.x], t.g + base + 128 * j);
          copy_async_16(&slots4[stage][2 + j][threadIdx.x], t.w + base + 128 * j);
          copy_async_4(&slots1[stage][j][threadIdx.x], v + 128 * j);
          copy_async_4(&slots1[stage][2 + j][threadIdx.x], s + 128 * j);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  AdamBlock ahead;
  ahead.which = 0;
  ahead.start(table, blockIdx.x);
  fetch(ahead, 0);
  for (int stage = 0; ahead.item < table.total; stage ^= 1) {
    const AdamBlock now = ahead;
    const float2 v_scale = both(scale_v), s_scale = both(scale_s);
    ahead.next(table);
    fetch(ahead, stage ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (!now.live) continue;
    const AdamTensor& t = table.t[now.which];
    const long long block = now.block, base = block * kAdamBlock8;
    float* w = t.w + base;
    unsigned char* vc = static_cast<unsigned char*>(t.v) + base;
    unsigned char* sc = static_cast<unsigned char*>(t.s) + base;
    const float2 wd = both(t.weight_decay);
    const unsigned key = seed * 0x9E3779B1u + (t.ordinal_vec >> 1) * 0x85EB9A77u + static_cast<unsigned>(base >> 1) + 2 * lane;
    const int count = static_cast<int>(min(static_cast<long long>(kAdamBlock8), t.count - base));
    const bool whole = now.whole;
    // pair i of a lane: elements 128 (i / 2) + 4 lane + 2 (i % 2) and the next
    float2 gv[4], wv[4], vv[4], rv[4];
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 a = slots4[stage][j][threadIdx.x], b = slots4[stage][2 + j][threadIdx.x];
        const unsigned vq = slots1[stage][j][threadIdx.x], sq = slots1[stage][2 + j][threadIdx.x];
        gv[2 * j] = make_float2(a.x, a.y); gv[2 * j + 1] = make_float2(a.z, a.w);
        wv[2 * j] = make_float2(b.x, b.y); wv[2 * j + 1] = make_float2(b.z, b.w);
        vv[2 * j] = adam8_decode2(static_cast<unsigned short>(vq)); vv[2 * j + 1] = adam8_decode2(static_cast<unsigned short>(vq >> 16));
        rv[2 * j] = adam8_decode2(static_cast<unsigned short>(sq)); rv[2 * j + 1] = adam8_decode2(static_cast<unsigned short>(sq >> 16));
      }
    } else {
      const float* g = t.g + base;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 128 * (i >> 1) + 4 * lane + 2 * (i & 1);
        const bool x = e < count, y = e + 1 < count;
        gv[i] = make_float2(x ? g[e] : 0.0f, y ? g[e + 1] : 0.0f);
        wv[i] = make_float2(x ? w[e] : 0.0f, y ? w[e + 1] : 0.0f);
        vv[i] = adam8_decode2(static_cast<unsigned short>((x ? vc[e] : 0u) | (y ? vc[e + 1] : 0u) << 8));
        rv[i] = adam8_decode2(static_cast<unsigned short>((x ? sc[e] : 0u) | (y ? sc[e + 1] : 0u) << 8));
      }
    }
    float v_max = 0.0f;
    unsigned r_max = 0, r_min = 0xffffffffu;           // r_min: of the bits less one, so that a zero is the largest
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 r = mul2(rv[i], s_scale);
      vv[i] = add2(fma2(b1, mul2(vv[i], v_scale), nothing), fma2(c1, gv[i], nothing));
      const float2 s = add2(fma2(b2, mul2(r, r), nothing), fma2(mul2(c2, gv[i]), gv[i], nothing));
      rv[i] = make_float2(__fsqrt_rn(s.x), __fsqrt_rn(s.y));
      const float2 d = add2(rv[i], both(c.eps)), n = mul2(both(c.factor), vv[i]);
      const float2 step = fma2(wd, wv[i], make_float2(__fdividef(n.x, d.x), __fdividef(n.y, d.y)));
      wv[i] = add2(wv[i], make_float2(-step.x, -step.y));
      v_max = fmaxf(v_max, fmaxf(fabsf(vv[i].x), fabsf(vv[i].y)));
      r_max = max(r_max, max(__float_as_uint(rv[i].x), __float_as_uint(rv[i].y)));
      r_min = min(r_min, min(__float_as_uint(rv[i].x) - 1u, __float_as_uint(rv[i].y) - 1u));
    }
    r_max = __reduce_max_sync(0xffffffffu, r_max);
    unsigned v_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(v_max));
    if (r_max >= 0x7f800000u) {                        // a gradient is not finite (the maximum of floats passes a NaN over)
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max(m, max(__float_as_uint(vv[i].x) & 0x7fffffffu, __float_as_uint(vv[i].y) & 0x7fffffffu));
      v_bits = __reduce_max_sync(0xffffffffu, m);
      r_max = 0x7f800000u;                             // (a NaN may carry its sign)
    }
    const float new_v_scale = adam8_scale(v_bits), new_s_scale = adam8_scale(r_max);
    const float2 v_inv = both(adam8_inverse(new_v_scale)), s_inv = both(adam8_inverse(new_s_scale));
    const bool low = r_min < __float_as_uint(0x1p-6f * new_s_scale) - 1u;
    unsigned vq[2], sq[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned rnd = adam8_hash(key + 64u * (i >> 1) + (i & 1));
      const unsigned ra = (rnd & 0xFFFFu) << 4, rb = (rnd >> 16) << 4;
      const float2 x = mul2(rv[i], s_inv);
      float2 y = make_float2(adam8_round(x.x, ra), adam8_round(x.y, rb));
      if (low) {
        if (x.x < 0x1p-6f && x.x > 0.0f) y.x = adam8_round_low(x.x, ra);
        if (x.y < 0x1p-6f && x.y > 0.0f) y.y = adam8_round_low(x.y, rb);
      }
      const unsigned v = adam8_encode2(mul2(vv[i], v_inv)), s = adam8_encode2(y);
      if (i & 1) { vq[i >> 1] |= v << 16; sq[i >> 1] |= s << 16; } else { vq[i >> 1] = v; sq[i >> 1] = s; }
    }
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        reinterpret_cast<float4*>(w)[32 * j + lane] = make_float4(wv[2 * j].x, wv[2 * j].y, wv[2 * j + 1].x, wv[2 * j + 1].y);
        reinterpret_cast<unsigned*>(vc)[32 * j + lane] = vq[j];
        reinterpret_cast<unsigned*>(sc)[32 * j + lane] = sq[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = 128 * (i >> 2) + 4 * lane + (i & 3);
        if (e < count) {
          w[e] = i & 1 ? wv[i >> 1].y : wv[i >> 1].x;
          vc[e] = static_cast<unsigned char>(vq[i >> 2] >> (8 * (i & 3)));
          sc[e] = static_cast<unsigned char>(sq[i >> 2] >> (8 * (i & 3)));
        }
      }
    }
    if (lane == 0) { t.v_scale[block] = new_v_scale; t.s_scale[block] = new_s_scale; }
  }
}

}  // namespace snb
