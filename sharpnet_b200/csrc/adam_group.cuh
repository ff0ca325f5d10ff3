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
constexpr int kAdamChunk8 = 2048;     // elements of one work item, moments in 8 bits: a block per warp

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
// tensors fill 30472; the small table keeps a small model's launch from copying as much.
constexpr int kAdamMaxTensors = 448;
template <int N> struct AdamTable {
  int n;
  unsigned total;          // work items of all tensors
  unsigned first[N];
  AdamTensor t[N];
};
struct AdamCoefficients { float beta1, beta2, eps, factor; };

// The tensor whose work items include `item`: the last one whose first item is not above it.
template <int N>
__device__ __forceinline__ int adam_find(const AdamTable<N>& table, unsigned item) {
  int lo = 0, hi = table.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table.first[mid] <= item) lo = mid; else hi = mid;
  }
  return lo;
}

// The update of adam_one (elementwise.cuh) with its roundings written out, so that an element's result does not depend
// on the access width that its tensor's alignment allows (the compiler contracts the two forms of adam_one differently).
__device__ __forceinline__ void adam32_one(const AdamCoefficients& c, float wd, float g, float& w, float& v, float& s) {
  v = __fmaf_rn(c.beta1, v, __fmul_rn(1.0f - c.beta1, g));
  s = __fmaf_rn(c.beta2, s, __fmul_rn(__fmul_rn(1.0f - c.beta2, g), g));
  w = __fsub_rn(w, __fmaf_rn(wd, w, __fdiv_rn(__fmul_rn(c.factor, v), __fadd_rn(__fsqrt_rn(s), c.eps))));
}

template <int N>
static __global__ void __launch_bounds__(kAdamThreads)
adam_group32_kernel(const __grid_constant__ AdamTable<N> table, const AdamCoefficients c) {
  pdl_prologue();
  for (unsigned item = blockIdx.x; item < table.total; item += gridDim.x) {
    const int which = adam_find(table, item);
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
// r * inverse(scale), rounded at random to an e4m3 value; rnd: 20 random bits.
__device__ __forceinline__ float adam8_round(float x, unsigned rnd) {
  const float high = __uint_as_float((__float_as_uint(x) + rnd) & ~0xFFFFFu);
  const float low = fmaxf(floorf(__fadd_rn(x * 512.0f, static_cast<float>(rnd) * 0x1p-20f)), 1.0f) * 0x1p-9f;
  return x < 0x1p-6f ? (x > 0.0f ? low : 0.0f) : high;
}
__device__ __forceinline__ float2 adam8_decode2(unsigned short codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ unsigned short adam8_encode2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// One element: moments in, moments and weight out; returns the root of s.
__device__ __forceinline__ float adam8_one(const AdamCoefficients& c, float wd, float g, float& w, float& v, float r) {
  v = __fadd_rn(__fmul_rn(c.beta1, v), __fmul_rn(1.0f - c.beta1, g));
  const float s = __fadd_rn(__fmul_rn(c.beta2, __fmul_rn(r, r)), __fmul_rn(__fmul_rn(1.0f - c.beta2, g), g));
  const float root = __fsqrt_rn(s);
  w = __fsub_rn(w, __fmaf_rn(wd, w, __fdiv_rn(__fmul_rn(c.factor, v), __fadd_rn(root, c.eps))));
  return root;
}

template <int N>
static __global__ void __launch_bounds__(kAdamThreads)
adam_group8_kernel(const __grid_constant__ AdamTable<N> table, const AdamCoefficients c, const unsigned seed) {
  pdl_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (unsigned item = blockIdx.x; item < table.total; item += gridDim.x) {
    const int which = adam_find(table, item);
    const AdamTensor& t = table.t[which];
    const long long block = static_cast<long long>(item - table.first[which]) * (kAdamChunk8 / kAdamBlock8) + warp;
    const long long base = block * kAdamBlock8;
    if (base >= t.count) continue;                     // the same for the whole warp
    const float wd = t.weight_decay;
    const float* g = t.g + base;
    float* w = t.w + base;
    unsigned char* vc = static_cast<unsigned char*>(t.v) + base;
    unsigned char* sc = static_cast<unsigned char*>(t.s) + base;
    const float v_scale = t.v_scale[block], s_scale = t.s_scale[block];
    const unsigned key = seed * 0x9E3779B1u + (t.ordinal_vec >> 1) * 0x85EB9A77u + static_cast<unsigned>(base >> 1);
    const int count = static_cast<int>(min(static_cast<long long>(kAdamBlock8), t.count - base));
    const bool whole = (t.ordinal_vec & 1) && count == kAdamBlock8;
    // lane's elements: 4 lane + k and 128 + 4 lane + k
    float gv[8], wv[8], vv[8], rv[8];
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 a = reinterpret_cast<const float4*>(g)[32 * j + lane], b = reinterpret_cast<const float4*>(w)[32 * j + lane];
        const unsigned vq = reinterpret_cast<const unsigned*>(vc)[32 * j + lane], sq = reinterpret_cast<const unsigned*>(sc)[32 * j + lane];
        gv[4 * j] = a.x; gv[4 * j + 1] = a.y; gv[4 * j + 2] = a.z; gv[4 * j + 3] = a.w;
        wv[4 * j] = b.x; wv[4 * j + 1] = b.y; wv[4 * j + 2] = b.z; wv[4 * j + 3] = b.w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 p = adam8_decode2(static_cast<unsigned short>(vq >> (16 * k))), q = adam8_decode2(static_cast<unsigned short>(sq >> (16 * k)));
          vv[4 * j + 2 * k] = p.x; vv[4 * j + 2 * k + 1] = p.y;
          rv[4 * j + 2 * k] = q.x; rv[4 * j + 2 * k + 1] = q.y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = 128 * (i >> 2) + 4 * lane + (i & 3);
        const bool live = e < count;
        gv[i] = live ? g[e] : 0.0f;
        wv[i] = live ? w[e] : 0.0f;
        vv[i] = live ? adam8_decode2(vc[e]).x : 0.0f;
        rv[i] = live ? adam8_decode2(sc[e]).x : 0.0f;
      }
    }
    unsigned v_max = 0, r_max = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      vv[i] *= v_scale;
      rv[i] = adam8_one(c, wd, gv[i], wv[i], vv[i], rv[i] * s_scale);
      v_max = max(v_max, __float_as_uint(vv[i]) & 0x7fffffffu);
      r_max = max(r_max, __float_as_uint(rv[i]) & 0x7fffffffu);
    }
    const float new_v_scale = adam8_scale(__reduce_max_sync(0xffffffffu, v_max));
    const float new_s_scale = adam8_scale(__reduce_max_sync(0xffffffffu, r_max));
    const float v_inv = adam8_inverse(new_v_scale), s_inv = adam8_inverse(new_s_scale);
    unsigned vq[2] = {0, 0}, sq[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const unsigned rnd = adam8_hash(key + static_cast<unsigned>((128 * (i >> 2) + 4 * lane + (i & 3)) >> 1));
      const float a = adam8_round(rv[i] * s_inv, (rnd & 0xFFFFu) << 4), b = adam8_round(rv[i + 1] * s_inv, (rnd >> 16) << 4);
      vq[i >> 2] |= static_cast<unsigned>(adam8_encode2(vv[i] * v_inv, vv[i + 1] * v_inv)) << (8 * (i & 3));
      sq[i >> 2] |= static_cast<unsigned>(adam8_encode2(a, b)) << (8 * (i & 3));
    }
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        reinterpret_cast<float4*>(w)[32 * j + lane] = make_float4(wv[4 * j], wv[4 * j + 1], wv[4 * j + 2], wv[4 * j + 3]);
        reinterpret_cast<unsigned*>(vc)[32 * j + lane] = vq[j];
        reinterpret_cast<unsigned*>(sc)[32 * j + lane] = sq[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = 128 * (i >> 2) + 4 * lane + (i & 3);
        if (e < count) {
          w[e] = wv[i];
          vc[e] = static_cast<unsigned char>(vq[i >> 2] >> (8 * (i & 3)));
          sc[e] = static_cast<unsigned char>(sq[i >> 2] >> (8 * (i & 3)));
        }
      }
    }
    if (lane == 0) { t.v_scale[block] = new_v_scale; t.s_scale[block] = new_s_scale; }
  }
}

}  // namespace snb
