// Rows of logits and operations over a wave's lanes: shared by the kernels that verify and draw tokens.
#pragma once
#include <cfloat>

#include "wq_common.h"

namespace agq {

// What a temperature makes of differences of logits.
struct Heat {
  bool greedy;
  float heat;
  // log2(e) / T in two parts: one of 24 bits alone shifts all exponents the same way, so the row's sum by up to 2^-24 times
  // the mean exponent.  T counts as at least fp32's smallest normal number, and as 1.44e30 at most.
  float scale, scale_lo;
  float least;  // a difference of logits whose weight is 0 (2^-300), as is that of all below: its products are numbers at any T
};
__device__ __forceinline__ Heat heat_of(float temp) {
  Heat s;
  s.greedy = !(temp > 0.0f);
  s.heat = s.greedy ? 1.0f : temp;
  const float heat = fminf(fmaxf(s.heat, FLT_MIN), 1.44e30f);
  const double scale = 1.44269504088896340736 / (double)heat;
  s.scale = (float)scale;
  s.scale_lo = (float)(scale - (double)s.scale);
  s.least = -208.0f * heat;
  return s;
}

// The weight of logit l in a row whose largest is top (not +inf).  The clamp takes a masked logit's -inf, and NaN, to a
// difference whose weight is 0.
__device__ __forceinline__ float weight(const Heat& s, float l, float top) {
  const float d = fmaxf(l - (top == -INFINITY ? 0.0f : top), s.least);
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, s.scale, d * s.scale_lo));
}
// Of any row: where the largest is +inf, all that are it weigh the same.
__device__ __forceinline__ float any_weight(const Heat& s, float l, float top) {
  return top == INFINITY ? (l == top ? 1.0f : 0.0f) : weight(s, l, top);
}
// 8 logits from token k on, -inf past the end.  Rows begin at any even address.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
__device__ __forceinline__ void load8(const uint16_t* row, int k, int vocab, float* l) {
  if (k + 8 <= vocab) {
    const u32x4 v = *reinterpret_cast<const u32x4_any*>(row + k);
#pragma unroll
    for (int i = 0; i < 8; ++i) l[i] = __uint_as_float(i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) l[i] = k + i < vocab ? bf2f(row[k + i]) : -INFINITY;
  }
}

// Over the lanes of a wave, by DPP (an LDS exchange takes several times as long): x of the lane `ctrl` names, `none` where
// there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t x, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xF, false);
}
// op over the lanes up to each one: row_shr 1, 2, 4, 8 within the rows of 16, then the rows' last lanes
template <class T, class Op>
__device__ __forceinline__ T wave_scan(T x, Op op) {
  x = op.template step<0x111, 0xF>(x);
  x = op.template step<0x112, 0xF>(x);
  x = op.template step<0x114, 0xF>(x);
  x = op.template step<0x118, 0xF>(x);
  x = op.template step<0x142, 0xA>(x);  // row_bcast 15
  return op.template step<0x143, 0xC>(x);  // row_bcast 31
}
struct Add {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ double step(double x) const {
    const uint64_t v = (uint64_t)__double_as_longlong(x);
    return x + __longlong_as_double((long long)((uint64_t)dpp<CTRL, ROWS>((uint32_t)(v >> 32), 0) << 32 |
                                                dpp<CTRL, ROWS>((uint32_t)v, 0)));
  }
};
struct Max {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ float step(float x) const {
    return fmaxf(x, __uint_as_float(dpp<CTRL, ROWS>(__float_as_uint(x), 0xFF800000u)));
  }
};
struct Min {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ int step(int x) const {
    return min(x, (int)dpp<CTRL, ROWS>((uint32_t)x, 0x7FFFFFFFu));
  }
};
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
__device__ __forceinline__ double wave_sum(double x) {
  const uint64_t v = (uint64_t)__double_as_longlong(wave_scan(x, Add()));
  return __longlong_as_double((long long)((uint64_t)last_lane((uint32_t)(v >> 32)) << 32 | last_lane((uint32_t)v)));
}
__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(last_lane(__float_as_uint(wave_scan(x, Max()))));
}
__device__ __forceinline__ int wave_min(int x) { return (int)last_lane((uint32_t)wave_scan(x, Min())); }

}  // namespace agq
