// Elements of a paged cache: fp16, or 8-bit codes with an fp16 scale per row and KV
// head.  A row of codes c and scale s stands for the fp16 values c s (one rounding: a
// code's and a scale's product has 19 bits), which is what every reader takes, so that
// rows read back are those that the attention sees.
#pragma once

#include <type_traits>

#include "ec_device.h"
#include "ec_kernels.h"

namespace ec {

// The scale of a row whose largest is `top`: the smallest fp16 number that is not below
// top / Q, so that no code passes Q.  Below the smallest normal fp16 its steps are coarse,
// and a code's step with them, but no value is further off than half the scale.  NaN for a
// row of infinities, or beyond what scales reach: such a row stands for NaN.
__device__ __forceinline__ uint16_t cache_scale(double top, int type) {
  const double t = top / (type == CACHE_I8 ? 127.0 : 448.0);
  uint16_t h = f2h((float)t);
  if ((double)h2f(h) < t) h++;
  return h >= 0x7C00 ? 0x7E00 : h;
}

// y / s to the nearest code, ties to the even one
__device__ __forceinline__ int cache_code_i8(double y, double s) {
  const double z = s > 0.0 ? rint(y / s) : 0.0;
  return (int)fmin(fmax(z, -127.0), 127.0);
}
// fp64 -> fp32 for a rounding to follow: towards zero, with the last bit set where that
// is inexact
__device__ __forceinline__ float to_odd(double z) {
  const float f = (float)z;
  uint32_t u = __builtin_bit_cast(uint32_t, f);
  if ((double)f != z) {
    if (fabs((double)f) > fabs(z)) u--;
    u |= 1;
  }
  return __builtin_bit_cast(float, u);
}
__device__ __forceinline__ float cache_code_e4m3(double y, double s) {  // not yet rounded
  return s > 0.0 ? to_odd(fmin(fmax(y / s, -448.0), 448.0)) : 0.0f;
}

__device__ __forceinline__ uint16_t cache_f16(double y) { return f2h(to_odd(y)); }

__device__ __forceinline__ void cache_store(void *p, int type, size_t at, double y, uint16_t scale) {
  const double s = h2f(scale);
  if (type == CACHE_F16) ((uint16_t *)p)[at] = cache_f16(y);
  else if (type == CACHE_I8) ((int8_t *)p)[at] = (int8_t)cache_code_i8(y, s);
  else ((uint8_t *)p)[at] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(cache_code_e4m3(y, s), 0.0f, 0, false);
}

typedef uint32_t v2u __attribute__((ext_vector_type(2)));
// two codes of a word (its low or high half) as fp16, times the scale
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
template <int TYPE, bool HI>
__device__ __forceinline__ v2h cache_pair(uint32_t w, v2h scale) {
  if constexpr (TYPE == CACHE_I8) {
    // 1024 + 128 + c has the bits 0x6400 + 128 + c
    const uint32_t b = __builtin_amdgcn_perm(w ^ 0x80808080u, 0x64646464u, HI ? 0x00070006u : 0x00050004u);
    return (__builtin_bit_cast(v2h, b) - (v2h)(_Float16)1152.0f) * scale;
  } else {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI) * scale;
  }
}

// eight elements of 16 or 8 bits as they come from the cache
template <int TYPE>
using Raw8 = std::conditional_t<TYPE == CACHE_F16, v4u, v2u>;
template <int TYPE>
__device__ __forceinline__ v4u to_f16(Raw8<TYPE> r, uint16_t scale) {
  if constexpr (TYPE == CACHE_F16) return r;
  else {
    const v2h s = (v2h)__builtin_bit_cast(_Float16, scale);
    return v4u{__builtin_bit_cast(uint32_t, cache_pair<TYPE, false>(r.x, s)), __builtin_bit_cast(uint32_t, cache_pair<TYPE, true>(r.x, s)),
               __builtin_bit_cast(uint32_t, cache_pair<TYPE, false>(r.y, s)), __builtin_bit_cast(uint32_t, cache_pair<TYPE, true>(r.y, s))};
  }
}
// element e of row `row`, in fp16 bits
__device__ __forceinline__ uint16_t cache_value(const void *p, const uint16_t *scale, int type, size_t row, int hd, int e) {
  const size_t at = row * hd + e;
  if (type == CACHE_F16) return ((const uint16_t *)p)[at];
  const uint32_t c = ((const uint8_t *)p)[at];
  const v2h s = (v2h)__builtin_bit_cast(_Float16, scale[row]);
  return __builtin_bit_cast(uint16_t, type == CACHE_I8 ? cache_pair<CACHE_I8, false>(c, s).x : cache_pair<CACHE_E4M3, false>(c, s).x);
}

}  // namespace ec
