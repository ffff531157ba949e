// What the attention kernels on 16-bit tiles share: fp32 numbers as two 16-bit
// parts, the tiles' places in LDS, reductions over the lanes of a row.
#pragma once

#include "ec_device.h"

namespace ec {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// chunk c (16 bytes) of a tile's row r is at chunk c ^ swz(r): the 16-byte reads
// of one chunk by 8 consecutive rows fall on distinct banks
template <int HD>
__device__ __forceinline__ int swz(int r) {
  return HD % 64 == 0 ? r & 7 : (r >> 1) & 3;
}

// the bits 0 .. n - 1 (n up to 64, below 0 none)
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0 : (1ull << n) - 1; }

// the maximum and the sum over the four lanes lr, lr + 16, lr + 32, lr + 48: the
// halves, then the odd and the even rows of 16 change places
__device__ __forceinline__ float row_max(float v) {
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  v2u x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(x.x), __uint_as_float(x.y));
  x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x.x), __uint_as_float(x.y));
}
__device__ __forceinline__ float row_sum(float v) {
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  v2u x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(x.x) + __uint_as_float(x.y);
  x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x.x) + __uint_as_float(x.y);
}

// two values times 2^LIFT in two 16-bit parts each: hi their nearest 11 bits (the lift
// comes with the rounding, in one addition to the value's bits), lo the rest, both stored
// as the nearest 16-bit value.  Nothing is cut: what is lost below the 16-bit
// steps, and of lo's products in the sums that the largest weights have filled, goes
// either way, so that many small weights lose nothing together (lo from cut bits, which
// is one instruction a value less, is never negative: 1.4e-5 instead of 1.9e-6 off over
// 32600 positions of which the first takes 0.99, and 2 of 42 us faster for the long
// contexts).  The nearest 16-bit value and a mixed-precision difference would be three
// instructions, not eight, but those take 8 cycles each, these 2: 43 us, and 20 instead
// of 16.5 for the one-token sequences.
struct Parts {
  uint32_t hi, lo;
};
template <int LIFT = 0>
__device__ __forceinline__ Parts split2(float x, float y) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  constexpr uint32_t up = 0x1000u + ((uint32_t)LIFT << 23);
  constexpr float lift = 1 << LIFT;
  const float hx = __uint_as_float((__float_as_uint(x) + up) & 0xFFFFE000u),
              hy = __uint_as_float((__float_as_uint(y) + up) & 0xFFFFE000u);
  return Parts{__builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{hx, hy}), v2h)),
               __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{__builtin_fmaf(x, lift, -hx), __builtin_fmaf(y, lift, -hy)}), v2h))};
}
__device__ __forceinline__ float half_of(v4u v, int e) { return h2f((uint16_t)(v[e >> 1] >> (16 * (e & 1)))); }

__device__ __forceinline__ v4f mma(v4u a, v4u b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Operands of ND groups of 16 elements, from rows 32 u .. 32 u + 31 of the
// tile: lane l of 16 names 8 bytes of row l / 4 and gets element l of the four
// rows.  The builtin would wait for every load that is on its way into LDS, the
// next tile's too.
template <int HD, int ND>
__device__ __forceinline__ void read_v(const uint32_t *at, uint32_t base, int u, v4u (&v)[ND]) {
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  static_assert(ND == 2 || ND == 4, "groups of elements");
  v2u x[2 * ND];
  if constexpr (ND == 2) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
        "ds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
        "ds_read_b64_tr_b16 %2, %5 offset:%6\n\t"
        "ds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
        : "v"(base + at[0]), "v"(base + at[1]), "i"(64 * HD * u), "i"(64 * HD * u + 32 * HD)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
        "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
        "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
        : "v"(base + at[0]), "v"(base + at[1]), "v"(base + at[2]), "v"(base + at[3]), "i"(64 * HD * u),
          "i"(64 * HD * u + 32 * HD)
        : "memory");
  }
#pragma unroll
  for (int e = 0; e < ND; e++) v[e] = v4u{x[2 * e].x, x[2 * e].y, x[2 * e + 1].x, x[2 * e + 1].y};
}

}  // namespace ec
