// 4-bit codes as matrix operands (gfx950), shared by w4.hip and kv4.hip.
//
// A code u in the top four mantissa bits of a 16-bit float whose exponent is that of 16 is the number
// 16 + u, exactly: bf16 0x4180 | u << 3, fp16 0x4c00 | u << 6.  So two codes, one in each half of a
// word, become two operand elements with a shift and an and-or, and the products are corrected once
// per group: sum (u - z) x = sum (16 + u) x - (16 + z) sum x.  (Offsets 128 + u and 1024 + u, which
// need no shift, would cost three to six more bits of the fp32 sums.)
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mq_device.h"

#define NB_OFFSET 16.0f

typedef float nb_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 nb_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 nb_f16x8 __attribute__((ext_vector_type(8)));

// Codes F and F + 4 of a word (bits 4F.. and 16 + 4F..) as the elements 16 + u.  The constants are in
// registers that the compiler cannot see through: as literals, the and and the or are an instruction each.
template <bool F16, int F> MQ_DEV uint32_t nb_pair(uint32_t w) {
  constexpr int at = F16 ? 6 : 3, sh = 4 * F - at;
  uint32_t m = F16 ? 0x03c003c0u : 0x00780078u, one = F16 ? 0x4c004c00u : 0x41804180u;
  asm("" : "+s"(m));
  asm("" : "+v"(one));
  return ((sh < 0 ? w << (sh < 0 ? -sh : 0) : w >> (sh > 0 ? sh : 0)) & m) | one;
}
// The 8 codes of a word as an operand: elements 2f and 2f + 1 are codes f and f + 4.
template <bool F16> MQ_DEV uint4 nb_expand8(uint32_t w) {
  return make_uint4(nb_pair<F16, 0>(w), nb_pair<F16, 1>(w), nb_pair<F16, 2>(w), nb_pair<F16, 3>(w));
}
// 8 consecutive 16-bit elements in the order of nb_expand8
MQ_DEV uint4 nb_order8(uint4 x) {
  return make_uint4(__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                    __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u));
}

// 16 x 16 x 32 product: lane l holds row (a) or column (b) l % 16 and the products' elements
// 8 (l / 16) .. + 8; the result's column l % 16, rows 4 (l / 16) .. + 4.
template <bool F16> MQ_DEV nb_f32x4 nb_mfma(uint4 a, uint4 b, nb_f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(nb_f16x8, a), __builtin_bit_cast(nb_f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(nb_bf16x8, a), __builtin_bit_cast(nb_bf16x8, b), c, 0, 0, 0);
}

template <bool F16> MQ_DEV float nb_lo(uint32_t w) {
  return F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)w) : bf16_lo(w);
}
template <bool F16> MQ_DEV float nb_hi(uint32_t w) {
  return F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)) : bf16_hi(w);
}
// 16 bytes at any 2-byte aligned address
struct __attribute__((packed, aligned(2))) NbLoose16 {
  uint32_t w[4];
};
MQ_DEV uint4 nb_load16(const uint16_t* p) {
  const NbLoose16 v = *(const NbLoose16*)p;
  return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}
