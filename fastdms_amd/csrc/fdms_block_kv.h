// The dense 8-bit block KV cache: layout and code conversions shared by its
// kernels (block tables, store, read-back, attention).
//
// Blocks of `bs` tokens (a power of two, 16 .. 256).  A kv head's part of a
// block holds, in 8-bit codes, K as rows [bs][D] and V as tiles of 16 tokens,
// each tile transposed: [bs / 16][D][16].  Both are what a lane of the matrix
// products reads: 16 consecutive channels of a K row, the 16 tokens of a tile
// for one V channel, one 16-byte load each.  One fp32 scale per (block, head)
// for K and one for V; a code stands for code * scale.  Codes are int8
// (-127 .. 127) or e4m3fn; neither ever holds a NaN or an infinity.
#pragma once

#include "fdms_common.h"

namespace fdms {

constexpr int kTile = 16;          // tokens of a V tile
constexpr int kMaxBlockLog2 = 8;   // block sizes 16 .. 256
constexpr int kMinBlockLog2 = 4;

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Four codes (byte i = code i) as halves, exactly: e4m3fn has 4 significant
// bits and exponents -9 .. 8, an int8 7 bits.  int8 goes through the halves
// 1024 + (code + 128), whose low byte is the offset code (one xor, a byte
// permute and one subtraction per pair).
template <bool FP8>
__device__ __forceinline__ void codes_to_f16(uint32_t c, uint32_t* lo, uint32_t* hi) {
  if constexpr (FP8) {
    *lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, 1.0f, false));
    *hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, 1.0f, true));
  } else {
    const uint32_t y = c ^ 0x80808080u;
    const f16x2_t off = {(f16_t)1152.0f, (f16_t)1152.0f};
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u);
    *lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, a) - off);
    *hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, b) - off);
  }
}
template <bool FP8>
__device__ __forceinline__ f16x8_t codes8_to_f16(uint32_t c0, uint32_t c1) {
  u32x4_t r;
  uint32_t a, b;
  codes_to_f16<FP8>(c0, &a, &b);
  r[0] = a;
  r[1] = b;
  codes_to_f16<FP8>(c1, &a, &b);
  r[2] = a;
  r[3] = b;
  return __builtin_bit_cast(f16x8_t, r);
}

// One code's value, byte `i` of c.
template <bool FP8>
__device__ __forceinline__ float code_value(uint32_t c, int i) {
  const uint32_t b = (c >> (8 * i)) & 0xFFu;
  if constexpr (FP8) return fp8_to_f32(b);
  return (float)(int)(int8_t)b;
}

// Codes of four values already divided by the scale (finite or infinite; the
// callers have turned NaN to 0): to nearest, ties to even, saturating.
template <bool FP8>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (FP8) return f32x4_to_fp8x4_finite(a, b, c, d);
  const float x[4] = {a, b, c, d};
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r |= ((uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_rintf(x[i]), -127.0f, 127.0f) & 0xFFu) << (8 * i);
  return r;
}

// The least power of two s with amax <= top * s, top the type's largest code
// (127 = 1.984375 * 2^6, 448 = 1.75 * 2^8), at least 2^-126.  An infinite amax
// counts as the largest float.  Powers of two keep x / s, code * s and a
// block's change of scale exact: the codes of a block are a function of its
// values, whatever computes them, and a code's value is a bf16.  They cost an
// int8 block at most one of its seven bits.
template <bool FP8>
__device__ __forceinline__ float block_scale(float amax) {
  constexpr int kExp = FP8 ? 8 : 6;
  const float top = FP8 ? 448.0f : 127.0f;
  amax = fminf(amax, 3.40282347e38f);
  int e = max((int)(__float_as_uint(amax) >> 23) - 127 - kExp, -126);
  if (amax > top * __uint_as_float((uint32_t)(e + 127) << 23)) ++e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ float nan_to_zero(float x) { return x == x ? x : 0.0f; }

}  // namespace fdms
