// Microscaled formats: blocks of 32 elements along a row share one power of two.
//
//   4 bits  codes sign | 2 exponent bits | 1 mantissa bit, magnitudes {0, .5, 1, 1.5, 2, 3, 4, 6}; the earlier element
//           in the low half of a byte, 16 bytes a block; block scale 2^(floor(log2 max|v|) - 2)
//   8 bits  integers -127..127 in units of scale / 64, 32 bytes a block; block scale 2^floor(log2 max|v|)
//
// A scale 2^e is the byte e + 127, at least 0; the byte 255 marks a block that held a NaN or an infinity and makes all
// of it NaN.  Rows are padded to whole blocks (codes 0).  Every quotient by a scale is exact, so the only rounding is
// the one to the code (nearest even), and a code times its scale is exact in bf16: 7 and 2 significant bits against 8,
// the smallest steps 2^-133 and 2^-128 against 2^-133.
#pragma once

#include "common.h"

namespace dimq {

constexpr int kMxBlock = 32;
constexpr uint32_t kMxNan = 255;

inline int64_t mx_blocks(int64_t cols) { return (cols + kMxBlock - 1) / kMxBlock; }

inline int mx_check_rows(const char* what, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld) {
  DIMQ_CHECK(dtype == DIMQ_F32 || dtype == DIMQ_F16 || dtype == DIMQ_BF16, "%s: dtype must be fp32, fp16 or bf16", what);
  DIMQ_CHECK(rows >= 0 && cols >= 0, "%s: sizes must not be negative", what);
  DIMQ_CHECK(rows <= 1 || ld >= cols, "%s: row stride %lld is below the row length %lld", what, (long long)ld,
             (long long)cols);
  DIMQ_CHECK(rows == 0 || cols == 0 || x, "%s: null pointer", what);
  return DIMQ_OK;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// The scale byte of a block whose largest magnitude has the fp32 bits `top`: its biased exponent less EMAX (2 for 4
// bits, 0 for 8), which is floor(log2) for normal numbers; subnormal ones have exponent field 0 and take the least scale.
template <int EMAX>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? kMxNan : (e > (uint32_t)EMAX ? e - EMAX : 0u);
}

// 2^(byte - 127) as the operand of the scaled conversions, which read its exponent field alone (field 0: 2^-127,
// field 255: NaN).
__device__ __forceinline__ float mx_scale_operand(uint32_t byte) { return __uint_as_float(byte << 23); }

// The value of one 8-bit step: 2^(byte - 127) / 64, NaN for byte 255.
__device__ __forceinline__ float mx_step8(uint32_t byte) {
  return byte == kMxNan ? __uint_as_float(0x7fc00000u) : ldexpf(1.0f, (int)byte - 133);
}

// Eight fp32 values -> eight 4-bit codes, to nearest even, saturating.
__device__ __forceinline__ uint32_t mx_codes4(const float (&v)[8], float scale) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
}

// Phi(-a) exp(a^2 / 2), 0 <= a, as t P(t) with t = 1 / (1 + k a): P by weighted least squares on Chebyshev nodes of t
// over a <= 14 with P(1) = 1/2, the weights moved towards equal relative errors, and so exact at a = 0, the value of most
// zeros of a quantized block.  FINE (fp32 outputs): 8 coefficients, 5e-7 as evaluated in fp32; otherwise 7, 1.2e-6.
template <bool FINE>
__device__ __forceinline__ float mx_tail_factor(float a) {
  if constexpr (FINE) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.2333452377915607f, a, 1.0f));
    float r = -0.067649900913238525f;
    r = fmaf(r, t, 0.23002518713474274f);
    r = fmaf(r, t, -0.17541733384132385f);
    r = fmaf(r, t, 0.2041075974702835f);
    r = fmaf(r, t, 0.023684635758399963f);
    r = fmaf(r, t, 0.10058960318565369f);
    r = fmaf(r, t, 0.091481544077396393f);
    r = fmaf(r, t, 0.09317866712808609f);
    return r * t;
  }
  const float t = __builtin_amdgcn_rcpf(fmaf(0.36f, a, 1.0f));
  float r = 0.04709881659085434f;
  r = fmaf(r, t, -0.17988737532749394f);
  r = fmaf(r, t, 0.18109358442700213f);
  r = fmaf(r, t, 0.02646958676291894f);
  r = fmaf(r, t, 0.13974328500731586f);
  r = fmaf(r, t, 0.14176884610587542f);
  r = fmaf(r, t, 0.14371325643352723f);
  return r * t;
}

// exp(-a^2 / 4).  Products take it twice, so that they reach the subnormal numbers, which the exponential itself flushes.
// FINE: the argument's roundings, 2^-24 of up to 150, are carried along and applied to first order.
template <bool FINE>
__device__ __forceinline__ float mx_exp_quarter(float a) {
  constexpr float kC = -0.36067376022224085f;  // -log2(e) / 4
  if constexpr (!FINE) return __builtin_amdgcn_exp2f(a * a * kC);
  constexpr float kLow = (float)(-0.36067376022224085187998 - (double)kC);
  const float q = a * a, t = q * kC;
  const float low = fmaf(q, kLow, fmaf(fmaf(a, a, -q), kC, fmaf(q, kC, -t)));
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, low * 0.69314718055994531f, e);
}

// h Phi(h) = max(h, 0) - a Phi(-a), a = |h|, which keeps the negative tail's relative error (1e-6; not FINE, for outputs of
// 16 bits: 1.5e-5 where the tail is 1e-37) where 1 + erf would cancel.  a stops at 40, where the tail is 0: infinity times 0.
template <bool FINE>
__device__ __forceinline__ float mx_gelu(float h) {
  const float a = fminf(fabsf(h), 40.0f), m = mx_tail_factor<FINE>(a);
  const float root = mx_exp_quarter<FINE>(a);
  return fmaf(-(a * m * root), root, 0.5f * (h + fabsf(h)));  // the last sum keeps NaN
}

// d gelu / dh = Phi(h) + h phi(h)
template <bool FINE>
__device__ __forceinline__ float mx_gelu_slope(float h) {
  const float a = fminf(fabsf(h), 40.0f), m = mx_tail_factor<FINE>(a), c = h * 0.39894228040143268f;
  const float root = mx_exp_quarter<FINE>(a), tail = m * root * root;
  return fmaf(c * root, root, h < 0.0f ? tail : 1.0f - tail);
}

}  // namespace dimq
