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

// GELU and its slope for outputs of type DT.  With a = |h|:
//
//   h Phi(h)              = max(h, 0) - a Phi(-a)
//   d gelu / dh = Phi(h) + h phi(h),  Phi(h) = Phi(-a) or 1 - Phi(-a)
//
// which keep the negative tail's relative error where 1 + erf would cancel.  Phi(-a) exp(a^2 / 2) is t P(t) with
// t = 1 / (1 + k a): P by weighted least squares on Chebyshev nodes of t over a <= 14 with P(1) = 1/2, the weights moved
// towards equal relative errors, and so exact at a = 0, the value of most zeros of a quantized block.  As evaluated in
// fp32: 8 coefficients for fp32 outputs 5e-7, 7 for fp16 1.2e-6, 6 for bf16 5.9e-6.  a comes as 64ths and stops at 64 (by
// the multiplication's own clamp), where the tail is 0: infinity times 0.
__device__ __forceinline__ float mx_64ths(float h) { return __builtin_amdgcn_fmed3f(fabsf(h) * 0.015625f, 0.0f, 1.0f); }

// SCALE: a power of two that the coefficients take along.
template <int DT, int SCALE = 1>
__device__ __forceinline__ float mx_tail_factor(float b) {
  if constexpr (DT == DIMQ_F32) {
    const float t = __builtin_amdgcn_rcpf(fmaf(64 * 0.2333452377915607f, b, 1.0f));
    float r = SCALE * -0.067649900913238525f;
    r = fmaf(r, t, SCALE * 0.23002518713474274f);
    r = fmaf(r, t, SCALE * -0.17541733384132385f);
    r = fmaf(r, t, SCALE * 0.2041075974702835f);
    r = fmaf(r, t, SCALE * 0.023684635758399963f);
    r = fmaf(r, t, SCALE * 0.10058960318565369f);
    r = fmaf(r, t, SCALE * 0.091481544077396393f);
    r = fmaf(r, t, SCALE * 0.09317866712808609f);
    return r * t;
  } else if constexpr (DT == DIMQ_F16) {
    const float t = __builtin_amdgcn_rcpf(fmaf(64 * 0.36f, b, 1.0f));
    float r = SCALE * 0.04709881659085434f;
    r = fmaf(r, t, SCALE * -0.17988737532749394f);
    r = fmaf(r, t, SCALE * 0.18109358442700213f);
    r = fmaf(r, t, SCALE * 0.02646958676291894f);
    r = fmaf(r, t, SCALE * 0.13974328500731586f);
    r = fmaf(r, t, SCALE * 0.14176884610587542f);
    r = fmaf(r, t, SCALE * 0.14371325643352723f);
    return r * t;
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(64 * 0.31f, b, 1.0f));
    float r = SCALE * -0.0733089938090878f;
    r = fmaf(r, t, SCALE * 0.17872215085737886f);
    r = fmaf(r, t, SCALE * 0.017563094188134135f);
    r = fmaf(r, t, SCALE * 0.13253454642465368f);
    r = fmaf(r, t, SCALE * 0.1206456834055663f);
    r = fmaf(r, t, SCALE * 0.12384351893335482f);
    return r * t;
  }
}

// exp(-a^2 / 4), b = a / 64.  Products take it twice, so that they reach the subnormal numbers, which the exponential itself
// flushes.  For fp32 outputs the argument's roundings, 2^-24 of up to 150, are carried along and applied to first order;
// otherwise the tail is 1.5e-5 off where it is 1e-37.
template <int DT>
__device__ __forceinline__ float mx_exp_quarter(float b) {
  constexpr float kC = -0.36067376022224085f;  // -log2(e) / 4
  if constexpr (DT != DIMQ_F32) return __builtin_amdgcn_exp2f(b * b * (4096 * kC));
  constexpr float kLow = (float)(-0.36067376022224085187998 - (double)kC);
  const float a = b * 64, q = a * a, t = q * kC;
  const float low = fmaf(q, kLow, fmaf(fmaf(a, a, -q), kC, fmaf(q, kC, -t)));
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, low * 0.69314718055994531f, e);
}

template <int DT>
__device__ __forceinline__ float mx_gelu(float h) {
  const float b = mx_64ths(h), m = mx_tail_factor<DT, -64>(b), root = mx_exp_quarter<DT>(b);
  const float top = fmaf(0.5f, fabsf(h), 0.5f * h);  // max(h, 0) that keeps NaN; halves, as the sum of both would overflow
  return fmaf(b * m * root, root, top);
}

template <int DT>
__device__ __forceinline__ float mx_gelu_slope(float h) {
  const float b = mx_64ths(h), m = mx_tail_factor<DT>(b), c = h * 0.39894228040143268f;
  float tail, density;
  if constexpr (DT == DIMQ_F32) {
    const float root = mx_exp_quarter<DT>(b);
    tail = m * root * root, density = c * root * root;
  } else {
    const float e = __builtin_amdgcn_exp2f(b * b * (4096 * -0.72134752044448170f));  // flushed below 2^-126
    tail = m * e, density = c * e;
  }
  return density + (h < 0.0f ? tail : 1.0f - tail);
}

}  // namespace dimq
