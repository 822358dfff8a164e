// Rows of elements eight at a time, shared by the quantizing kernels.
#pragma once

#include "mx.h"

namespace dimq {

// Sixteen bytes at an address that is a multiple of the element's size (the memory pipeline takes any).
__device__ __forceinline__ uint4 mx_read16(const void* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ void mx_write16(void* p, uint4 v) { __builtin_memcpy(p, &v, 16); }

// Elements c .. c + 7 of a row of `cols` as fp32, zeros past its end.
template <int DT>
__device__ __forceinline__ void mx_load_row8(const void* x, int64_t at, int64_t c, int64_t cols, float (&v)[8]) {
  if (c + 8 <= cols) {
    if constexpr (DT == DIMQ_F32) {
      const float* p = static_cast<const float*>(x) + at + c;
      const uint4 a = mx_read16(p), b = mx_read16(p + 4);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else {
      const uint4 a = mx_read16(static_cast<const uint16_t*>(x) + at + c);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = DT == DIMQ_F16 ? f16_bits_to_float(w[j] & 0xffffu) : bf16_bits_to_float(w[j] & 0xffffu);
        v[2 * j + 1] = DT == DIMQ_F16 ? f16_bits_to_float(w[j] >> 16) : bf16_bits_to_float(w[j] >> 16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? load_as_float(x, DT, at + c + j) : 0.0f;
  }
}

template <int DT>
__device__ __forceinline__ void mx_store_row8(void* y, int64_t at, int64_t c, int64_t cols, const float (&v)[8]) {
  if (c + 8 <= cols) {
    if constexpr (DT == DIMQ_F32) {
      float* p = static_cast<float*>(y) + at + c;
      mx_write16(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
      mx_write16(p + 4, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = DT == DIMQ_F16 ? f16x2_rne(v[2 * j], v[2 * j + 1]) : bf16x2_rne(v[2 * j], v[2 * j + 1]);
      mx_write16(static_cast<uint16_t*>(y) + at + c, make_uint4(w[0], w[1], w[2], w[3]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) store_from_float(y, DT, at + c + j, v[j]);
  }
}

// Eight codes of `BITS` (4: one dword, 8: two) -> values.
template <int BITS>
__device__ __forceinline__ void mx_decode8(const void* codes, uint32_t byte, int64_t unit, float (&v)[8]) {
  if constexpr (BITS == 4) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const uint32_t w = static_cast<const uint32_t*>(codes)[unit];
    const float s = mx_scale_operand(byte);
    const f2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
    const f2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
    v[0] = p0.x; v[1] = p0.y; v[2] = p1.x; v[3] = p1.y;
    v[4] = p2.x; v[5] = p2.y; v[6] = p3.x; v[7] = p3.y;
  } else {
    const uint2 w = static_cast<const uint2*>(codes)[unit];
    const float s = mx_step8(byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * s;
  }
}

// Whether rows of cols elements, ld apart, are 16-byte aligned and whole groups of 8.
inline bool mx_vec_rows(const void* p, int dt, int64_t cols, int64_t ld) {
  return aligned(p, 16) && cols % 8 == 0 && (ld * dtype_size(dt)) % 16 == 0;
}

// Scales [n, blocks] to bring into the order of the tiled products, [stages of 8 blocks, rows, 8].
struct MxScaleTurn {
  const uint8_t* in = nullptr;
  uint8_t* out = nullptr;
  int64_t n = 0, blocks = 0, rows = 0, stages = 0;
  uint32_t groups = 0;  // work-groups that do it
};

// A tensor [rows, cols] to become an operand of the tiled products: codes [rows, blocks, 16] and scales [stages of 8
// blocks, scale_rows, 8], zeros past the row; its row-major scales and its 8-bit form where those are given.
struct MxTiledOperand {
  const void* x;
  int dtype;
  int64_t rows, cols, ld;
  uint8_t *codes, *tiled;
  int64_t scale_rows;
  uint8_t* scales;
  int8_t* codes8;
  uint8_t* scales8;
};

// In one launch (mx_quant.hip): x, and packed weights' scales turned; x and weights.
int mx_quantize_tiled(const MxTiledOperand& x, MxScaleTurn turn, hipStream_t s);
int mx_quantize_pair(const MxTiledOperand& x, const MxTiledOperand& w, hipStream_t s);

// dimq_mx_linear_route of the forward product (mx_gemm.hip).
int mx_forward_route(bool f32, int64_t M, int64_t K, int64_t N);

}  // namespace dimq
