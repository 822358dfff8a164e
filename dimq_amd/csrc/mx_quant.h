// Rows of elements eight at a time, shared by the quantizing kernels.
#pragma once

#include "mx.h"

namespace dimq {

// Elements c .. c + 7 of a row of `cols` as fp32, zeros past its end.  VEC: the row is 16-byte aligned and cols % 8 == 0.
template <int DT, bool VEC>
__device__ __forceinline__ void mx_load_row8(const void* x, int64_t at, int64_t c, int64_t cols, float (&v)[8]) {
  if constexpr (VEC) {
    if (c >= cols) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    } else if constexpr (DT == DIMQ_F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at + c);
      const float4 a = p[0], b = p[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at + c);
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

template <int DT, bool VEC>
__device__ __forceinline__ void mx_store_row8(void* y, int64_t at, int64_t c, int64_t cols, const float (&v)[8]) {
  if constexpr (VEC) {
    if (c >= cols) return;
    if constexpr (DT == DIMQ_F32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(y) + at + c);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = DT == DIMQ_F16 ? f16x2_rne(v[2 * j], v[2 * j + 1]) : bf16x2_rne(v[2 * j], v[2 * j + 1]);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + at + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) store_from_float(y, DT, at + c + j, v[j]);
  }
}

// Whether rows of cols elements, ld apart, can be read (written) 16 bytes at a time.
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

// x in 4 bits as an operand of the tiled products: codes [rows, blocks, 16] and scales [blocks / 8, scale_rows, 8]
// (blocks % 8 == 0, zeros past the row), its 8-bit form where codes8 is given, and the other operand's scales turned, in
// one launch (mx_quant.hip).
int mx_quantize_tiled(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes, uint8_t* scales,
                      int64_t blocks, int64_t scale_rows, int8_t* codes8, uint8_t* scales8, MxScaleTurn turn, hipStream_t s);

}  // namespace dimq
