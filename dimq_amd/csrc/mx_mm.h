// Shared parts of the microscaled products: arguments and epilogue.
#pragma once

#include "mx.h"

namespace dimq {

// act(acc + bias[n] + residual[m, n]) in fp32, rounded once to the output's type.
struct MxOut {
  void* y;
  int dtype;
  int64_t ld, cols;
  const void* bias;
  int bias_dtype;
  const void* res;  // y's shape
  int res_dtype;
  int act;
};

struct MxProduct {
  const uint8_t* xcodes;  // [M, xblocks, 16]
  const uint8_t* xscales;
  const uint8_t* wcodes;  // [N, blocks, 16]
  const uint8_t* wscales;
  int64_t M, N, blocks, xblocks;
  MxOut out;
};

// Outputs n .. n + 3 (n % 4 == 0) of row m from a lane's four accumulators.
__device__ __forceinline__ void mx_store4(const MxOut& o, int64_t m, int64_t n, f32x4 acc) {
  if (n >= o.cols) return;
  float v[4] = {acc[0], acc[1], acc[2], acc[3]};
  const int64_t at = m * o.ld + n;
  const int left = o.cols - n < 4 ? (int)(o.cols - n) : 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j < left) {
      if (o.bias) v[j] += load_as_float(o.bias, o.bias_dtype, n + j);
      if (o.res) v[j] += load_as_float(o.res, o.res_dtype, at + j);
    }
    if (o.act == DIMQ_ACT_RELU) v[j] = v[j] < 0.0f ? 0.0f : v[j];
    if (o.act == DIMQ_ACT_GELU) v[j] = mx_gelu<true>(v[j]);
  }
  if (left == 4 && o.ld % 4 == 0 && aligned(o.y, 16)) {
    if (o.dtype == DIMQ_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(o.y) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      const bool h = o.dtype == DIMQ_F16;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(o.y) + at) =
          h ? make_uint2(f16x2_rne(v[0], v[1]), f16x2_rne(v[2], v[3]))
            : make_uint2(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) store_from_float(o.y, o.dtype, at + j, v[j]);
}

}  // namespace dimq
