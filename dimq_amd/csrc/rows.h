// Rows of a matrix in registers, for kernels that give T threads to a row: 8 elements a thread and chunk.
//
//   VEC 8  chunk c of thread t is elements 8 (t + T c) .. + 7, moved in 16-byte pieces (rows of a multiple of 8 elements,
//          16-byte aligned)
//   VEC 1  elements t + T (8 c + j), one at a time, for every other size and alignment
//
// Elements past the row re-read its first one and count as 0: no branch stands between the loads.
#pragma once

#include "common.h"

namespace dimq {

template <int T, int VEC>
__device__ __forceinline__ int row_at(int t, int c, int j) {
  return VEC == 8 ? 8 * (t + T * c) + j : t + T * (8 * c + j);
}

template <int XT, int T, int VEC>
__device__ __forceinline__ void row_load(const void* row, int t, int c, int D, float (&v)[8]) {
  if constexpr (VEC == 8) {
    const int at = 8 * (t + T * c);
    const bool in = at < D;
    if constexpr (XT == DIMQ_F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + (in ? at : 0));
      const float4 a = p[0], b = p[1];
      const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = in ? f[j] : 0.0f;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + (in ? at : 0));
      const uint32_t u[4] = {in ? a.x : 0, in ? a.y : 0, in ? a.z : 0, in ? a.w : 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = XT == DIMQ_F16 ? f16_bits_to_float(u[j] & 0xffffu) : bf16_bits_to_float(u[j] & 0xffffu);
        v[2 * j + 1] = XT == DIMQ_F16 ? f16_bits_to_float(u[j] >> 16) : bf16_bits_to_float(u[j] >> 16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = row_at<T, VEC>(t, c, j);
      const float f = load_as_float(row, XT, at < D ? at : 0);
      v[j] = at < D ? f : 0.0f;
    }
  }
}

// row_load of a dtype known at run time only (the same for the whole launch).
template <int T, int VEC>
__device__ __forceinline__ void row_load_dt(const void* row, int dt, int t, int c, int D, float (&v)[8]) {
  if (dt == DIMQ_F32) row_load<DIMQ_F32, T, VEC>(row, t, c, D, v);
  else if (dt == DIMQ_F16) row_load<DIMQ_F16, T, VEC>(row, t, c, D, v);
  else row_load<DIMQ_BF16, T, VEC>(row, t, c, D, v);
}

template <int XT, int T, int VEC>
__device__ __forceinline__ void row_store(void* row, int t, int c, int D, const float (&v)[8]) {
  if constexpr (VEC == 8) {
    const int at = 8 * (t + T * c);
    if (at >= D) return;
    if constexpr (XT == DIMQ_F32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(row) + at);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = XT == DIMQ_F16 ? f16x2_rne(v[2 * j], v[2 * j + 1]) : bf16x2_rne(v[2 * j], v[2 * j + 1]);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + at) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = row_at<T, VEC>(t, c, j);
      if (at < D) store_from_float(row, XT, at, v[j]);
    }
  }
}

template <int T, int VEC>
__device__ __forceinline__ void row_store_dt(void* row, int dt, int t, int c, int D, const float (&v)[8]) {
  if (dt == DIMQ_F32) row_store<DIMQ_F32, T, VEC>(row, t, c, D, v);
  else if (dt == DIMQ_F16) row_store<DIMQ_F16, T, VEC>(row, t, c, D, v);
  else row_store<DIMQ_BF16, T, VEC>(row, t, c, D, v);
}

// One element rounded to the dtype and back.
template <int XT>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (XT == DIMQ_F16) return f16_bits_to_float(float_to_f16_bits(v));
  else if constexpr (XT == DIMQ_BF16) return bf16_bits_to_float(float_to_bf16_bits(v));
  else return v;
}

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

// Over the T threads of a row, the same value for each of them; T = 64: a wave of its own, else the whole work-group.
// `red` (T / 64 floats) is free again after the next barrier.
template <int T, bool MAX = false>
__device__ __forceinline__ float row_reduce(float v, float* red) {
  v = MAX ? wave_max(v) : wave_add(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) v = MAX ? fmaxf(v, red[w]) : v + red[w];
  }
  return v;
}

}  // namespace dimq
