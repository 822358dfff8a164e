// Products of a gradient with a microscaled matrix (mx.h), out[p, k] = sum_r A[p, r] B[r, k]:
//   input gradient   A = g [M, N],           B = the 4-bit weights [N, K]
//   weight gradient  A = g [M, N] transposed, B = the 8-bit checkpoint [M, K]
// Codes times scales are exact in bf16, and so is a gradient of 16 or 32 bits as a sum of bf16 parts (one for bf16, two
// for fp16's 11 bits, three for fp32's 24), so that every product is exact and only the fp32 sums round.
#include "mx_mm.h"

namespace dimq {
namespace {

// x as NS bf16 parts that add up to it, by truncation (rounding could carry the first part to infinity); a NaN or an
// infinity is the first part alone.
template <int NS>
__device__ __forceinline__ void bf16_parts(float x, uint16_t (&h)[NS]) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) >= 0x7f800000u) {
    h[0] = (uint16_t)((u >> 16) | ((u & 0x7fffffffu) > 0x7f800000u ? 0x40u : 0u));
#pragma unroll
    for (int i = 1; i < NS; ++i) h[i] = 0;
    return;
  }
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const uint32_t t = __float_as_uint(x) & 0xffff0000u;
    h[i] = (uint16_t)(t >> 16);
    x -= __uint_as_float(t);
  }
}

struct GradArgs {
  const void* a;
  int64_t lda;
  const uint8_t* codes;  // [R, blocks, 16 or 32]
  const uint8_t* scales;
  int64_t P, R, K, blocks;
  MxOut out;
};

__device__ __forceinline__ uint32_t decode_one(const uint8_t* codes, int bits, int64_t block, int j, uint32_t byte) {
  if (bits == 4) {
    const uint32_t c = (codes[block * 16 + j / 2] >> (4 * (j & 1))) & 15u;
    const bf16x2 t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, mx_scale_operand(byte), 0);
    return __builtin_bit_cast(uint32_t, t) & 0xffffu;
  }
  return __float_as_uint((float)(int8_t)codes[block * 32 + j] * mx_step8(byte)) >> 16;
}

// Simple form: 64 x 64 outputs a work-group, 32 terms a step through the LDS, element by element.
template <int AT, bool TRANS, int BITS>
__global__ __launch_bounds__(256) void mx_grad_simple(GradArgs p) {
  constexpr int NS = AT == DIMQ_BF16 ? 1 : AT == DIMQ_F16 ? 2 : 3;
  __shared__ __align__(16) uint16_t As[NS][64][40], Bs[64][40];
  const int t = threadIdx.x, l = t & 63, w = t >> 6, c = l & 15, g = l >> 4;
  const int64_t p0 = (int64_t)blockIdx.x * 64, k0 = (int64_t)blockIdx.y * 64;
  f32x4 acc[4] = {};
  for (int64_t r0 = 0; r0 < p.R; r0 += 32) {
    __syncthreads();
    for (int e = t; e < 2048; e += 256) {
      const int i = TRANS ? e & 63 : e >> 5, j = TRANS ? e >> 6 : e & 31;
      const int64_t pp = p0 + i, r = r0 + j;
      uint16_t h[NS];
      const float v = pp < p.P && r < p.R ? load_as_float(p.a, AT, TRANS ? r * p.lda + pp : pp * p.lda + r) : 0.0f;
      bf16_parts<NS>(v, h);
#pragma unroll
      for (int s = 0; s < NS; ++s) As[s][i][j] = h[s];
      const int kk = e & 63, jj = e >> 6;
      const int64_t k = k0 + kk, rb = r0 + jj;
      uint32_t b = 0;
      if (k < p.K && rb < p.R) {
        const int64_t block = rb * p.blocks + k / 32;
        b = decode_one(p.codes, BITS, block, (int)(k & 31), p.scales[block]);
      }
      Bs[kk][jj] = (uint16_t)b;
    }
    __syncthreads();
    const bf16x8 bf = *reinterpret_cast<const bf16x8*>(&Bs[w * 16 + c][g * 8]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const bf16x8 af = *reinterpret_cast<const bf16x8*>(&As[s][i * 16 + c][g * 8]);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf, af, acc[i], 0, 0, 0);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = p0 + 16 * i + c;
    if (m < p.P) mx_store4(p.out, m, k0 + w * 16 + 4 * g, acc[i]);
  }
}

// Sums over the rows, one column a lane.
__global__ __launch_bounds__(64) void mx_row_sum_simple(const void* g, int dt, int64_t M, int64_t N, int64_t ld, void* out,
                                                        int odt) {
  const int64_t n = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (n >= N) return;
  float s[8] = {};
  for (int64_t m = 0; m < M; m += 8)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (m + i < M) s[i] += load_as_float(g, dt, (m + i) * ld + n);
  store_from_float(out, odt, n, ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])));
}

template <bool TRANS, int BITS>
int grad_any(int a_dtype, const GradArgs& p, hipStream_t s) {
  DIMQ_CHECK((p.K + 63) / 64 <= 65535, "mx gradient: too many columns");
  const dim3 grid((unsigned)((p.P + 63) / 64), (unsigned)((p.K + 63) / 64));
  switch (a_dtype) {
    case DIMQ_F32: mx_grad_simple<DIMQ_F32, TRANS, BITS><<<grid, 256, 0, s>>>(p); break;
    case DIMQ_F16: mx_grad_simple<DIMQ_F16, TRANS, BITS><<<grid, 256, 0, s>>>(p); break;
    default: mx_grad_simple<DIMQ_BF16, TRANS, BITS><<<grid, 256, 0, s>>>(p);
  }
  return check_launch("mx gradient");
}

int check_grad(const char* what, const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, const void* codes,
               const void* scales, int64_t K, const void* out, int out_dtype) {
  const int rc = mx_check_rows(what, g, g_dtype, M, N, ldg);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(out_dtype == DIMQ_F32 || out_dtype == DIMQ_F16 || out_dtype == DIMQ_BF16,
             "%s: output dtype must be fp32, fp16 or bf16", what);
  DIMQ_CHECK(K > 0 && N > 0, "linear dimensions must be positive");
  DIMQ_CHECK(M == 0 || (codes && scales), "%s: null pointer", what);
  DIMQ_CHECK(M == 0 || out, "%s: null pointer", what);
  DIMQ_CHECK(aligned(codes, 16), "%s: codes must be 16-byte aligned", what);
  return DIMQ_OK;
}

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_mx_grad_input_workspace_bytes(int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K) {
  return 0;
}

extern "C" int64_t dimq_mx_grad_weight_workspace_bytes(int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K) {
  return 0;
}

extern "C" int dimq_mxfp4_linear_grad_input(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg,
                                            const uint8_t* codes, const uint8_t* scales, int64_t K, void* gx,
                                            int gx_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_grad("mxfp4_linear_grad_input", g, g_dtype, M, N, ldg, codes, scales, K, gx, gx_dtype);
  if (rc != DIMQ_OK || M == 0) return rc;
  const GradArgs p{g, ldg, codes, scales, M, N, K, mx_blocks(K), MxOut{gx, gx_dtype, K, K, nullptr, 0, nullptr, 0, 0}};
  return grad_any<false, 4>(g_dtype, p, as_stream(stream));
}

extern "C" int dimq_mx_linear_grad_weight(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg,
                                          const int8_t* codes8, const uint8_t* scales8, int64_t K, void* gw, int gw_dtype,
                                          void* gb, int gb_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_grad("mx_linear_grad_weight", g, g_dtype, M, N, ldg, codes8, scales8, K, gw, gw_dtype);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(gw, "mx_linear_grad_weight: null pointer");
  DIMQ_CHECK(!gb || is_float_dtype(gb_dtype), "bias gradient must be floating point");
  const GradArgs p{g, ldg, reinterpret_cast<const uint8_t*>(codes8), scales8, N, M, K, mx_blocks(K),
                   MxOut{gw, gw_dtype, K, K, nullptr, 0, nullptr, 0, 0}};
  if (gb) {
    mx_row_sum_simple<<<dim3((unsigned)((N + 63) / 64)), 64, 0, as_stream(stream)>>>(g, g_dtype, M, N, ldg, gb, gb_dtype);
    const int e = check_launch("mx_linear_grad_weight");
    if (e != DIMQ_OK) return e;
  }
  return grad_any<true, 8>(g_dtype, p, as_stream(stream));
}
