// y = act(Q4(x) W^T + bias + residual) on 4-bit microscaled weights (mx.h): x is quantized on the way in, the products
// run on the scaled matrix instructions, whose operand of 32 codes a lane is one block and takes that block's scale.
#include "mx_mm.h"

namespace dimq {
namespace {

// Simple form: a wave owns 16 outputs of 64 rows and reads its operands from memory; lane l holds the blocks l / 16 of a
// step's four for row l % 16, the weights as the first operand, so that a lane ends with four neighbouring outputs.
__global__ __launch_bounds__(256) void mx4_gemm_simple(MxProduct p) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, r = l & 15, g = l >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 64 + w * 16, m0 = (int64_t)blockIdx.y * 64;
  if (n0 >= p.N) return;
  const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1;
  f32x4 acc[4] = {};
  for (int64_t b0 = 0; b0 < p.blocks; b0 += 4) {
    const int64_t b = b0 + g;
    i32x8 wf = {};
    int ws = 0;
    if (b < p.blocks) {
      const int4 t = *reinterpret_cast<const int4*>(p.wcodes + (n * p.blocks + b) * 16);
      wf = i32x8{t.x, t.y, t.z, t.w, 0, 0, 0, 0};
      ws = p.wscales[n * p.blocks + b];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + 16 * i + r < p.M ? m0 + 16 * i + r : p.M - 1;
      i32x8 xf = {};
      int xs = 0;
      if (b < p.blocks) {
        const int4 t = *reinterpret_cast<const int4*>(p.xcodes + (m * p.xblocks + b) * 16);
        xf = i32x8{t.x, t.y, t.z, t.w, 0, 0, 0, 0};
        xs = p.xscales[m * p.xblocks + b];
      }
      acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[i], 4, 4, 0, ws, 0, xs);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + 16 * i + r;
    if (m < p.M) mx_store4(p.out, m, n0 + 4 * g, acc[i]);
  }
}

// Workspace: x's codes and scales, its rows padded to whole steps of four blocks.
int64_t x_blocks(int64_t K) { return (mx_blocks(K) + 3) / 4 * 4; }
int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  return pad256(M * x_blocks(K) * 16) + pad256(M * x_blocks(K));
}

extern "C" int dimq_mxfp4_linear(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* codes,
                                 const uint8_t* scales, const void* bias, int bias_dtype, int64_t N, void* y, int y_dtype,
                                 const void* residual, int residual_dtype, int activation, int8_t* codes8,
                                 uint8_t* scales8, void* workspace, int64_t workspace_bytes, void* stream) {
  DIMQ_CHECK(M >= 0 && K > 0 && N > 0, "linear dimensions must be positive");
  DIMQ_CHECK(activation >= DIMQ_ACT_NONE && activation <= DIMQ_ACT_GELU, "unknown activation %d", activation);
  DIMQ_CHECK(y_dtype == DIMQ_F32 || y_dtype == DIMQ_F16 || y_dtype == DIMQ_BF16, "output dtype must be fp32, fp16 or bf16");
  DIMQ_CHECK(!bias || is_float_dtype(bias_dtype), "bias must be floating point");
  DIMQ_CHECK(!residual || is_float_dtype(residual_dtype), "residual must be floating point");
  int rc = mx_check_rows("mxfp4_linear", x, x_dtype, M, K, ldx);
  if (rc != DIMQ_OK || M == 0) return rc;
  DIMQ_CHECK(codes && scales && y, "mxfp4_linear: null pointer");
  DIMQ_CHECK(aligned(codes, 16), "mxfp4_linear: codes must be 16-byte aligned");
  DIMQ_CHECK(workspace && aligned(workspace, 256) && workspace_bytes >= dimq_mxfp4_linear_workspace_bytes(M, K, N),
             "mxfp4_linear: the workspace is too small or not 256-byte aligned");
  uint8_t* xc = static_cast<uint8_t*>(workspace);
  uint8_t* xs = xc + pad256(M * x_blocks(K) * 16);
  rc = dimq_mx_quantize(x, x_dtype, M, K, ldx, xc, xs, x_blocks(K), codes8, scales8, stream);
  if (rc != DIMQ_OK) return rc;
  const MxProduct p{xc, xs, codes, scales, M, N, mx_blocks(K), x_blocks(K),
                    MxOut{y, y_dtype, N, N, bias, bias_dtype, residual, residual_dtype, activation}};
  DIMQ_CHECK((M + 63) / 64 <= 65535 && (N + 63) / 64 < (1ll << 31), "mxfp4_linear: too many rows");
  mx4_gemm_simple<<<dim3((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64)), 256, 0, as_stream(stream)>>>(p);
  return check_launch("mxfp4_linear");
}
