// y = act(Q4(x) W^T + bias + residual) on 4-bit microscaled weights (mx.h).  Two routes:
//
//   few rows    one launch: each work-group quantizes x on the way to its 16 outputs, its waves share the reduction
//   otherwise   x is quantized into the workspace, then the tiled product (mx_mm.h) runs on both operands' codes
//
// Both run on the scaled matrix instructions, whose operand of 32 codes a lane is one block and takes that block's scale.
#include "mx_mm.h"
#include "mx_quant.h"

namespace dimq {
namespace {

struct FewArgs {
  const void* x;
  int64_t ldx, M, K;
  const uint8_t* codes;   // [N, blocks, 16]
  const uint8_t* scales;  // [N, blocks]
  int64_t N, blocks;
  bool wide_scales;       // four scales can be read at once
  MxOut out;
};

// The lane's block of x in 4 bits: 32 elements from column c of a row.  16-bit elements stay in pairs: integer maxima of
// their magnitudes and the conversions that take pairs, 50 instructions a block where fp32 copies take 150, which is what
// the kernel spends its time on from 8 rows on (16 x 4096 -> 4096: 13.3 us with copies).
template <int XT>
__device__ __forceinline__ void quantize_block(const void* x, int64_t at, int64_t c, int64_t cols, uint4& codes, uint32_t& byte) {
  if constexpr (XT != DIMQ_F32) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* p = static_cast<const uint16_t*>(x) + at + c + 8 * i;
      uint4 t = make_uint4(0, 0, 0, 0);
      if (c + 8 * i + 8 <= cols) {
        t = mx_read16(p);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + 8 * i + j < cols) (&t.x)[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
      }
      w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
    }
    u16x2 top = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    const uint32_t m = top.x > top.y ? top.x : top.y;
    byte = mx_scale_byte<2>(XT == DIMQ_BF16 ? m << 16 : __float_as_uint(f16_bits_to_float(m)));
    const float s = mx_scale_operand(byte);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t q = 0;
      mx_each<4>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        if constexpr (XT == DIMQ_BF16) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[4 * i + j]), s, j);
        else q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[4 * i + j]), s, j);
      });
      o[i] = byte == kMxNan ? 0u : q;
    }
    codes = make_uint4(o[0], o[1], o[2], o[3]);
    return;
  }
  float v[4][8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mx_load_row8<XT>(x, at, c + 8 * i, cols, v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t m = __float_as_uint(v[i][j]) & 0x7fffffffu;
      top = top > m ? top : m;
    }
  }
  byte = mx_scale_byte<2>(top);
  const float s = mx_scale_operand(byte);
  codes = make_uint4(mx_codes4(v[0], s), mx_codes4(v[1], s), mx_codes4(v[2], s), mx_codes4(v[3], s));
  if (byte == kMxNan) codes = make_uint4(0, 0, 0, 0);
}

// Up to 16 MT rows.  A work-group owns 16 outputs; its waves take the reduction in turns of 16 blocks, lane l the blocks
// 4 (l / 16) .. + 3 of a turn for row l % 16 of either operand: 64 contiguous bytes of codes and one dword of scales,
// whose bytes the four instructions select.  Bound by latency: all of a turn's loads are in flight at once, and with 16
// outputs and 8 waves a work-group the 8.4 MB of a 4096 x 4096 layer are requested by the first turn of 256 work-groups.
template <int XT, int MT>
__global__ __launch_bounds__(512) void mx4_few_rows(const FewArgs p) {
  __shared__ f32x4 red[8 * MT * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1;
  const uint8_t* wrow = p.codes + n * p.blocks * 16;
  const uint8_t* srow = p.scales + n * p.blocks;
  f32x4 acc[MT] = {};
  for (int64_t b0 = wave * 16; b0 < p.blocks; b0 += waves * 16) {
    const int64_t b = b0 + 4 * g;
    uint4 w[4];
    uint32_t ws = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      w[s] = b + s < p.blocks ? *reinterpret_cast<const uint4*>(wrow + (b + s) * 16) : make_uint4(0, 0, 0, 0);
    if (p.wide_scales) {
      if (b < p.blocks) ws = *reinterpret_cast<const uint32_t*>(srow + b);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (b + s < p.blocks) ws |= (uint32_t)srow[b + s] << (8 * s);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int64_t m = 16 * t + r < p.M ? 16 * t + r : p.M - 1;
      uint4 x[4];
      uint32_t xs = 0;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint32_t byte;
        quantize_block<XT>(p.x, m * p.ldx, (b + s) * 32, p.K, x[s], byte);
        xs |= byte << (8 * s);
      }
      mx_each<4>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        const i32x8 a = {(int)w[s].x, (int)w[s].y, (int)w[s].z, (int)w[s].w, 0, 0, 0, 0};
        const i32x8 c = {(int)x[s].x, (int)x[s].y, (int)x[s].z, (int)x[s].w, 0, 0, 0, 0};
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, c, acc[t], 4, 4, s, (int)ws, s, (int)xs);
      });
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) red[(wave * MT + t) * 64 + lane] = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 64; i += blockDim.x) {
    f32x4 sum = red[i];
    for (int w = 1; w < waves; ++w) sum += red[w * MT * 64 + i];
    const int64_t m = i / 64 * 16 + (i & 15), n4 = n0 + ((i >> 4) & 3) * 4;
    if (m < p.M) mx_store4(p.out, m, n4, sum);
  }
}

template <int XT>
void few_rows(const FewArgs& p, hipStream_t s) {
  const int64_t turns = (p.blocks + 15) / 16;
  int waves = 1;
  while (waves < 8 && waves < turns) waves *= 2;
  const dim3 grid((unsigned)((p.N + 15) / 16));
  if (p.M <= 16) mx4_few_rows<XT, 1><<<grid, 64 * waves, 0, s>>>(p);
  else if (p.M <= 32) mx4_few_rows<XT, 2><<<grid, 64 * waves, 0, s>>>(p);
  else mx4_few_rows<XT, 4><<<grid, 64 * waves, 0, s>>>(p);
}

int few_rows_any(int x_dtype, const FewArgs& p, hipStream_t s) {
  switch (x_dtype) {
    case DIMQ_F32: few_rows<DIMQ_F32>(p, s); break;
    case DIMQ_F16: few_rows<DIMQ_F16>(p, s); break;
    default: few_rows<DIMQ_BF16>(p, s);
  }
  return check_launch("mxfp4_linear");
}

// Rows up to which the one launch is taken.
constexpr int64_t kFewRows = 16;

// Workspace: x's codes and scales, the weights' scales, the slices of a split reduction.
struct Layout {
  int64_t xc = 0, xs = 0, ws = 0, part = 0, bytes = 0;
  MxPlan plan;
  Layout(int64_t M, int64_t K, int64_t N) {
    const int64_t b = mx_pad8(mx_blocks(K));
    auto take = [&](int64_t& at, int64_t n) { at = bytes, bytes += (n + 255) / 256 * 256; };
    plan = mx_plan(true, M, N, b / 8);
    take(xc, M * b * 16);
    take(xs, mx_scale_rows(M) * b);
    take(ws, mx_scale_rows(N) * b);
    take(part, mx_partial_bytes(plan, M, N));
  }
};

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  return Layout(M, K, N).bytes;
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
  if (codes8) {
    DIMQ_CHECK(scales8, "mxfp4_linear: null pointer");
    DIMQ_CHECK(aligned(codes8, 16), "mxfp4_linear: codes must be 16-byte aligned");
  }
  const int64_t blocks = mx_blocks(K), pitch = mx_pad8(blocks);
  hipStream_t s = as_stream(stream);
  const MxOut out{y, y_dtype, N, N, bias, bias_dtype, residual, residual_dtype, activation};
  if (M <= kFewRows && !codes8) {
    DIMQ_CHECK((N + 15) / 16 < (1ll << 31), "mxfp4_linear: too many outputs");
    return few_rows_any(x_dtype, {x, ldx, M, K, codes, scales, N, blocks, blocks % 4 == 0 && aligned(scales, 4), out}, s);
  }
  const Layout at(M, K, N);
  DIMQ_CHECK(workspace && aligned(workspace, 256) && workspace_bytes >= at.bytes,
             "mxfp4_linear: the workspace is too small or not 256-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MxScaleTurn turn;
  turn.in = scales, turn.out = ws + at.ws, turn.n = N, turn.blocks = blocks, turn.rows = mx_scale_rows(N);
  rc = mx_quantize_tiled(x, x_dtype, M, K, ldx, ws + at.xc, ws + at.xs, pitch, mx_scale_rows(M), codes8, scales8, turn, s);
  if (rc != DIMQ_OK) return rc;
  const MxMm p{{ws + at.xc, pitch * 16, ws + at.xs, mx_scale_rows(M)}, {codes, blocks * 16, ws + at.ws, mx_scale_rows(N)},
               M, N, blocks, 1, 0, 0, out};
  return mx_mm<true, false, false>(p, at.plan, reinterpret_cast<float*>(ws + at.part), s, "mxfp4_linear");
}
