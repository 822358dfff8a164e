// y = act(Q4(x) W^T + bias + residual) on 4-bit microscaled weights (mx.h).  Two routes:
//
//   few rows    one launch: each work-group quantizes 16 rows of x on the way to 16 outputs, its waves share the reduction
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

// A block of x as it lies in memory, and how its loads are bounded: kWhole no bound, kGroups whole groups of 8 elements
// only (addresses past the row go to its start, their values to zero: loads stay free of branches, so that all of a turn's
// are in flight together), kAny element by element.
enum { kWhole, kGroups, kAny };
template <int XT>
struct RawBlock {
  static constexpr int N = XT == DIMQ_F32 ? 8 : 4;  // 16-byte pieces
  uint4 v[N];
};

template <int XT, int BOUND>
__device__ __forceinline__ void load_block(const void* x, int64_t at, int64_t c, int64_t cols, RawBlock<XT>& o) {
  constexpr int E = XT == DIMQ_F32 ? 4 : 8;  // elements a piece
  constexpr int SIZE = XT == DIMQ_F32 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < RawBlock<XT>::N; ++i) {
    const int64_t e = c + E * i;
    const char* p = static_cast<const char*>(x) + at * SIZE;
    if constexpr (BOUND != kAny) {
      o.v[i] = mx_read16(p + (BOUND == kWhole || e < cols ? e : 0) * SIZE);
    } else {
      o.v[i] = make_uint4(0, 0, 0, 0);
      if (e + E <= cols) {
        o.v[i] = mx_read16(p + e * SIZE);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          if (e + j >= cols) break;
          if constexpr (SIZE == 4) (&o.v[i].x)[j] = reinterpret_cast<const uint32_t*>(p)[e + j];
          else (&o.v[i].x)[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e + j] << (16 * (j & 1));
        }
      }
    }
  }
}

template <int XT>
__device__ __forceinline__ void clear_past_end(int64_t c, int64_t cols, RawBlock<XT>& o) {
  constexpr int E = XT == DIMQ_F32 ? 4 : 8;
#pragma unroll
  for (int i = 0; i < RawBlock<XT>::N; ++i)
    if (c + E * i >= cols) o.v[i] = make_uint4(0, 0, 0, 0);
}

// Its 4-bit codes and scale.  16-bit elements stay in pairs: integer maxima of their magnitudes and the conversions that
// take pairs, 50 instructions a block where fp32 copies take 150.
template <int XT>
__device__ __forceinline__ void quantize_block(const RawBlock<XT>& x, uint4& codes, uint32_t& byte) {
  uint32_t o[4];
  if constexpr (XT == DIMQ_F32) {
    float v[4][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w[4] = {x.v[i].x, x.v[i].y, x.v[i].z, x.v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i / 2][4 * (i & 1) + j] = __uint_as_float(w[j]);
        const uint32_t m = w[j] & 0x7fffffffu;
        top = top > m ? top : m;
      }
    }
    byte = mx_scale_byte<2>(top);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = mx_codes4(v[i], mx_scale_operand(byte));
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[4 * i] = x.v[i].x, w[4 * i + 1] = x.v[i].y, w[4 * i + 2] = x.v[i].z, w[4 * i + 3] = x.v[i].w;
    u16x2 top = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    const uint32_t m = top.x > top.y ? top.x : top.y;
    byte = mx_scale_byte<2>(XT == DIMQ_BF16 ? m << 16 : __float_as_uint(f16_bits_to_float(m)));
    const float s = mx_scale_operand(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t q = 0;
      mx_each<4>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        if constexpr (XT == DIMQ_BF16)
          q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[4 * i + j]), s, j);
        else
          q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[4 * i + j]), s, j);
      });
      o[i] = q;
    }
  }
  codes = byte == kMxNan ? make_uint4(0, 0, 0, 0) : make_uint4(o[0], o[1], o[2], o[3]);
}

// A turn of a wave: 16 blocks from b0, lane l the blocks b0 + 4 (l / 16) .. + 3 for row l % 16 of either operand.
template <int XT, int BOUND>
__device__ __forceinline__ void few_rows_turn(const FewArgs& p, const uint8_t* wrow, const uint8_t* srow, int64_t xat, bool row,
                                              int64_t b, f32x4& acc) {
  constexpr bool whole = BOUND == kWhole;
  uint4 w[4];
  uint32_t ws = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s) w[s] = *reinterpret_cast<const uint4*>(wrow + (whole || b + s < p.blocks ? b + s : 0) * 16);
  if (p.wide_scales) {  // blocks % 4 == 0
    ws = *reinterpret_cast<const uint32_t*>(srow + (whole || b < p.blocks ? b : 0));
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) ws |= (uint32_t)srow[whole || b + s < p.blocks ? b + s : 0] << (8 * s);
  }
  RawBlock<XT> raw[4] = {};
  if (row) {  // rows that are not there cost no loads
#pragma unroll
    for (int s = 0; s < 4; ++s) load_block<XT, BOUND>(p.x, xat, (b + s) * 32, p.K, raw[s]);
  }
  uint32_t xs = 0;
  uint4 x[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    if constexpr (BOUND == kGroups) clear_past_end<XT>((b + s) * 32, p.K, raw[s]);
    uint32_t byte;
    quantize_block<XT>(raw[s], x[s], byte);
    xs |= byte << (8 * s);
  }
  // past the weights' last block: codes of x are zero there, and so has to be the scale (another block's may be NaN)
  if constexpr (!whole) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (b + s >= p.blocks) ws &= ~(255u << (8 * s));
  }
  mx_each<4>([&](auto sc) {
    constexpr int s = decltype(sc)::value;
    const i32x8 u = {(int)w[s].x, (int)w[s].y, (int)w[s].z, (int)w[s].w, 0, 0, 0, 0};
    const i32x8 v = {(int)x[s].x, (int)x[s].y, (int)x[s].z, (int)x[s].w, 0, 0, 0, 0};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(u, v, acc, 4, 4, s, (int)ws, s, (int)xs);
  });
}

// A work-group owns 16 outputs of 16 rows; its waves take the reduction in turns of 16 blocks: 64 contiguous bytes of
// codes and one dword of scales a lane, whose bytes the four instructions select.  Bound by latency: with 8 waves a
// work-group the 8.4 MB of a 4096 x 4096 layer are requested by the first turn of 256 work-groups, 5.5 us for one row; with
// 16 rows, 7.8 us, also by the reads and the quantization of x, which every work-group does for itself (a launch of its own
// and the tiled product take 11.3).
template <int XT>
__global__ __launch_bounds__(512) void mx4_few_rows(const FewArgs p) {
  __shared__ f32x4 red[8 * 64];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1;
  const uint8_t* wrow = p.codes + n * p.blocks * 16;
  const uint8_t* srow = p.scales + n * p.blocks;
  const int64_t m = (int64_t)blockIdx.y * 16 + r;
  const bool row = m < p.M;
  const int64_t xat = (row ? m : 0) * p.ldx;
  f32x4 acc = {};
  for (int64_t b0 = wave * 16; b0 < p.blocks; b0 += waves * 16) {
    const int64_t b = b0 + 4 * g;
    if ((b0 + 16) * 32 <= p.K) few_rows_turn<XT, kWhole>(p, wrow, srow, xat, row, b, acc);
    else if (p.K % 8 == 0) few_rows_turn<XT, kGroups>(p, wrow, srow, xat, row, b, acc);
    else few_rows_turn<XT, kAny>(p, wrow, srow, xat, row, b, acc);
  }
  // the first wave adds up and stores: lane l the outputs n0 + 4 (l / 16) .. + 3 of row m
  const int64_t n4 = n0 + g * 4;
  const int left = p.N - n4 < 4 ? (int)(p.N - n4) : 4;
  float bias[4] = {}, res[4] = {};
  if (wave == 0 && row) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (p.out.bias && j < left) bias[j] = load_as_float(p.out.bias, p.out.bias_dtype, n4 + j);
      if (p.out.res && j < left) res[j] = load_as_float(p.out.res, p.out.res_dtype, m * p.out.ld + n4 + j);
    }
  }
  red[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave != 0 || !row) return;
  for (int w = 1; w < waves; ++w) acc += red[w * 64 + lane];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float t = acc[j] + bias[j] + res[j];
    if (p.out.act == DIMQ_ACT_RELU) t = t < 0.0f ? 0.0f : t;
    if (p.out.act == DIMQ_ACT_GELU) t = mx_gelu<DIMQ_F32>(t);
    if (j < left) store_from_float(p.out.y, p.out.dtype, m * p.out.ld + n4 + j, t);
  }
}

template <int XT>
void few_rows(const FewArgs& p, hipStream_t s) {
  const int64_t turns = (p.blocks + 15) / 16;
  int waves = 1;
  while (waves < 8 && waves < turns) waves *= 2;
  mx4_few_rows<XT><<<dim3((unsigned)((p.N + 15) / 16), (unsigned)((p.M + 15) / 16)), 64 * waves, 0, s>>>(p);
}

int few_rows_any(int x_dtype, const FewArgs& p, hipStream_t s) {
  switch (x_dtype) {
    case DIMQ_F32: few_rows<DIMQ_F32>(p, s); break;
    case DIMQ_F16: few_rows<DIMQ_F16>(p, s); break;
    default: few_rows<DIMQ_BF16>(p, s);
  }
  return check_launch("mxfp4_linear");
}

// Whether the one launch is the faster route.  It takes 3.6 us and, for each 4,096 of K and each work-group of a CU, 2.3 us
// and 0.17 a row (fp32 x: 4.0, 2.8 and 0.31); the other route 5 us for its launches and the tiled product.  Measured with
// 16-bit x up to 256 rows, one launch / other route: 768 -> 768 with 64 rows 5.0 us / 7.3, with 256 7.5 / 7.6; 768 -> 2304 with
// 96 8.5 / 7.4; 4096 -> 4096 with 16 8.4 / 11.3, with 32 13.9 / 12.0; 8192 -> 8192 with 1 14.3 / 16.3, with 16 24.4 / 16.7.
bool few_rows_pay(bool f32, int64_t M, int64_t K, int64_t N) {
  if (M > 256) return false;
  const int64_t groups = (N + 15) / 16 * ((M + 15) / 16), rows = M < 16 ? M : 16;
  const double units = K / 4096.0 * (double)((groups + 255) / 256);
  const double us = f32 ? 4.0 + units * (2.8 + 0.31 * rows) : 3.6 + units * (2.3 + 0.17 * rows);
  return us <= 5.0 + mx_plan(true, M, N, (mx_blocks(K) + 7) / 8).us;
}

// Workspace: x's codes and scales, the weights' scales, the slices of a split reduction.
struct Layout {
  int64_t xc = 0, xs = 0, ws = 0, part = 0, bytes = 0;
  MxPlan plan;
  Layout(int64_t M, int64_t K, int64_t N) {
    const int64_t n = mx_blocks(K), b = mx_pad8(n);
    auto take = [&](int64_t& at, int64_t n) { at = bytes, bytes += (n + 255) / 256 * 256; };
    plan = mx_plan(true, M, N, b / 8);
    take(xc, M * n * 16);
    take(xs, mx_scale_rows(M) * b);
    take(ws, mx_scale_rows(N) * b);
    take(part, mx_partial_bytes(plan, M, N));
  }
};

}  // namespace

int mx_forward_route(bool f32, int64_t M, int64_t K, int64_t N) {
  const int64_t stages = (mx_blocks(K) + 7) / 8;
  return few_rows_pay(f32, M, K, N) ? 0 : mx_route(mx_plan(true, M, N, stages), M, N, stages);
}

}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0 || (few_rows_pay(false, M, K, N) && few_rows_pay(true, M, K, N))) return 0;
  return Layout(M, K, N).bytes;
}

namespace dimq {
namespace {

// The layer on packed weights or, where w is given, on weights that are packed into codes and scales on the way.
struct Layer {
  const char* what;
  const void* x;
  int x_dtype;
  int64_t M, K, ldx;
  const void* w;
  int w_dtype;
  int64_t ldw;
  uint8_t *codes, *scales;
  int64_t N;
  int8_t* codes8;
  uint8_t* scales8;
  MxOut out;
  void* workspace;
  int64_t workspace_bytes;
};

int run(const Layer& a, hipStream_t s) {
  const char* what = a.what;
  DIMQ_CHECK(a.M >= 0 && a.K > 0 && a.N > 0, "linear dimensions must be positive");
  DIMQ_CHECK(a.out.act >= DIMQ_ACT_NONE && a.out.act <= DIMQ_ACT_GELU, "unknown activation %d", a.out.act);
  DIMQ_CHECK(a.out.dtype == DIMQ_F32 || a.out.dtype == DIMQ_F16 || a.out.dtype == DIMQ_BF16,
             "output dtype must be fp32, fp16 or bf16");
  DIMQ_CHECK(!a.out.bias || is_float_dtype(a.out.bias_dtype), "bias must be floating point");
  DIMQ_CHECK(!a.out.res || is_float_dtype(a.out.res_dtype), "residual must be floating point");
  int rc = mx_check_rows(what, a.x, a.x_dtype, a.M, a.K, a.ldx);
  if (rc != DIMQ_OK || (a.M == 0 && !a.w)) return rc;
  DIMQ_CHECK(a.codes && a.scales, "%s: null pointer", what);
  DIMQ_CHECK(aligned(a.codes, 16), "%s: codes must be 16-byte aligned", what);
  if (a.w && (rc = mx_check_rows(what, a.w, a.w_dtype, a.N, a.K, a.ldw)) != DIMQ_OK) return rc;
  const int64_t blocks = mx_blocks(a.K);
  if (a.M == 0) return dimq_mx_quantize(a.w, a.w_dtype, a.N, a.K, a.ldw, a.codes, a.scales, blocks, nullptr, nullptr, s);
  DIMQ_CHECK(a.out.y, "%s: null pointer", what);
  if (a.codes8) {
    DIMQ_CHECK(a.scales8, "%s: null pointer", what);
    DIMQ_CHECK(aligned(a.codes8, 16), "%s: codes must be 16-byte aligned", what);
  }
  if (few_rows_pay(a.x_dtype == DIMQ_F32, a.M, a.K, a.N)) {
    if (a.w) rc = dimq_mx_quantize(a.w, a.w_dtype, a.N, a.K, a.ldw, a.codes, a.scales, blocks, nullptr, nullptr, s);
    if (rc == DIMQ_OK && a.codes8)
      rc = dimq_mx_quantize(a.x, a.x_dtype, a.M, a.K, a.ldx, nullptr, nullptr, 0, a.codes8, a.scales8, s);
    if (rc != DIMQ_OK) return rc;
    DIMQ_CHECK((a.N + 15) / 16 < (1ll << 31), "%s: too many outputs", what);
    return few_rows_any(a.x_dtype, {a.x, a.ldx, a.M, a.K, a.codes, a.scales, a.N, blocks,
                                    blocks % 4 == 0 && aligned(a.scales, 4), a.out}, s);
  }
  DIMQ_CHECK(a.M <= kMxMaxRows && a.N <= kMxMaxRows, "%s: too large", what);
  const Layout at(a.M, a.K, a.N);
  DIMQ_CHECK(a.workspace && aligned(a.workspace, 256) && a.workspace_bytes >= at.bytes,
             "%s: the workspace is too small or not 256-byte aligned", what);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  const int64_t xr = mx_scale_rows(a.M), wr = mx_scale_rows(a.N);
  const MxTiledOperand x{a.x, a.x_dtype, a.M, a.K, a.ldx, ws + at.xc, ws + at.xs, xr, nullptr, a.codes8, a.scales8};
  if (a.w) {
    rc = mx_quantize_pair(x, {a.w, a.w_dtype, a.N, a.K, a.ldw, a.codes, ws + at.ws, wr, a.scales, nullptr, nullptr}, s);
  } else {
    MxScaleTurn turn;
    turn.in = a.scales, turn.out = ws + at.ws, turn.n = a.N, turn.blocks = blocks, turn.rows = wr;
    rc = mx_quantize_tiled(x, turn, s);
  }
  if (rc != DIMQ_OK) return rc;
  const MxMm p{{ws + at.xc, blocks * 16, ws + at.xs, xr}, {a.codes, blocks * 16, ws + at.ws, wr},
               a.M, a.N, blocks, 1, 0, 0, a.out};
  return mx_mm<true, false, false>(p, at.plan, reinterpret_cast<float*>(ws + at.part), s, what);
}

}  // namespace
}  // namespace dimq

extern "C" int dimq_mxfp4_linear(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* codes,
                                 const uint8_t* scales, const void* bias, int bias_dtype, int64_t N, void* y, int y_dtype,
                                 const void* residual, int residual_dtype, int activation, int8_t* codes8,
                                 uint8_t* scales8, void* workspace, int64_t workspace_bytes, void* stream) {
  return run({"mxfp4_linear", x, x_dtype, M, K, ldx, nullptr, 0, 0, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scales), N,
              codes8, scales8, MxOut{y, y_dtype, N, N, bias, bias_dtype, residual, residual_dtype, activation}, workspace,
              workspace_bytes}, as_stream(stream));
}

extern "C" int dimq_mx_linear_forward(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const void* w, int w_dtype,
                                      int64_t ldw, const void* bias, int bias_dtype, int64_t N, void* y, int y_dtype,
                                      uint8_t* codes, uint8_t* scales, int8_t* codes8, uint8_t* scales8, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  DIMQ_CHECK(w, "mx_linear_forward: null pointer");
  return run({"mx_linear_forward", x, x_dtype, M, K, ldx, w, w_dtype, ldw, codes, scales, N, codes8, scales8,
              MxOut{y, y_dtype, N, N, bias, bias_dtype, nullptr, 0, 0}, workspace, workspace_bytes}, as_stream(stream));
}
