// Microscaled formats (mx.h): quantization to 4 and 8 bits, the way back, and GELU with its input kept in 8 bits.
#include "mx_quant.h"

namespace dimq {
namespace {

// n / d for n < 2^31 as (n * mul) >> shift: mul = ceil(2^(31 + s) / d), s = ceil(log2 d), is above the quotient by less
// than 2^-(31 + s) of it, which times n stays below 1 / d.
struct FastDiv {
  uint32_t mul = 0, shift = 0, d = 1;
  explicit FastDiv(uint32_t div) : d(div) {
    uint32_t s = 0;
    while ((1ull << s) < div) ++s;
    shift = 31 + s;
    mul = (uint32_t)(((1ull << shift) + div - 1) / div);
  }
  __device__ __forceinline__ uint32_t quot(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> shift); }
};

// Largest magnitude of a block's four lanes, as fp32 bits: integer order is the magnitudes' order, NaN above all.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true);  // lanes 1 0 3 2
  m = m > a ? m : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true);  // lanes 2 3 0 1
  return m > b ? m : b;
}

// Eight fp32 values -> 8-bit codes in two dwords: v 2^(133 - byte) is exact or, below any rounding step, flushed;
// clamped first (127.5 and more would round to 128), then rounded to nearest even by adding 1.5 * 2^23.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], uint32_t byte) {
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = __builtin_amdgcn_fmed3f(ldexpf(v[j], 133 - (int)byte), -127.0f, 127.0f);
    b[j] = __float_as_uint(t + 12582912.0f);
  }
  uint2 w;
  w.x = perm(perm(b[3], b[2], 0x00000400u), perm(b[1], b[0], 0x00000400u), 0x05040100u);
  w.y = perm(perm(b[7], b[6], 0x00000400u), perm(b[5], b[4], 0x00000400u), 0x05040100u);
  return w;
}

struct QuantArgs {
  const void* x;
  int64_t ldx, rows, cols;
  uint8_t* codes4;   // rows of blocks4 * 16 bytes
  uint8_t* scales4;
  int8_t* codes8;    // rows of blocks8 * 32 bytes
  uint8_t* scales8;
  int64_t blocks, blocks4, blocks8;  // blocks of a row in all (the padded ones are zeros), in the 4- and the 8-bit output
  void* y = nullptr;                 // GELU's output rows of cols
  uint8_t* tiled = nullptr;          // the 4-bit scales as [stages of 8 blocks, scale_rows, 8] (mx_mm.h)
  int64_t scale_rows = 0, row0 = 0;  // this launch's rows from row0
};

// Eight scales of a row a thread, zeros past the row's end.
__device__ __forceinline__ void turn_scales(const MxScaleTurn& t, uint32_t group) {
  const int64_t i = (int64_t)group * 256 + threadIdx.x;
  if (i >= t.stages * t.n) return;
  const int64_t stage = i / t.n, row = i - stage * t.n;
  const uint8_t* src = t.in + row * t.blocks + stage * 8;
  uint2 w = make_uint2(0, 0);
  if (t.blocks % 8 == 0 && aligned(t.in, 8)) {
    w = *reinterpret_cast<const uint2*>(src);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (stage * 8 + j < t.blocks) (j < 4 ? w.x : w.y) |= (uint32_t)src[j] << (8 * (j & 3));
  }
  *reinterpret_cast<uint2*>(t.out + (stage * t.rows + row) * 8) = w;
}

// A lane takes eight elements, four lanes a block: loads of 16 bytes and stores of 4, 8 and 16 next to one another
// across the wave, the block's maximum by two lane exchanges.  Bound by the bytes: 4096 x 4096 fp32 to both formats
// moves 67 MB in and 26 MB out, 15.9 to 16.3 us or 5.8 TB/s.
// TILED: the 4-bit output is a tiled product's operand; its scales go there in that order, to scales4 where that is given.
template <int XT, bool Q4, bool Q8, bool GELU, bool TILED>
__device__ __forceinline__ void quant_unit(const QuantArgs& a, const FastDiv& div, uint32_t u, uint32_t units) {
  if (u >= units) return;  // whole blocks: the four lanes leave together
  const uint32_t q = threadIdx.x & 3u, row = div.quot(u), blk = u - row * div.d;
  const int64_t c = (int64_t)blk * kMxBlock + q * 8;
  float v[8];
  mx_load_row8<XT>(a.x, row * a.ldx, c, a.cols, v);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t m = __float_as_uint(v[j]) & 0x7fffffffu;
    top = top > m ? top : m;
  }
  top = quad_max(top);
  if constexpr (Q4) {
    const uint32_t byte = mx_scale_byte<2>(top);
    if (!TILED || blk < a.blocks4) {
      const int64_t b = (int64_t)row * a.blocks4 + blk;
      reinterpret_cast<uint32_t*>(a.codes4)[b * 4 + q] = byte == kMxNan ? 0u : mx_codes4(v, mx_scale_operand(byte));
      if (q == 0 && (!TILED || a.scales4)) a.scales4[b] = (uint8_t)byte;
    }
    if (TILED && q == 0) a.tiled[((int64_t)(blk >> 3) * a.scale_rows + a.row0 + row) * 8 + (blk & 7)] = (uint8_t)byte;
  }
  if constexpr (Q8) {
    if (blk < a.blocks8) {
      const uint32_t byte = mx_scale_byte<0>(top);
      const int64_t b = (int64_t)row * a.blocks8 + blk;
      reinterpret_cast<uint2*>(a.codes8)[b * 4 + q] = byte == kMxNan ? make_uint2(0u, 0u) : codes8(v, byte);
      if (q == 0) a.scales8[b] = (uint8_t)byte;
    }
  }
  if constexpr (GELU) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = mx_gelu<XT>(v[j]);
    mx_store_row8<XT>(a.y, row * a.cols, c, a.cols, y);
  }
}

template <int XT, bool Q4, bool Q8, bool GELU>
__global__ __launch_bounds__(256) void mx_quant_kernel(QuantArgs a, FastDiv div, uint32_t units) {
  quant_unit<XT, Q4, Q8, GELU, false>(a, div, (blockIdx.x * 256u + threadIdx.x) >> 2, units);
}

// x as a tiled product's operand, after `turn`'s work-groups.
template <int XT, bool Q8>
__global__ __launch_bounds__(256) void mx_quant_tiled_kernel(QuantArgs a, FastDiv div, uint32_t units, MxScaleTurn turn) {
  if (blockIdx.x < turn.groups) turn_scales(turn, blockIdx.x);
  else quant_unit<XT, true, Q8, false, true>(a, div, ((blockIdx.x - turn.groups) * 256u + threadIdx.x) >> 2, units);
}

// Both operands of a tiled product, the weights' work-groups first.
template <int XT, int WT, bool Q8>
__global__ __launch_bounds__(256) void mx_quant_pair_kernel(QuantArgs x, FastDiv xdiv, uint32_t xunits, QuantArgs w, FastDiv wdiv,
                                                            uint32_t wunits, uint32_t wgroups) {
  if (blockIdx.x < wgroups) quant_unit<WT, true, false, false, true>(w, wdiv, (blockIdx.x * 256u + threadIdx.x) >> 2, wunits);
  else quant_unit<XT, true, Q8, false, true>(x, xdiv, ((blockIdx.x - wgroups) * 256u + threadIdx.x) >> 2, xunits);
}

struct BackArgs {
  const void* codes;
  const uint8_t* scales;
  int64_t cols;
  const void* g;  // GELU's upstream gradient (rows of ldg), null for the plain way back
  int64_t ldg;
  void* y;
};

// Codes to values (SLOPE 0), or the upstream gradient times GELU's slope at them.  Eight elements a lane, as above.  Bound
// by the bytes: 4096 x 4096 to fp32 15 and 16 us, 5.2 TB/s; GELU of 12608 x 2048 bf16 and its gradient, which move 130 MB
// each in 25 to 31 and 24 to 27 us, also by 30 instructions an element.
template <int BITS, int YT, bool SLOPE>
__global__ __launch_bounds__(256) void mx_back_kernel(BackArgs a, FastDiv div, uint32_t units) {
  const uint32_t u = (blockIdx.x * 256u + threadIdx.x) >> 2;
  if (u >= units) return;
  const uint32_t q = threadIdx.x & 3u, row = div.quot(u), blk = u - row * div.d;
  const int64_t c = (int64_t)blk * kMxBlock + q * 8, b = (int64_t)u;
  float v[8];
  mx_decode8<BITS>(a.codes, a.scales[b], b * 4 + q, v);
  if constexpr (SLOPE) {
    float g[8];
    mx_load_row8<YT>(a.g, row * a.ldg, c, a.cols, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = g[j] * mx_gelu_slope<YT>(v[j]);
  }
  mx_store_row8<YT>(a.y, row * a.cols, c, a.cols, v);
}

// Units of a launch stay below 2^29 (FastDiv, grid of 2^31 threads): more rows go in several.
template <typename F>
int launch_rows(int64_t rows, int64_t blocks, const char* what, F&& f) {
  DIMQ_CHECK(blocks < (1 << 29), "%s: rows of %lld blocks are not supported", what, (long long)blocks);
  const int64_t step = (1 << 29) / blocks;
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t n = rows - r < step ? rows - r : step;
    const uint32_t units = (uint32_t)(n * blocks);
    f(r, FastDiv((uint32_t)blocks), units, dim3((units + 63) / 64));
    const int rc = check_launch(what);
    if (rc != DIMQ_OK) return rc;
  }
  return DIMQ_OK;
}

template <int XT>
int quant_launch(const QuantArgs& a, MxScaleTurn turn, hipStream_t s) {
  return launch_rows(a.rows, a.blocks, "mx_quantize", [&](int64_t r, FastDiv div, uint32_t units, dim3 grid) {
    QuantArgs b = a;
    const int64_t e = dtype_size(XT);
    b.x = static_cast<const char*>(a.x) + r * a.ldx * e;
    if (b.codes4) b.codes4 += r * a.blocks4 * 16;
    if (b.scales4) b.scales4 += r * a.blocks4;
    if (b.codes8) b.codes8 += r * a.blocks8 * 32, b.scales8 += r * a.blocks8;
    if (b.y) b.y = static_cast<char*>(a.y) + r * a.cols * e;
    b.row0 = r;
    if (r > 0) turn.groups = 0;
    const dim3 more(grid.x + turn.groups);
    if (b.y && b.codes8) mx_quant_kernel<XT, false, true, true><<<grid, 256, 0, s>>>(b, div, units);
    else if (b.y) mx_quant_kernel<XT, false, false, true><<<grid, 256, 0, s>>>(b, div, units);
    else if (b.tiled && b.codes8) mx_quant_tiled_kernel<XT, true><<<more, 256, 0, s>>>(b, div, units, turn);
    else if (b.tiled) mx_quant_tiled_kernel<XT, false><<<more, 256, 0, s>>>(b, div, units, turn);
    else if (b.codes4 && b.codes8) mx_quant_kernel<XT, true, true, false><<<grid, 256, 0, s>>>(b, div, units);
    else if (b.codes4) mx_quant_kernel<XT, true, false, false><<<grid, 256, 0, s>>>(b, div, units);
    else mx_quant_kernel<XT, false, true, false><<<grid, 256, 0, s>>>(b, div, units);
  });
}

template <int XT, int WT>
void pair_launch(const QuantArgs& x, const QuantArgs& w, hipStream_t s) {
  const uint32_t xu = (uint32_t)(x.rows * x.blocks), wu = (uint32_t)(w.rows * w.blocks), wg = (wu + 63) / 64;
  const dim3 grid((xu + 63) / 64 + wg);
  const FastDiv xd((uint32_t)x.blocks), wd((uint32_t)w.blocks);
  if (x.codes8) mx_quant_pair_kernel<XT, WT, true><<<grid, 256, 0, s>>>(x, xd, xu, w, wd, wu, wg);
  else mx_quant_pair_kernel<XT, WT, false><<<grid, 256, 0, s>>>(x, xd, xu, w, wd, wu, wg);
}

template <int XT>
void pair_any(int w_dtype, const QuantArgs& x, const QuantArgs& w, hipStream_t s) {
  switch (w_dtype) {
    case DIMQ_F32: pair_launch<XT, DIMQ_F32>(x, w, s); break;
    case DIMQ_F16: pair_launch<XT, DIMQ_F16>(x, w, s); break;
    default: pair_launch<XT, DIMQ_BF16>(x, w, s);
  }
}

int quant_any(int x_dtype, const QuantArgs& a, hipStream_t s, const MxScaleTurn& turn = {}) {
  if (a.rows == 0 || a.cols == 0) return DIMQ_OK;
  switch (x_dtype) {
    case DIMQ_F32: return quant_launch<DIMQ_F32>(a, turn, s);
    case DIMQ_F16: return quant_launch<DIMQ_F16>(a, turn, s);
    default: return quant_launch<DIMQ_BF16>(a, turn, s);
  }
}

template <int BITS, int YT, bool SLOPE>
int back_launch(int64_t rows, int64_t blocks, const BackArgs& a, hipStream_t s) {
  return launch_rows(rows, blocks, "mx_dequantize", [&](int64_t r, FastDiv div, uint32_t units, dim3 grid) {
    BackArgs b = a;
    const int64_t e = dtype_size(YT);
    b.codes = static_cast<const char*>(a.codes) + r * blocks * (BITS * 4);
    b.scales = a.scales + r * blocks;
    if (b.g) b.g = static_cast<const char*>(a.g) + r * a.ldg * e;
    b.y = static_cast<char*>(a.y) + r * a.cols * e;
    mx_back_kernel<BITS, YT, SLOPE><<<grid, 256, 0, s>>>(b, div, units);
  });
}

template <int BITS, bool SLOPE>
int back_any(int y_dtype, int64_t rows, const BackArgs& a, hipStream_t s) {
  if (rows == 0 || a.cols == 0) return DIMQ_OK;
  const int64_t blocks = mx_blocks(a.cols);
  switch (y_dtype) {
    case DIMQ_F32: return back_launch<BITS, DIMQ_F32, SLOPE>(rows, blocks, a, s);
    case DIMQ_F16: return back_launch<BITS, DIMQ_F16, SLOPE>(rows, blocks, a, s);
    default: return back_launch<BITS, DIMQ_BF16, SLOPE>(rows, blocks, a, s);
  }
}

int check_codes(const char* what, const void* codes, const void* scales) {
  DIMQ_CHECK(codes && scales, "%s: null pointer", what);
  DIMQ_CHECK(aligned(codes, 16), "%s: codes must be 16-byte aligned", what);
  return DIMQ_OK;
}

}  // namespace
}  // namespace dimq

namespace dimq {

static QuantArgs tiled_args(const MxTiledOperand& o) {
  QuantArgs a{o.x, o.ld, o.rows, o.cols, o.codes, o.scales, o.codes8, o.scales8, (mx_blocks(o.cols) + 7) / 8 * 8,
              mx_blocks(o.cols), mx_blocks(o.cols)};
  a.tiled = o.tiled, a.scale_rows = o.scale_rows;
  return a;
}

int mx_quantize_tiled(const MxTiledOperand& x, MxScaleTurn turn, hipStream_t s) {
  turn.stages = (turn.blocks + 7) / 8;
  const int64_t groups = (turn.stages * turn.n + 255) / 256;
  DIMQ_CHECK(groups < (1 << 28), "mxfp4_linear: too many outputs");
  turn.groups = (uint32_t)groups;
  return quant_any(x.dtype, tiled_args(x), s, turn);
}

int mx_quantize_pair(const MxTiledOperand& x, const MxTiledOperand& w, hipStream_t s) {
  const QuantArgs a = tiled_args(x), b = tiled_args(w);
  if (a.blocks >= (1 << 29) / a.rows || b.blocks >= (1 << 29) / b.rows) {  // not in one launch
    const int rc = quant_any(w.dtype, b, s);
    return rc != DIMQ_OK ? rc : quant_any(x.dtype, a, s);
  }
  switch (x.dtype) {
    case DIMQ_F32: pair_any<DIMQ_F32>(w.dtype, a, b, s); break;
    case DIMQ_F16: pair_any<DIMQ_F16>(w.dtype, a, b, s); break;
    default: pair_any<DIMQ_BF16>(w.dtype, a, b, s);
  }
  return check_launch("mx_quantize");
}

}  // namespace dimq

using namespace dimq;

extern "C" int dimq_mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes4,
                                uint8_t* scales4, int64_t blocks4, int8_t* codes8, uint8_t* scales8, void* stream) {
  int rc = mx_check_rows("mx_quantize", x, x_dtype, rows, cols, ldx);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0 || cols == 0) return DIMQ_OK;
  DIMQ_CHECK(codes4 || codes8, "mx_quantize: no output");
  if (codes4 && (rc = check_codes("mx_quantize", codes4, scales4)) != DIMQ_OK) return rc;
  if (codes8 && (rc = check_codes("mx_quantize", codes8, scales8)) != DIMQ_OK) return rc;
  const int64_t nb = mx_blocks(cols);
  DIMQ_CHECK(!codes4 || blocks4 >= nb, "mx_quantize: %lld blocks do not hold a row of %lld", (long long)blocks4,
             (long long)cols);
  return quant_any(x_dtype, {x, ldx, rows, cols, codes4, scales4, codes8, scales8, codes4 ? blocks4 : nb, codes4 ? blocks4 : nb, nb},
                   as_stream(stream));
}

extern "C" int dimq_mx_dequantize(const void* codes, const uint8_t* scales, int bits, int64_t rows, int64_t cols, void* y,
                                  int y_dtype, void* stream) {
  int rc = mx_check_rows("mx_dequantize", y, y_dtype, rows, cols, cols);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(bits == 4 || bits == 8, "mx_dequantize: bits must be 4 or 8");
  if (rows == 0 || cols == 0) return DIMQ_OK;
  if ((rc = check_codes("mx_dequantize", codes, scales)) != DIMQ_OK) return rc;
  const BackArgs a{codes, scales, cols, nullptr, 0, y};
  return bits == 4 ? back_any<4, false>(y_dtype, rows, a, as_stream(stream))
                   : back_any<8, false>(y_dtype, rows, a, as_stream(stream));
}

extern "C" int dimq_mx_gelu_forward(const void* h, int dtype, int64_t rows, int64_t cols, int64_t ldh, void* y,
                                    int8_t* codes8, uint8_t* scales8, void* stream) {
  int rc = mx_check_rows("mx_gelu_forward", h, dtype, rows, cols, ldh);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0 || cols == 0) return DIMQ_OK;
  if ((codes8 || scales8) && (rc = check_codes("mx_gelu_forward", codes8, scales8)) != DIMQ_OK) return rc;
  DIMQ_CHECK(y, "mx_gelu_forward: null pointer");
  const int64_t nb = mx_blocks(cols);
  return quant_any(dtype, {h, ldh, rows, cols, nullptr, nullptr, codes8, scales8, nb, nb, nb, y}, as_stream(stream));
}

extern "C" int dimq_mx_gelu_backward(const void* g, int dtype, int64_t rows, int64_t cols, int64_t ldg,
                                     const int8_t* codes8, const uint8_t* scales8, void* gh, void* stream) {
  int rc = mx_check_rows("mx_gelu_backward", g, dtype, rows, cols, ldg);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0 || cols == 0) return DIMQ_OK;
  if ((rc = check_codes("mx_gelu_backward", codes8, scales8)) != DIMQ_OK) return rc;
  DIMQ_CHECK(gh, "mx_gelu_backward: null pointer");
  return back_any<8, true>(dtype, rows, {codes8, scales8, cols, g, ldg, gh}, as_stream(stream));
}
