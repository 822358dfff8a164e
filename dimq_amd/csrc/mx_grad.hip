// Straight-through gradients of the microscaled layers (mx.h):
//   to the input   gx = g W        W the 4-bit weights [N, K], summed over N
//   to the weight  gw = g^T X      X the 8-bit checkpoint [M, K], summed over M, and gb = sum of g over M
// Codes times scales are exact in bf16, and so is a gradient of 16 or 32 bits as a sum of bf16 parts (one for bf16, two
// for fp16's 11 bits, three for fp32's 24), so that every product is exact and only the fp32 sums round.  W or X is
// decoded to bf16 in the workspace once (a 256 x 256 tile would decode it again for every row tile), g is split into
// planes of parts there unless it is bf16 and its rows can be read 16 bytes at a time, and the tiled product (mx_mm.h)
// sums over the planes one after another.
#include "mx_mm.h"
#include "mx_quant.h"

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

constexpr int parts_of(int dt) { return dt == DIMQ_BF16 ? 1 : dt == DIMQ_F16 ? 2 : 3; }

// g [M, N] -> planes [NS, rows, pitch] of its bf16 parts, zeros past M and N; eight elements a thread.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void split_planes(const void* g, int64_t M, int64_t N, int64_t ld, int64_t rows,
                                                    int64_t pitch, uint16_t* out) {
  constexpr int NS = parts_of(DT);
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= rows * pitch) return;
  const int64_t m = i / pitch, n = i - m * pitch;
  float v[8];
  mx_load_row8<DT, VEC>(g, m * ld, n, m < M ? N : 0, v);
  uint16_t h[8][NS];
#pragma unroll
  for (int j = 0; j < 8; ++j) bf16_parts<NS>(v[j], h[j]);
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = h[2 * j][s] | ((uint32_t)h[2 * j + 1][s] << 16);
    *reinterpret_cast<uint4*>(out + s * rows * pitch + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

int split_any(int dt, const void* g, int64_t M, int64_t N, int64_t ld, int64_t rows, int64_t pitch, uint16_t* out, hipStream_t s) {
  const int64_t grid = (rows * pitch / 8 + 255) / 256;
  DIMQ_CHECK(grid < (1ll << 31), "mx gradient: the gradient is too large");
  const bool vec = mx_vec_rows(g, dt, N, ld);
#define DIMQ_MX_SPLIT(T)                                                                       \
  if (vec) split_planes<T, true><<<dim3((unsigned)grid), 256, 0, s>>>(g, M, N, ld, rows, pitch, out); \
  else split_planes<T, false><<<dim3((unsigned)grid), 256, 0, s>>>(g, M, N, ld, rows, pitch, out);    \
  break
  switch (dt) {
    case DIMQ_F32: DIMQ_MX_SPLIT(DIMQ_F32);
    case DIMQ_F16: DIMQ_MX_SPLIT(DIMQ_F16);
    default: DIMQ_MX_SPLIT(DIMQ_BF16);
  }
#undef DIMQ_MX_SPLIT
  return check_launch("mx gradient");
}

// Rows from .. to - 1 of [to, cols] 16-bit values, cols % 32 == 0, become zeros.
__global__ __launch_bounds__(256) void zero_rows_kernel(uint4* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = make_uint4(0, 0, 0, 0);
}
int zero_rows(uint8_t* p, int64_t from, int64_t to, int64_t cols, hipStream_t s) {
  const int64_t n = (to - from) * cols / 8;  // fewer than 64 rows
  if (n <= 0) return DIMQ_OK;
  DIMQ_CHECK((n + 255) / 256 < (1ll << 31), "mx gradient: too many columns");
  zero_rows_kernel<<<dim3((unsigned)((n + 255) / 256)), 256, 0, s>>>(reinterpret_cast<uint4*>(p + from * cols * 2), n);
  return check_launch("mx gradient");
}

// Sums over the rows, two launches: work-group (i, j) adds rows j, j + 4 rows ... of 64 column groups of 8; the slices
// are added in their order by mx_reduce_kernel.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void row_sums(const void* g, int64_t M, int64_t N, int64_t ld, int64_t rows, float* part,
                                                int64_t pitch) {
  __shared__ float red[4][8][64];
  const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t n = ((int64_t)blockIdx.x * 64 + c) * 8, m0 = (int64_t)blockIdx.y * rows;
  const int64_t m1 = m0 + rows < M ? m0 + rows : M;
  float s[8] = {};
  if (n < N)
#pragma unroll 4
    for (int64_t m = m0 + w; m < m1; m += 4) {
      float v[8];
      mx_load_row8<DT, VEC>(g, m * ld, n, N, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
#pragma unroll
  for (int j = 0; j < 8; ++j) red[w][j][c] = s[j];
  __syncthreads();
  if (w == 0 && n < N) {
    float* o = part + blockIdx.y * pitch + n;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = (red[0][j][c] + red[1][j][c]) + (red[2][j][c] + red[3][j][c]);
    *reinterpret_cast<float4*>(o) = make_float4(t[0], t[1], t[2], t[3]);
    *reinterpret_cast<float4*>(o + 4) = make_float4(t[4], t[5], t[6], t[7]);
  }
}

constexpr int64_t kSumRows = 64;
int64_t sum_slices(int64_t M) { return M < 1 ? 1 : M > kSumRows * 256 ? 256 : (M + kSumRows - 1) / kSumRows; }

int sums_any(int dt, const void* g, int64_t M, int64_t N, int64_t ld, float* part, void* gb, int gb_dtype, hipStream_t s) {
  const int64_t slices = sum_slices(M), rows = (M + slices - 1) / slices, pitch = mx_pad8(N);
  const dim3 grid((unsigned)((N + 511) / 512), (unsigned)slices);
  const bool vec = mx_vec_rows(g, dt, N, ld);
#define DIMQ_MX_SUM(T)                                                         \
  if (vec) row_sums<T, true><<<grid, 256, 0, s>>>(g, M, N, ld, rows, part, pitch); \
  else row_sums<T, false><<<grid, 256, 0, s>>>(g, M, N, ld, rows, part, pitch);    \
  break
  switch (dt) {
    case DIMQ_F32: DIMQ_MX_SUM(DIMQ_F32);
    case DIMQ_F16: DIMQ_MX_SUM(DIMQ_F16);
    default: DIMQ_MX_SUM(DIMQ_BF16);
  }
#undef DIMQ_MX_SUM
  int rc = check_launch("mx_linear_grad_weight");
  if (rc != DIMQ_OK) return rc;
  mx_reduce_kernel<<<dim3((unsigned)((pitch / 8 + 255) / 256)), 256, 0, s>>>(part, pitch, (int)slices, 1, pitch,
                                                                             MxOut{gb, gb_dtype, N, N, nullptr, 0, nullptr, 0, 0});
  return check_launch("mx_linear_grad_weight");
}

// Workspace of a gradient product over the codes' rows (M or N of them): the decoded operand [rows, blocks, 32], g's
// planes where it is copied, the slices of a split reduction, the bias gradient's.  Where there are several planes, the
// reduction is padded with zeros to whole stages in both operands.
struct GradLayout {
  int64_t dec = 0, planes = 0, part = 0, sums = 0, bytes = 0;
  bool copy;
  int64_t len, gm, gn;  // the reduction's length; rows and pitch of a plane
  MxPlan plan;
  GradLayout(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K, bool weight) {
    const int64_t ns = parts_of(g_dtype);
    len = weight ? M : N;
    if (ns > 1) len = (len + 63) / 64 * 64;
    gm = weight ? len : M, gn = weight ? mx_pad8(N) : mx_pad8(len);
    auto take = [&](int64_t& at, int64_t n) { at = bytes, bytes += (n + 255) / 256 * 256; };
    copy = ns > 1 || !mx_vec_rows(g, g_dtype, N, ldg);
    plan = mx_plan(false, weight ? N : M, K, (len + 63) / 64 * ns);
    take(dec, len * mx_blocks(K) * 64);
    if (copy) take(planes, ns * gm * gn * 2);
    take(part, mx_partial_bytes(plan, weight ? N : M, K));
    if (weight) take(sums, sum_slices(M) * mx_pad8(N) * 4);
  }
};

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

extern "C" int64_t dimq_mx_grad_input_workspace_bytes(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return GradLayout(g, g_dtype, M, N, ldg, K, false).bytes;
}

extern "C" int64_t dimq_mx_grad_weight_workspace_bytes(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K) {
  if (M < 0 || N <= 0 || K <= 0) return 0;
  return GradLayout(g, g_dtype, M, N, ldg, K, true).bytes;
}

extern "C" int dimq_mxfp4_linear_grad_input(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg,
                                            const uint8_t* codes, const uint8_t* scales, int64_t K, void* gx,
                                            int gx_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_grad("mxfp4_linear_grad_input", g, g_dtype, M, N, ldg, codes, scales, K, gx, gx_dtype);
  if (rc != DIMQ_OK || M == 0) return rc;
  const GradLayout at(g, g_dtype, M, N, ldg, K, false);
  DIMQ_CHECK(workspace && aligned(workspace, 256) && workspace_bytes >= at.bytes,
             "mxfp4_linear_grad_input: the workspace is too small or not 256-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t kp = mx_blocks(K) * 32;
  rc = dimq_mx_dequantize(codes, scales, 4, N, kp, ws + at.dec, DIMQ_BF16, stream);
  if (rc != DIMQ_OK || (rc = zero_rows(ws + at.dec, N, at.len, kp, as_stream(stream))) != DIMQ_OK) return rc;
  MxOperand r{static_cast<const uint8_t*>(g), ldg * 2, nullptr, 0};
  if (at.copy) {
    rc = split_any(g_dtype, g, M, N, ldg, at.gm, at.gn, reinterpret_cast<uint16_t*>(ws + at.planes), as_stream(stream));
    if (rc != DIMQ_OK) return rc;
    r = {ws + at.planes, at.gn * 2, nullptr, 0};
  }
  const MxMm p{r, {ws + at.dec, kp * 2, nullptr, 0}, M, K, at.len, parts_of(g_dtype), at.gm * at.gn * 2, 0,
               MxOut{gx, gx_dtype, K, K, nullptr, 0, nullptr, 0, 0}};
  return mx_mm<false, true, false>(p, at.plan, reinterpret_cast<float*>(ws + at.part), as_stream(stream),
                                   "mxfp4_linear_grad_input");
}

extern "C" int dimq_mx_linear_grad_weight(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg,
                                          const int8_t* codes8, const uint8_t* scales8, int64_t K, void* gw, int gw_dtype,
                                          void* gb, int gb_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_grad("mx_linear_grad_weight", g, g_dtype, M, N, ldg, codes8, scales8, K, gw, gw_dtype);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(gw, "mx_linear_grad_weight: null pointer");
  DIMQ_CHECK(!gb || is_float_dtype(gb_dtype), "bias gradient must be floating point");
  const GradLayout at(g, g_dtype, M, N, ldg, K, true);
  DIMQ_CHECK(workspace && aligned(workspace, 256) && workspace_bytes >= at.bytes,
             "mx_linear_grad_weight: the workspace is too small or not 256-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t kp = mx_blocks(K) * 32;
  rc = dimq_mx_dequantize(codes8, scales8, 8, M, kp, ws + at.dec, DIMQ_BF16, stream);
  if (rc != DIMQ_OK || (rc = zero_rows(ws + at.dec, M, at.len, kp, as_stream(stream))) != DIMQ_OK) return rc;
  if (gb) {
    rc = sums_any(g_dtype, g, M, N, ldg, reinterpret_cast<float*>(ws + at.sums), gb, gb_dtype, as_stream(stream));
    if (rc != DIMQ_OK) return rc;
  }
  MxOperand r{static_cast<const uint8_t*>(g), ldg * 2, nullptr, 0};
  if (at.copy) {
    if (M > 0) rc = split_any(g_dtype, g, M, N, ldg, at.gm, at.gn, reinterpret_cast<uint16_t*>(ws + at.planes), as_stream(stream));
    if (rc != DIMQ_OK) return rc;
    r = {ws + at.planes, at.gn * 2, nullptr, 0};
  }
  const MxMm p{r, {ws + at.dec, kp * 2, nullptr, 0}, N, K, at.len, parts_of(g_dtype), at.gm * at.gn * 2, 0,
               MxOut{gw, gw_dtype, K, K, nullptr, 0, nullptr, 0, 0}};
  return mx_mm<false, true, true>(p, at.plan, reinterpret_cast<float*>(ws + at.part), as_stream(stream),
                                  "mx_linear_grad_weight");
}
