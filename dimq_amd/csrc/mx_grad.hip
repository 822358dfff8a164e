// Straight-through gradients of the microscaled layers (mx.h):
//   to the input   gx = g W        W the 4-bit weights [N, K], summed over N
//   to the weight  gw = g^T X      X the 8-bit checkpoint [M, K], summed over M, and gb = sum of g over M
// Codes times scales are exact in bf16, and so is a gradient of 16 or 32 bits as a sum of bf16 parts (one for bf16, two
// for fp16's 11 bits, three for fp32's 24), so that every product is exact and only the fp32 sums round; but fp32 gradients
// below 2^-110 reach past bf16's least step 2^-133 and are taken to its nearest multiple.  W or X is
// decoded to bf16 in the workspace once (a 256 x 256 tile would decode it again for every row tile), g is split into
// planes of parts there unless it is bf16 in aligned rows, and the tiled product (mx_mm.h) sums over the planes one after
// another.  One launch makes all that ready, for both gradients at once.
#include "mx_mm.h"
#include "mx_quant.h"

namespace dimq {
namespace {

// x as NS bf16 parts that add up to it, by truncation (rounding could carry the first part to infinity).  The last of
// three is rounded: that changes nothing where |x| is 2^-110 or more, and below takes x to the nearest multiple of a part's
// least step 2^-133.  A NaN or an infinity is the first part alone.
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
    const uint32_t t = i == 2 ? float_to_bf16_bits(x) << 16 : __float_as_uint(x) & 0xffff0000u;
    h[i] = (uint16_t)(t >> 16);
    x -= __uint_as_float(t);
  }
}

constexpr int parts_of(int dt) { return dt == DIMQ_BF16 ? 1 : dt == DIMQ_F16 ? 2 : 3; }

constexpr int64_t kSumRows = 64;  // of g that a work-group adds up
int64_t sum_slices(int64_t M) { return M < 1 ? 1 : M > kSumRows * 256 ? 256 : (M + kSumRows - 1) / kSumRows; }

// The parts of the first launch, work-groups one part after another.
struct PrepArgs {
  // codes -> bf16, eight elements a thread; `units` groups of eight hold codes, the rest up to `all` become zeros
  struct Decode {
    const void* codes;
    const uint8_t* scales;
    uint16_t* out;
    int64_t units, all;
    uint32_t groups;
  } w, x;
  // g [M, N] -> planes [parts, rows, pitch], zeros past M and N, eight elements a thread
  const void* g;
  int64_t M, N, ld;
  uint16_t* planes;
  uint32_t rows, chunks;  // chunks of 8 a row
  uint32_t split_groups;
  // sums of sum_rows rows each, [slices, pitch]: 64 column groups of 8 a work-group, a row a wave in turn
  float* part;
  int64_t sum_rows, pitch;
  uint32_t sum_cols, sum_groups;
};

template <int BITS>
__device__ __forceinline__ void decode_part(const PrepArgs::Decode& d, uint32_t group) {
  const int64_t u = (int64_t)group * 256 + threadIdx.x;
  if (u >= d.all) return;
  uint4 o = make_uint4(0, 0, 0, 0);
  if (u < d.units) {
    float v[8];
    mx_decode8<BITS>(d.codes, d.scales[u >> 2], u, v);
    o = make_uint4(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]), bf16x2_rne(v[4], v[5]), bf16x2_rne(v[6], v[7]));
  }
  reinterpret_cast<uint4*>(d.out)[u] = o;
}

template <int DT>
__device__ __forceinline__ void split_part(const PrepArgs& p, uint32_t group) {
  constexpr int NS = parts_of(DT);
  const uint32_t i = group * 256u + threadIdx.x;
  if (i >= p.rows * p.chunks) return;
  const uint32_t m = i / p.chunks, n = (i - m * p.chunks) * 8;
  float v[8];
  mx_load_row8<DT>(p.g, m * p.ld, n, m < p.M ? p.N : 0, v);
  uint16_t h[8][NS];
#pragma unroll
  for (int j = 0; j < 8; ++j) bf16_parts<NS>(v[j], h[j]);
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = h[2 * j][s] | ((uint32_t)h[2 * j + 1][s] << 16);
    reinterpret_cast<uint4*>(p.planes)[(int64_t)s * p.rows * p.chunks + i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int DT>
__device__ __forceinline__ void sum_part(const PrepArgs& p, uint32_t group, float (&red)[4][8][64]) {
  const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t slice = group / p.sum_cols;
  // a last group that is not whole starts earlier: its first columns are its neighbour's, summed alike
  int64_t n = ((int64_t)(group - slice * p.sum_cols) * 64 + c) * 8, m0 = slice * p.sum_rows;
  if (n < p.N && n + 8 > p.N && p.N >= 8) n = p.N - 8;
  const int64_t m1 = m0 + p.sum_rows < p.M ? m0 + p.sum_rows : p.M;
  float s[8] = {};
  auto add = [&](int64_t m, int64_t cols) {
    float v[8];
    mx_load_row8<DT>(p.g, m * p.ld + n, 0, cols, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += v[j];
  };
  if (n < p.N) {
    int64_t m = m0 + w;
    if (p.N >= 8) {  // eight rows' loads in flight, with no branch between them
      for (; m + 28 < m1; m += 32)
#pragma unroll
        for (int i = 0; i < 8; ++i) add(m + 4 * i, 8);
    }
    for (; m < m1; m += 4) add(m, p.N - n);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) red[w][j][c] = s[j];
  __syncthreads();
  if (w == 0 && n < p.N) {
    float* o = p.part + slice * p.pitch + n;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = (red[0][j][c] + red[1][j][c]) + (red[2][j][c] + red[3][j][c]);
    mx_write16(o, make_uint4(__float_as_uint(t[0]), __float_as_uint(t[1]), __float_as_uint(t[2]), __float_as_uint(t[3])));
    mx_write16(o + 4, make_uint4(__float_as_uint(t[4]), __float_as_uint(t[5]), __float_as_uint(t[6]), __float_as_uint(t[7])));
  }
}

// Bound by the bytes: 8192 x 4096 -> 4096 decodes 42 MB of codes to 101 MB and reads 67 MB of g, 36 us or 5.8 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void prepare_kernel(const PrepArgs p) {
  __shared__ float red[4][8][64];
  uint32_t group = blockIdx.x;
  if (group < p.sum_groups) return sum_part<DT>(p, group, red);  // first: the longest-running work-groups
  group -= p.sum_groups;
  if (group < p.split_groups) return split_part<DT>(p, group);
  group -= p.split_groups;
  if (group < p.w.groups) return decode_part<4>(p.w, group);
  decode_part<8>(p.x, group - p.w.groups);
}

// The slices of the sums, added in a fixed order: 8 lanes a column take every eighth, then a tree.
__global__ __launch_bounds__(256) void add_sums_kernel(const float* part, int64_t pitch, int slices, int64_t N, void* out,
                                                       int dtype) {
  __shared__ float red[8][32];
  const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + c;
  float s = 0.0f;
  if (n < N)
#pragma unroll 8
    for (int i = w; i < slices; i += 8) s += part[i * pitch + n];
  red[w][c] = s;
  __syncthreads();
  if (w == 0 && n < N)
    store_from_float(out, dtype, n, ((red[0][c] + red[1][c]) + (red[2][c] + red[3][c])) +
                                        ((red[4][c] + red[5][c]) + (red[6][c] + red[7][c])));
}

// What is asked for, and the workspace: the decoded operands [rows, blocks, 32], g's planes where it is copied, the slices
// of split reductions (one product after the other), the bias gradient's.  Where there are several planes, both reductions
// are padded with zeros to whole stages.
struct Backward {
  int64_t w = 0, x = 0, planes = 0, part = 0, sums = 0, bytes = 0;
  int64_t parts, gm, gn, wrows, xrows;  // rows and pitch of a plane; rows of the decoded operands
  bool copy;
  MxPlan gx, gw;
  Backward(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K, bool to_x, bool to_w, bool to_b) {
    auto take = [&](int64_t& at, int64_t n) { at = bytes, bytes += (n + 255) / 256 * 256; };
    parts = parts_of(g_dtype);
    copy = parts > 1 || !mx_vec_rows(g, g_dtype, N, ldg) || ldg >= (1 << 22);  // mx_mm's limit on a row's bytes
    const int64_t whole = parts > 1 ? 64 : 1;
    wrows = (N + whole - 1) / whole * whole, xrows = (M + whole - 1) / whole * whole;
    gm = xrows, gn = mx_pad8(wrows);
    gx = mx_plan(false, M, K, (wrows + 63) / 64 * parts);
    gw = mx_plan(false, N, K, (xrows + 63) / 64 * parts);
    if (to_x) take(w, wrows * mx_blocks(K) * 64);
    if (to_w) take(x, xrows * mx_blocks(K) * 64);
    if (copy && (to_x || to_w)) take(planes, parts * gm * gn * 2);
    const int64_t px = to_x ? mx_partial_bytes(gx, M, K) : 0, pw = to_w ? mx_partial_bytes(gw, N, K) : 0;
    take(part, px > pw ? px : pw);
    if (to_b) take(sums, sum_slices(M) * mx_pad8(N) * 4);
  }
};

int check_out(const char* what, const void* out, int dtype) {
  DIMQ_CHECK(dtype == DIMQ_F32 || dtype == DIMQ_F16 || dtype == DIMQ_BF16, "%s: output dtype must be fp32, fp16 or bf16", what);
  DIMQ_CHECK(out, "%s: null pointer", what);
  return DIMQ_OK;
}
int check_codes(const char* what, const void* codes, const void* scales, int64_t rows) {
  DIMQ_CHECK(rows == 0 || (codes && scales), "%s: null pointer", what);
  DIMQ_CHECK(aligned(codes, 16), "%s: codes must be 16-byte aligned", what);
  return DIMQ_OK;
}

int backward(const char* what, const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, const uint8_t* codes,
             const uint8_t* scales, const int8_t* codes8, const uint8_t* scales8, int64_t K, void* gx, int gx_dtype, void* gw,
             int gw_dtype, void* gb, int gb_dtype, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  const Backward at(g, g_dtype, M, N, ldg, K, gx, gw, gb);
  DIMQ_CHECK(at.bytes == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= at.bytes),
             "%s: the workspace is too small or not 256-byte aligned", what);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t pitch = mx_blocks(K) * 32, slices = sum_slices(M);
  auto groups = [](int64_t threads) { return (threads + 255) / 256; };
  const int64_t wg = gx ? groups(at.wrows * pitch / 8) : 0, xg = gw ? groups(at.xrows * pitch / 8) : 0;
  const int64_t sg = at.copy && (gx || gw) ? groups(at.gm * at.gn / 8) : 0, cols = (N + 511) / 512;
  const int64_t bg = gb ? cols * slices : 0, all = wg + xg + sg + bg;
  DIMQ_CHECK(all < (1ll << 31) && sg < (1ll << 24) && at.gm < (1ll << 31), "%s: too large", what);
  const PrepArgs p{{codes, scales, reinterpret_cast<uint16_t*>(ws + at.w), N * pitch / 8, at.wrows * pitch / 8, (uint32_t)wg},
                   {codes8, scales8, reinterpret_cast<uint16_t*>(ws + at.x), M * pitch / 8, at.xrows * pitch / 8, (uint32_t)xg},
                   g, M, N, ldg, reinterpret_cast<uint16_t*>(ws + at.planes), (uint32_t)at.gm, (uint32_t)(at.gn / 8),
                   (uint32_t)sg, reinterpret_cast<float*>(ws + at.sums), (M + slices - 1) / slices, mx_pad8(N),
                   (uint32_t)cols, (uint32_t)bg};
  int rc = DIMQ_OK;
  if (all > 0) {
    const dim3 grid((unsigned)all);
    switch (g_dtype) {
      case DIMQ_F32: prepare_kernel<DIMQ_F32><<<grid, 256, 0, s>>>(p); break;
      case DIMQ_F16: prepare_kernel<DIMQ_F16><<<grid, 256, 0, s>>>(p); break;
      default: prepare_kernel<DIMQ_BF16><<<grid, 256, 0, s>>>(p);
    }
    if ((rc = check_launch(what)) != DIMQ_OK) return rc;
  }
  if (gb) {
    add_sums_kernel<<<dim3((unsigned)((N + 31) / 32)), 256, 0, s>>>(p.part, p.pitch, (int)slices, N, gb, gb_dtype);
    if ((rc = check_launch(what)) != DIMQ_OK) return rc;
  }
  const MxOperand r = at.copy ? MxOperand{ws + at.planes, at.gn * 2, nullptr, 0}
                              : MxOperand{static_cast<const uint8_t*>(g), ldg * 2, nullptr, 0};
  float* part = reinterpret_cast<float*>(ws + at.part);
  if (gx) {
    const MxMm m{r, {ws + at.w, pitch * 2, nullptr, 0}, M, K, at.wrows, at.parts, at.gm * at.gn * 2, 0,
                 MxOut{gx, gx_dtype, K, K, nullptr, 0, nullptr, 0, 0}};
    if ((rc = mx_mm<false, true, false>(m, at.gx, part, s, what)) != DIMQ_OK) return rc;
  }
  if (gw) {
    const MxMm m{r, {ws + at.x, pitch * 2, nullptr, 0}, N, K, at.xrows, at.parts, at.gm * at.gn * 2, 0,
                 MxOut{gw, gw_dtype, K, K, nullptr, 0, nullptr, 0, 0}};
    rc = mx_mm<false, true, true>(m, at.gw, part, s, what);
  }
  return rc;
}

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_mx_linear_backward_workspace_bytes(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg,
                                                           int64_t K, int outputs) {
  if (M < 0 || N <= 0 || K <= 0) return 0;
  return Backward(g, g_dtype, M, N, ldg, K, M > 0 && (outputs & 1), outputs & 2, outputs & 4).bytes;
}

extern "C" int dimq_mx_linear_backward(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, const uint8_t* codes,
                                       const uint8_t* scales, const int8_t* codes8, const uint8_t* scales8, int64_t K,
                                       void* gx, int gx_dtype, void* gw, int gw_dtype, void* gb, int gb_dtype,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "mx_linear_backward";
  int rc = mx_check_rows(what, g, g_dtype, M, N, ldg);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(K > 0 && N > 0, "linear dimensions must be positive");
  if (M == 0) gx = nullptr;  // no rows: nothing to write
  if (gx && ((rc = check_out(what, gx, gx_dtype)) != DIMQ_OK || (rc = check_codes(what, codes, scales, N)) != DIMQ_OK)) return rc;
  if (gw && ((rc = check_out(what, gw, gw_dtype)) != DIMQ_OK || (rc = check_codes(what, codes8, scales8, M)) != DIMQ_OK)) return rc;
  DIMQ_CHECK(!gb || is_float_dtype(gb_dtype), "bias gradient must be floating point");
  return backward(what, g, g_dtype, M, N, ldg, codes, scales, codes8, scales8, K, gx, gx_dtype, gw, gw_dtype, gb, gb_dtype,
                  workspace, workspace_bytes, as_stream(stream));
}

extern "C" int dimq_mx_linear_route(int product, int dtype, int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0 || product < 0 || product > 2 || (dtype != DIMQ_F32 && dtype != DIMQ_F16 && dtype != DIMQ_BF16))
    return -1;
  if (product == 0) return mx_forward_route(dtype == DIMQ_F32, M, K, N);
  const Backward at(nullptr, dtype, M, N, N, K, true, true, false);
  return product == 1 ? mx_route(at.gx, M, K, (at.wrows + 63) / 64 * at.parts)
                      : mx_route(at.gw, N, K, (at.xrows + 63) / 64 * at.parts);
}

extern "C" int64_t dimq_mx_grad_input_workspace_bytes(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K) {
  return dimq_mx_linear_backward_workspace_bytes(g, g_dtype, M, N, ldg, K, 1);
}

extern "C" int64_t dimq_mx_grad_weight_workspace_bytes(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg, int64_t K) {
  return dimq_mx_linear_backward_workspace_bytes(g, g_dtype, M, N, ldg, K, 6);
}

extern "C" int dimq_mxfp4_linear_grad_input(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg,
                                            const uint8_t* codes, const uint8_t* scales, int64_t K, void* gx,
                                            int gx_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "mxfp4_linear_grad_input";
  int rc = mx_check_rows(what, g, g_dtype, M, N, ldg);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(K > 0 && N > 0, "linear dimensions must be positive");
  if (M == 0) return DIMQ_OK;
  if ((rc = check_out(what, gx, gx_dtype)) != DIMQ_OK || (rc = check_codes(what, codes, scales, N)) != DIMQ_OK) return rc;
  return backward(what, g, g_dtype, M, N, ldg, codes, scales, nullptr, nullptr, K, gx, gx_dtype, nullptr, 0, nullptr, 0,
                  workspace, workspace_bytes, as_stream(stream));
}

extern "C" int dimq_mx_linear_grad_weight(const void* g, int g_dtype, int64_t M, int64_t N, int64_t ldg,
                                          const int8_t* codes8, const uint8_t* scales8, int64_t K, void* gw, int gw_dtype,
                                          void* gb, int gb_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "mx_linear_grad_weight";
  int rc = mx_check_rows(what, g, g_dtype, M, N, ldg);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(K > 0 && N > 0, "linear dimensions must be positive");
  DIMQ_CHECK(!gb || is_float_dtype(gb_dtype), "bias gradient must be floating point");
  if ((rc = check_out(what, gw, gw_dtype)) != DIMQ_OK || (rc = check_codes(what, codes8, scales8, M)) != DIMQ_OK) return rc;
  return backward(what, g, g_dtype, M, N, ldg, nullptr, nullptr, codes8, scales8, K, nullptr, 0, gw, gw_dtype, gb, gb_dtype,
                  workspace, workspace_bytes, as_stream(stream));
}
