// RMS norm with the residual stream's addition, and its gradients.
//
//   h = x + r, rounded to their type (the stream that the next layer adds to)
//   y = h s w,  s = 1 / sqrt(mean(h^2) + eps)
//
// y in any float type, or as e4m3 codes of y / scale with scale = max|y| / 448 per row (448: the largest e4m3 value), the
// form that dimq_linear_grouped takes.  With u = h s (a row's normalised values) and the upstream gradients gy, gh:
//
//   c = mean(gy w u),  grad h = s (gy w - u c) + gh (x's and r's alike),  grad w = sum over rows of gy u
//
// Sums and the normalised values are fp32; y and the gradients are rounded once.  Bound by bytes: a row stays in
// registers between its reductions (T threads a row, rows.h), so x and r are read once and h, y written once.
// Measured: 16384 x 4096 bf16 with the residual to e4m3 98 us (4.8 TB/s; copies reach 5.07), 8191 x 1000 fp16 12.5 us forward,
// 14.3 + 3 backward; one row of 4096 3.9 us of kernel, 6.8 of call.
#include "rows.h"

namespace dimq {
namespace {

struct RmsArgs {
  const void* x;
  const void* r;
  int64_t ldx, ldr, rows;
  int D;
  const void* w;
  int wdt;
  float eps;
  void* y;
  int ydt;
  float* scale;  // e4m3 only
  void* h;
  // backward
  const void* gy;
  int gydt;
  int64_t ldgy;
  const void* gh;
  int64_t ldgh;
  void* gx;
  float* part;  // [groups of rows][D] sums of gy u
};

constexpr float kE4m3Max = 448.0f;

// Codes of a row.  With s = f 2^e, 1 <= f < 2, the row's y is n f for n = (h 2^e) w, which is exact for bf16 and fp16 rows
// and weights, and a code is the rounded 448 n / max|n|: f cancels, and the quotient, corrected by its remainder, meets the
// ties between two codes as exactly as they are (with y / scale formed through s, a third of the rows of 4,096 bf16 elements
// had a code on the wrong side of one).  The least scale is 2^-126: below it there would be no reciprocal.
struct E4m3Row {
  float den, inv, scale;
  // top: max|n|, infinite where a y is not finite
  __device__ __forceinline__ E4m3Row(float top, float f) {
    den = fmaxf(top, kE4m3Max * 0x1p-126f / f);
    inv = 1.0f / den;
    scale = den * f / kE4m3Max;
    if (top == 0.0f) scale = 0.0f;
    if (!(top * f < __uint_as_float(0x7f800000u))) inv = 0.0f, den = 0.0f, scale = __uint_as_float(0x7fc00000u);
  }
  __device__ __forceinline__ float code(float n) const {
    const float a = n * (kE4m3Max / 512), q = a * inv;  // by 512 at the end: 448 n may be beyond fp32
    return __builtin_amdgcn_fmed3f(512 * fmaf(fmaf(-q, den, a), inv, q), -kE4m3Max, kE4m3Max);
  }
};

// s as f 2^e; a mean square beyond fp32 gives s = 0, y = 0.
__device__ __forceinline__ float power_below(float s) { return __uint_as_float(__float_as_uint(s) & 0x7f800000u); }
__device__ __forceinline__ float factor_above(float s) {
  return __uint_as_float((__float_as_uint(s) & 0x007fffffu) | 0x3f800000u);
}

__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], const E4m3Row& r) {
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = r.code(v[j]);
  uint32_t a = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], a, true);
  uint32_t b = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], b, true);
  return make_uint2(a, b);
}

template <int T>
constexpr int threads_of() {
  return T < 256 ? 256 : T;
}

// T threads to a row (64: four rows to a work-group).  Q: e4m3 output.
template <int XT, int T, int NCH, int VEC, bool RES, bool Q>
__global__ __launch_bounds__(threads_of<T>()) void rms_norm_kernel(const RmsArgs a) {
  constexpr int kRows = threads_of<T>() / T;
  __shared__ float red[2][T / 64];
  const int t = threadIdx.x % T;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / T;
  if (row >= a.rows) return;  // uniform over a row's threads
  float w[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (a.w) {
      row_load_dt<T, VEC>(a.w, a.wdt, t, c, a.D, w[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[c][j] = 1.0f;
    }
  }
  constexpr int kSize = XT == DIMQ_F32 ? 4 : 2;
  for (; row < a.rows; row += stride) {
    const char* xr = static_cast<const char*>(a.x) + row * a.ldx * kSize;
    float v[NCH][8], q[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) row_load<XT, T, VEC>(xr, t, c, a.D, v[c]);
    if constexpr (RES) {
      const char* rr = static_cast<const char*>(a.r) + row * a.ldr * kSize;
#pragma unroll
      for (int c = 0; c < NCH; ++c) row_load<XT, T, VEC>(rr, t, c, a.D, q[c]);
      char* hr = static_cast<char*>(a.h) + row * a.D * kSize;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = rounded<XT>(v[c][j] + q[c][j]);
        row_store<XT, T, VEC>(hr, t, c, a.D, v[c]);
      }
    }
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(v[c][j], v[c][j], sq);
    sq = row_reduce<T>(sq, red[0]);
    const float s = 1.0f / sqrtf(sq / static_cast<float>(a.D) + a.eps);
    if constexpr (Q) {
      const float e = power_below(s);
      float top = 0.0f;
      bool fine = true;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[c][j] = v[c][j] * e * w[c][j];
          top = fmaxf(top, fabsf(v[c][j]));
          fine &= fabsf(v[c][j]) < __uint_as_float(0x7f800000u);
        }
      // a value that is not finite becomes the row's largest
      top = row_reduce<T, true>(fine ? top : __uint_as_float(0x7f800000u), red[1]);
      const E4m3Row q8(top, factor_above(s));
      uint8_t* yr = static_cast<uint8_t*>(a.y) + row * a.D;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const uint2 o = e4m3x8(v[c], q8);
        if constexpr (VEC == 8) {
          if (8 * (t + T * c) < a.D) *reinterpret_cast<uint2*>(yr + 8 * (t + T * c)) = o;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at = row_at<T, VEC>(t, c, j);
            if (at < a.D) yr[at] = static_cast<uint8_t>((j < 4 ? o.x : o.y) >> (8 * (j & 3)));
          }
        }
      }
      if (t == 0) a.scale[row] = q8.scale;
    } else {
      char* yr = static_cast<char*>(a.y) + row * a.D * (a.ydt == DIMQ_F32 ? 4 : 2);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = v[c][j] * s * w[c][j];
        row_store_dt<T, VEC>(yr, a.ydt, t, c, a.D, v[c]);
      }
    }
    if constexpr (T > 64) __syncthreads();  // red is free for the next row
  }
}

// Rows of any length, from memory in each pass: those that do not fit the registers.
template <bool Q>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(const RmsArgs a, int xdt) {
  __shared__ float red[2][16];
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t hrow = row * a.D;
    float sq = 0.0f;
    for (int i = t; i < a.D; i += 1024) {
      float v = load_as_float(a.x, xdt, row * a.ldx + i);
      if (a.r) {
        v += load_as_float(a.r, xdt, row * a.ldr + i);
        store_from_float(a.h, xdt, hrow + i, v);
        v = load_as_float(a.h, xdt, hrow + i);
      }
      sq = fmaf(v, v, sq);
    }
    sq = row_reduce<1024>(sq, red[0]);
    const float s = 1.0f / sqrtf(sq / static_cast<float>(a.D) + a.eps);
    const void* src = a.r ? a.h : a.x;  // each thread reads back what it wrote itself
    const int64_t base = a.r ? hrow : row * a.ldx;
    const float e = Q ? power_below(s) : s;
    E4m3Row q8(1.0f, 1.0f);
    if constexpr (Q) {
      float top = 0.0f;
      bool fine = true;
      for (int i = t; i < a.D; i += 1024) {
        const float v = load_as_float(src, xdt, base + i) * e * (a.w ? load_as_float(a.w, a.wdt, i) : 1.0f);
        top = fmaxf(top, fabsf(v));
        fine &= fabsf(v) < __uint_as_float(0x7f800000u);
      }
      top = row_reduce<1024, true>(fine ? top : __uint_as_float(0x7f800000u), red[1]);
      q8 = E4m3Row(top, factor_above(s));
      if (t == 0) a.scale[row] = q8.scale;
    }
    for (int i = t; i < a.D; i += 1024) {
      const float v = load_as_float(src, xdt, base + i) * e * (a.w ? load_as_float(a.w, a.wdt, i) : 1.0f);
      if constexpr (Q) {
        const float q = q8.code(v);
        static_cast<uint8_t*>(a.y)[hrow + i] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false));
      } else {
        store_from_float(a.y, a.ydt, hrow + i, v);
      }
    }
    __syncthreads();
  }
}

// Gradients; s is formed again from h.  Each work-group keeps the sums of gy u of its rows in registers and writes them
// as one row of `part` (a.part null: not asked for), which rms_norm_sum_kernel adds in a fixed order.
template <int XT, int T, int NCH, int VEC>
__global__ __launch_bounds__(threads_of<T>()) void rms_norm_grad_kernel(const RmsArgs a) {
  constexpr int kRows = threads_of<T>() / T;
  __shared__ float red[2][T / 64];
  const int t = threadIdx.x % T;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows, first = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / T;
  float w[NCH][8], gw[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[c][j] = 1.0f, gw[c][j] = 0.0f;
    if (a.w) row_load_dt<T, VEC>(a.w, a.wdt, t, c, a.D, w[c]);
  }
  constexpr int kSize = XT == DIMQ_F32 ? 4 : 2;
  for (int64_t row = first; row < a.rows; row += stride) {
    const char* hr = static_cast<const char*>(a.x) + row * a.ldx * kSize;
    const char* gr = static_cast<const char*>(a.gy) + row * a.ldgy * (a.gydt == DIMQ_F32 ? 4 : 2);
    float v[NCH][8], g[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) row_load<XT, T, VEC>(hr, t, c, a.D, v[c]);
    if (a.gydt == XT) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) row_load<XT, T, VEC>(gr, t, c, a.D, g[c]);
    } else {
#pragma unroll
      for (int c = 0; c < NCH; ++c) row_load_dt<T, VEC>(gr, a.gydt, t, c, a.D, g[c]);
    }
    float sq = 0.0f, dot = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sq = fmaf(v[c][j], v[c][j], sq);
        dot = fmaf(g[c][j] * w[c][j], v[c][j], dot);
      }
    sq = row_reduce<T>(sq, red[0]);
    dot = row_reduce<T>(dot, red[1]);
    const float s = 1.0f / sqrtf(sq / static_cast<float>(a.D) + a.eps);
    const float k = dot * s / static_cast<float>(a.D);  // c: the dot product was with h = u / s
    float u[NCH][8];
    if (a.gh) {
      const char* ur = static_cast<const char*>(a.gh) + row * a.ldgh * kSize;
#pragma unroll
      for (int c = 0; c < NCH; ++c) row_load<XT, T, VEC>(ur, t, c, a.D, u[c]);
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = v[c][j] * s;
        gw[c][j] = fmaf(g[c][j], n, gw[c][j]);
        o[j] = s * (g[c][j] * w[c][j] - n * k);
        if (a.gh) o[j] += u[c][j];
      }
      if (a.gx) row_store<XT, T, VEC>(static_cast<char*>(a.gx) + row * a.D * kSize, t, c, a.D, o);
    }
    if constexpr (T > 64) __syncthreads();
  }
  if (!a.part) return;
  float* pr = a.part + static_cast<int64_t>(blockIdx.x) * a.D;
  if constexpr (kRows > 1) {  // the waves' sums, added in order through the LDS
    __shared__ float sum[kRows][T * NCH * 8];
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[threadIdx.x / T][(8 * c + j) * T + t] = gw[c][j];
    __syncthreads();
    if (threadIdx.x >= T) return;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = (8 * c + j) * T + t;
        gw[c][j] = (sum[0][i] + sum[1][i]) + (sum[2][i] + sum[3][i]);
      }
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) row_store<DIMQ_F32, T, VEC>(pr, t, c, a.D, gw[c]);
}

// Rows that do not fit the registers: a row at a time, all passes from memory; part [gridDim.x][D] zeroed by its owner.
__global__ __launch_bounds__(1024) void rms_norm_grad_long_kernel(const RmsArgs a, int xdt) {
  __shared__ float red[2][16];
  const int t = threadIdx.x;
  float* pr = a.part ? a.part + static_cast<int64_t>(blockIdx.x) * a.D : nullptr;
  if (pr)
    for (int i = t; i < a.D; i += 1024) pr[i] = 0.0f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float sq = 0.0f, dot = 0.0f;
    for (int i = t; i < a.D; i += 1024) {
      const float v = load_as_float(a.x, xdt, row * a.ldx + i);
      sq = fmaf(v, v, sq);
      dot = fmaf(load_as_float(a.gy, a.gydt, row * a.ldgy + i) * (a.w ? load_as_float(a.w, a.wdt, i) : 1.0f), v, dot);
    }
    sq = row_reduce<1024>(sq, red[0]);
    dot = row_reduce<1024>(dot, red[1]);
    const float s = 1.0f / sqrtf(sq / static_cast<float>(a.D) + a.eps);
    const float k = dot * s / static_cast<float>(a.D);
    for (int i = t; i < a.D; i += 1024) {
      const float n = load_as_float(a.x, xdt, row * a.ldx + i) * s, g = load_as_float(a.gy, a.gydt, row * a.ldgy + i);
      if (pr) pr[i] = fmaf(g, n, pr[i]);
      if (a.gx) {
        float o = s * (g * (a.w ? load_as_float(a.w, a.wdt, i) : 1.0f) - n * k);
        if (a.gh) o += load_as_float(a.gh, xdt, row * a.ldgh + i);
        store_from_float(a.gx, xdt, row * a.D + i, o);
      }
    }
    __syncthreads();
  }
}

// gw[d] = sum of part's rows: 64 columns a work-group, 16 waves take every sixteenth row each.
__global__ __launch_bounds__(1024) void rms_norm_sum_kernel(const float* __restrict__ part, int n, int D, void* gw, int dt) {
  __shared__ float sum[16][64];
  const int d = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  float s = 0.0f;
  if (d < D) {
    int i = wave;
    for (; i + 112 < n; i += 128) {  // eight loads in flight
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = part[static_cast<int64_t>(i + 16 * j) * D + d];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; i < n; i += 16) s += part[static_cast<int64_t>(i) * D + d];
  }
  sum[wave][threadIdx.x & 63] = s;
  __syncthreads();
  if (wave != 0 || d >= D) return;
  s = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += sum[w][threadIdx.x];
  store_from_float(gw, dt, d, s);
}

// Threads a row and 8-element chunks a thread: a wave for rows of up to 1,024 elements, a work-group of 256 for up to
// 8,192, of 1,024 for up to 32,768; 0 beyond.
struct RowPlan {
  int threads, chunks;
};
RowPlan row_plan(int64_t D) {
  if (D <= 512) return {64, 1};
  if (D <= 1024) return {64, 2};
  if (D <= 2048) return {256, 1};
  if (D <= 4096) return {256, 2};
  if (D <= 8192) return {256, 4};
  if (D <= 32768) return {1024, 4};
  return {0, 0};
}

// Work-groups that keep the CUs full; with more rows than that each takes several.
unsigned row_groups(int64_t rows, const RowPlan& p, int64_t most) {
  const int64_t per = p.threads == 64 ? 4 : 1, want = (rows + per - 1) / per;
  return static_cast<unsigned>(want < most ? want : most);
}

template <int XT, int VEC, bool RES, bool Q>
void launch_rms(const RmsArgs& a, const RowPlan& p, hipStream_t s) {
  const dim3 grid(row_groups(a.rows, p, 2048));
#define DIMQ_RMS(T, NCH) hipLaunchKernelGGL((rms_norm_kernel<XT, T, NCH, VEC, RES, Q>), grid, dim3(threads_of<T>()), 0, s, a)
  if (p.threads == 64) {
    if (p.chunks == 1) DIMQ_RMS(64, 1);
    else DIMQ_RMS(64, 2);
  } else if (p.threads == 256) {
    if (p.chunks == 1) DIMQ_RMS(256, 1);
    else if (p.chunks == 2) DIMQ_RMS(256, 2);
    else DIMQ_RMS(256, 4);
  } else {
    DIMQ_RMS(1024, 4);
  }
#undef DIMQ_RMS
}

template <int XT, int VEC>
void launch_rms_grad(const RmsArgs& a, const RowPlan& p, unsigned groups, hipStream_t s) {
#define DIMQ_RMS(T, NCH) hipLaunchKernelGGL((rms_norm_grad_kernel<XT, T, NCH, VEC>), dim3(groups), dim3(threads_of<T>()), 0, s, a)
  if (p.threads == 64) {
    if (p.chunks == 1) DIMQ_RMS(64, 1);
    else DIMQ_RMS(64, 2);
  } else if (p.threads == 256) {
    if (p.chunks == 1) DIMQ_RMS(256, 1);
    else if (p.chunks == 2) DIMQ_RMS(256, 2);
    else DIMQ_RMS(256, 4);
  } else {
    DIMQ_RMS(1024, 4);
  }
#undef DIMQ_RMS
}

bool vec_rows(const void* p, int64_t ld, int64_t rows, int size) {
  return p == nullptr || (aligned(p, 16) && (rows <= 1 || ld * size % 16 == 0));
}

bool float_of_row(int dt) { return dt == DIMQ_F32 || dt == DIMQ_F16 || dt == DIMQ_BF16; }

int check_rms(const char* what, const void* x, int x_dtype, int64_t rows, int64_t dim, int64_t ldx, const void* w, int w_dtype,
              double eps) {
  DIMQ_CHECK(float_of_row(x_dtype), "%s: input must be fp32, fp16 or bf16", what);
  DIMQ_CHECK(rows >= 0 && dim > 0, "%s: dimensions must be positive", what);
  DIMQ_CHECK(dim < (int64_t)1 << 30, "%s: rows of 2^30 elements or more are not supported", what);
  DIMQ_CHECK(rows <= 1 || ldx >= dim, "%s: row stride is below the row length", what);
  DIMQ_CHECK(!w || float_of_row(w_dtype), "%s: weight must be fp32, fp16 or bf16", what);
  DIMQ_CHECK(eps >= 0.0, "%s: eps must be non-negative", what);
  DIMQ_CHECK(rows == 0 || x, "%s: null pointer", what);
  DIMQ_CHECK(aligned(x, dtype_size(x_dtype)), "%s: misaligned input", what);
  return DIMQ_OK;
}

// Work-groups of the backward pass: each writes its sums of gy u, so no more than half the forward pass's.
unsigned grad_groups(int64_t rows, int64_t dim) { return row_groups(rows, row_plan(dim), 1024); }

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int dimq_rms_norm(const void* x, int x_dtype, int64_t rows, int64_t dim, int64_t ldx, const void* residual,
                             int64_t ldr, const void* weight, int w_dtype, double eps, void* y, int y_dtype, float* scales,
                             void* h, void* stream) {
  const int rc = check_rms("rms_norm", x, x_dtype, rows, dim, ldx, weight, w_dtype, eps);
  if (rc != DIMQ_OK) return rc;
  const bool q = scales != nullptr;
  DIMQ_CHECK(q ? y_dtype == DIMQ_E4M3 : float_of_row(y_dtype), "rms_norm writes fp32, fp16 or bf16, or e4m3 with scales");
  DIMQ_CHECK((residual != nullptr) == (h != nullptr), "rms_norm: the residual and its sum's place go together");
  DIMQ_CHECK(rows <= 1 || !residual || ldr >= dim, "rms_norm: residual row stride is below the row length");
  if (rows == 0) return DIMQ_OK;
  DIMQ_CHECK(y, "rms_norm: null pointer");
  const hipStream_t s = as_stream(stream);
  RmsArgs a{};
  a.x = x, a.r = residual, a.ldx = ldx, a.ldr = ldr, a.rows = rows, a.D = static_cast<int>(dim);
  a.w = weight, a.wdt = w_dtype, a.eps = static_cast<float>(eps), a.y = y, a.ydt = y_dtype, a.scale = scales, a.h = h;
  const RowPlan p = row_plan(dim);
  if (p.threads == 0) {
    const dim3 grid(static_cast<unsigned>(rows < 1024 ? rows : 1024));
    if (q) hipLaunchKernelGGL((rms_norm_long_kernel<true>), grid, dim3(1024), 0, s, a, x_dtype);
    else hipLaunchKernelGGL((rms_norm_long_kernel<false>), grid, dim3(1024), 0, s, a, x_dtype);
    return check_launch("rms_norm");
  }
  const int size = dtype_size(x_dtype);
  const bool vec = dim % 8 == 0 && vec_rows(x, ldx, rows, size) && vec_rows(residual, ldr, rows, size) &&
                   vec_rows(h, dim, rows, size) && vec_rows(weight, 0, 1, 1) &&
                   (q ? aligned(y, 8) : vec_rows(y, dim, rows, dtype_size(y_dtype)));
#define DIMQ_RMS_Q(XT, VEC, RES)                         \
  if (q) launch_rms<XT, VEC, RES, true>(a, p, s);        \
  else launch_rms<XT, VEC, RES, false>(a, p, s)
#define DIMQ_RMS_RES(XT, VEC)                  \
  if (residual) { DIMQ_RMS_Q(XT, VEC, true); } \
  else { DIMQ_RMS_Q(XT, VEC, false); }
#define DIMQ_RMS_VEC(XT)               \
  if (vec) { DIMQ_RMS_RES(XT, 8) }     \
  else { DIMQ_RMS_RES(XT, 1) }
  switch (x_dtype) {
    case DIMQ_F32: DIMQ_RMS_VEC(DIMQ_F32) break;
    case DIMQ_F16: DIMQ_RMS_VEC(DIMQ_F16) break;
    default: DIMQ_RMS_VEC(DIMQ_BF16) break;
  }
#undef DIMQ_RMS_VEC
#undef DIMQ_RMS_RES
#undef DIMQ_RMS_Q
  return check_launch("rms_norm");
}

extern "C" int64_t dimq_rms_norm_backward_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return row_plan(dim).threads == 0 ? (rows < 256 ? rows : 256) * dim * 4 : static_cast<int64_t>(grad_groups(rows, dim)) * dim * 4;
}

extern "C" int dimq_rms_norm_backward(const void* h, int h_dtype, int64_t rows, int64_t dim, int64_t ldh, const void* weight,
                                      int w_dtype, double eps, const void* gy, int gy_dtype, int64_t ldgy, const void* gh,
                                      int64_t ldgh, void* gx, void* gw, int gw_dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const int rc = check_rms("rms_norm_backward", h, h_dtype, rows, dim, ldh, weight, w_dtype, eps);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(float_of_row(gy_dtype), "rms_norm_backward: the gradient must be fp32, fp16 or bf16");
  DIMQ_CHECK(!gw || float_of_row(gw_dtype), "rms_norm_backward: the weight's gradient must be fp32, fp16 or bf16");
  DIMQ_CHECK(rows <= 1 || (ldgy >= dim && (!gh || ldgh >= dim)), "rms_norm_backward: row stride is below the row length");
  DIMQ_CHECK(!gw || workspace_bytes >= dimq_rms_norm_backward_workspace_bytes(rows, dim),
             "rms_norm_backward: the workspace is too small");
  DIMQ_CHECK(rows == 0 || gy, "rms_norm_backward: null pointer");
  if (!gx && !gw) return DIMQ_OK;
  const hipStream_t s = as_stream(stream);
  RmsArgs a{};
  a.x = h, a.ldx = ldh, a.rows = rows, a.D = static_cast<int>(dim), a.w = weight, a.wdt = w_dtype;
  a.eps = static_cast<float>(eps), a.gy = gy, a.gydt = gy_dtype, a.ldgy = ldgy, a.gh = gh, a.ldgh = ldgh, a.gx = gx;
  a.part = gw ? static_cast<float*>(workspace) : nullptr;
  const RowPlan p = row_plan(dim);
  int64_t parts = 0;
  if (rows > 0) {
    if (p.threads == 0) {
      parts = rows < 256 ? rows : 256;
      hipLaunchKernelGGL(rms_norm_grad_long_kernel, dim3(static_cast<unsigned>(parts)), dim3(1024), 0, s, a, h_dtype);
    } else {
      parts = grad_groups(rows, dim);
      const int size = dtype_size(h_dtype);
      const bool vec = dim % 8 == 0 && vec_rows(h, ldh, rows, size) && vec_rows(gy, ldgy, rows, dtype_size(gy_dtype)) &&
                       vec_rows(gh, ldgh, rows, size) && vec_rows(gx, dim, rows, size) && vec_rows(weight, 0, 1, 1) &&
                       vec_rows(a.part, 0, 1, 1);
      const unsigned groups = grad_groups(rows, dim);
      switch (h_dtype) {
        case DIMQ_F32: vec ? launch_rms_grad<DIMQ_F32, 8>(a, p, groups, s) : launch_rms_grad<DIMQ_F32, 1>(a, p, groups, s); break;
        case DIMQ_F16: vec ? launch_rms_grad<DIMQ_F16, 8>(a, p, groups, s) : launch_rms_grad<DIMQ_F16, 1>(a, p, groups, s); break;
        default: vec ? launch_rms_grad<DIMQ_BF16, 8>(a, p, groups, s) : launch_rms_grad<DIMQ_BF16, 1>(a, p, groups, s); break;
      }
    }
  }
  if (gw)  // no rows: zeros
    hipLaunchKernelGGL(rms_norm_sum_kernel, dim3(static_cast<unsigned>((dim + 63) / 64)), dim3(1024), 0, s,
                       static_cast<const float*>(workspace), static_cast<int>(parts), static_cast<int>(dim), gw, gw_dtype);
  return check_launch("rms_norm_backward");
}
