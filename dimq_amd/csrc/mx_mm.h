// Tiled products of the microscaled layers: out[i, j] = sum_r R[i, r] C[j, r], i the output's rows, j its columns.
//
// Two forms of operands:
//   FP4   4-bit codes with block scales on the scaled matrix instructions (y = Q4(x) W^T: R = x, C = the weights)
//   bf16  exact bf16 values (the gradients: C the decoded weights or checkpoint, R the gradient's bf16 parts, one plane
//         after another along the reduction)
// An operand lies in memory either with its reduction index fastest ("plain") or slowest ("turned"): the gradients need
// the weights [N, K] summed over N and the checkpoint [M, K] and g [M, N] summed over M; turned tiles go into the LDS as
// they lie and are read back through the transposing LDS loads, so that no pass over memory turns them.
//
// A work-group owns WGR x WGC waves of RB x CB blocks of 32 x 32 outputs.  A stage is 128 bytes of reduction of every
// tile row (256 codes or 64 bf16), four steps of the matrix instructions, brought in by direct global-to-LDS loads of 16
// bytes a lane into a ring of S slots; no register holds operands in flight and the main loop has no vector arithmetic.
// C is the instructions' first operand, so a lane's accumulators are four neighbouring columns of one row.
//
// Measured: 16384 x 8192 codes summed over 8192 507 to 522 us (4,210 to 4,340 TFLOP/s); both bf16 gradients of
// 8192 x 4096 -> 4096 209 and 203 us (1,315 and 1,354 TFLOP/s; the library's product of 8192^3 reaches 1,448 there).  The
// matrix unit is busy 59 % (codes) and 70 % of the cycles, at the 1.7 GHz that the card holds under this load.  Not bound by
// memory: without any load in the loop the same data take 514 us of 520 and 187 of 204.  How the rest divides among the LDS
// reads, the barriers and scheduling fences of the steps and the epilogue is not known.
#pragma once

#include <type_traits>
#include <utility>

#include "mx_quant.h"

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

struct MxOperand {
  const uint8_t* p;
  int64_t ld;              // bytes between rows (plain: of the output index; turned: of the reduction index)
  const uint8_t* scales;   // FP4: [stages, scale_rows, 8] bytes, as many rows as whole tiles read (mx_scale_rows)
  int64_t scale_rows;
};

struct MxMm {
  MxOperand r, c;
  int64_t rows, cols;      // of the output
  int64_t len;             // reduction length of a plane: blocks (FP4) or elements; with several planes a multiple of 64
  int64_t planes, plane_bytes;  // of r
  int64_t partial;         // elements between the slices of a split reduction (fp32, out.y)
  MxOut out;
};

#ifdef __HIPCC__

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void mx_lds_void;

// What reduction tails read.
static __device__ const uint4 kMxZero = {0, 0, 0, 0};

// 16 bytes a lane from base + off into the LDS at lds + 16 lane.  Inline, as dma16 (common.h), so that the waits are the
// kernel's.
__device__ __forceinline__ void mx_dma16(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
// A pointer that is the same in all lanes, in scalar registers.
__device__ __forceinline__ const uint8_t* mx_uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const uint8_t*>(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ void mx_dma4(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("global_load_lds_dword %0, %1" ::"v"(off), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}

// On every lambda of the tile kernel: an accumulator that one takes by reference has to stay in registers.
#define MX_INLINE __attribute__((always_inline))

template <class F, int... I>
__device__ __forceinline__ void mx_each_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void mx_each(F&& f) {
  mx_each_impl(f, std::make_integer_sequence<int, N>{});
}

// Columns n .. n + 7 of a bias or residual; those from `left` on are 0.
__device__ __forceinline__ void mx_load8(const void* p, int dt, int64_t at, int left, float (&v)[8]) {
  if (left >= 8 && dt != DIMQ_F64) {
    if (dt == DIMQ_F32) mx_load_row8<DIMQ_F32>(p, at, 0, 8, v);
    else if (dt == DIMQ_F16) mx_load_row8<DIMQ_F16>(p, at, 0, 8, v);
    else mx_load_row8<DIMQ_BF16>(p, at, 0, 8, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < left ? load_as_float(p, dt, at + j) : 0.0f;
}

// 16 bytes to a multiple of the element's size.
template <bool STREAM>
__device__ __forceinline__ void mx_put(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  const u4 v = {a, b, c, d};
  if constexpr (STREAM) __builtin_nontemporal_store(v, static_cast<u4*>(p));
  else *static_cast<u4*>(p) = v;
}

// Outputs n .. n + 7 (n % 8 == 0) of row m; bias: the column's (zeros without one); STREAM: past the L2.
template <bool STREAM>
__device__ __forceinline__ void mx_store8(const MxOut& o, int64_t m, int64_t n, float (&v)[8], const float (&bias)[8]) {
  const int64_t at = m * o.ld + n;
  const int left = o.cols - n < 8 ? (int)(o.cols - n) : 8;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] += bias[j];
  if (o.res) {
    float r[8];
    mx_load8(o.res, o.res_dtype, at, left, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
  }
  if (o.act == DIMQ_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];  // NaN passes
  } else if (o.act == DIMQ_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = mx_gelu<DIMQ_F32>(v[j]);
  }
  if (left == 8) {
    if (o.dtype == DIMQ_F32) {
      float* y = static_cast<float*>(o.y) + at;
      mx_put<STREAM>(y, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      mx_put<STREAM>(y + 4, __float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = o.dtype == DIMQ_F16 ? f16x2_rne(v[2 * j], v[2 * j + 1]) : bf16x2_rne(v[2 * j], v[2 * j + 1]);
      mx_put<STREAM>(static_cast<uint16_t*>(o.y) + at, w[0], w[1], w[2], w[3]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) store_from_float(o.y, o.dtype, at + j, v[j]);
}

// Tiles in the order of their work-groups: those of one XCD (work-groups i, i + 8, ...) are a contiguous run, in columns
// of 8 row tiles, so that the 32 tiles an XCD works on share few operand rows in its L2: 8 x 4 tiles read 12 tile edges,
// 1 x 32 would read 33.
__device__ __forceinline__ void mx_tile(uint32_t row_tiles, uint32_t col_tiles, uint32_t& rt, uint32_t& ct) {
  constexpr uint32_t kXCD = 8, kGroup = 8;
  const uint32_t T = gridDim.x, per = T / kXCD;
  uint32_t id = blockIdx.x;
  if (id < per * kXCD) id = (id % kXCD) * per + id / kXCD;
  const uint32_t run = row_tiles > kGroup ? kGroup * col_tiles : T;  // tiles of a column group; T below 2^31
  const uint32_t first = id / run * kGroup;
  const uint32_t high = row_tiles - first < kGroup ? row_tiles - first : kGroup;
  const uint32_t in = id - first * col_tiles;
  rt = first + in % high;
  ct = in / high;
}

template <bool FP4_, bool CT_, bool RT_, int WGR_, int WGC_, int RB_, int CB_, int S_>
struct MxTile {
  static constexpr bool FP4 = FP4_, CT = CT_, RT = RT_;  // turned operands
  static constexpr int WGR = WGR_, WGC = WGC_, RB = RB_, CB = CB_, S = S_;
  static constexpr int NW = WGR * WGC, NT = 64 * NW, BR = WGR * RB * 32, BC = WGC * CB * 32;
  static constexpr int DATA = (BC + BR) * 128, STAGE = DATA + (FP4 ? (BC + BR) * 8 : 0);
  // loads of a wave a stage: C, R, their scales (waves past the last 32 rows repeat the first ones)
  static constexpr int LC = BC / 8 / NW, LR = BR / 8 / NW, LD = LC + LR;
  static constexpr int LCS = FP4 ? (BC / 32 + NW - 1) / NW : 0, LRS = FP4 ? (BR / 32 + NW - 1) / NW : 0;
  static constexpr int LPT = LD + LCS + LRS;
  static constexpr int UNIT = FP4 ? 8 : 64;  // of len a stage
  static_assert(LC * NW * 8 == BC && LR * NW * 8 == BR, "even loads");
  static_assert(S >= 2 && (S - 1) * LPT < 64, "vmcnt is 6 bits");
  static_assert(S * STAGE <= 160 * 1024, "LDS");
  static_assert(NW * 32 * CB * 128 <= S * STAGE, "a parked block of every wave fits the ring");
  static_assert(!(FP4 && (CT || RT)), "codes are plain");
};

// Position of 16-byte chunk c of tile row r, plain: 16 rows of one chunk, which one LDS read serves, lie in 16 places of
// the 256 bytes that the banks span.
__device__ __forceinline__ int mx_swz(int r) { return (r >> 1) & 7; }
// Turned (rows of `pitch` bytes, one reduction index each): a transposing read takes 64 bytes of each of 4 consecutive
// rows; they lie in 4 quarters of the 256 bytes (of a 128- or 384-byte pitch: in the halves of two rows).
template <int PITCH>
__device__ __forceinline__ int mx_swz_turned(int k) {
  return PITCH % 256 == 0 ? 4 * (k & 3) : 4 * ((k >> 1) & 1);
}

template <class T>
__global__ __launch_bounds__(T::NT) void mx_mm_kernel(const MxMm p) {
  constexpr int S = T::S, NW = T::NW, RB = T::RB, CB = T::CB, BC = T::BC, BR = T::BR;
  __shared__ __attribute__((aligned(16))) uint8_t sm[S * T::STAGE];
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave / T::WGC, wc = wave - wr * T::WGC;
  uint32_t rt, ct;
  mx_tile((uint32_t)((p.rows + BR - 1) / BR), (uint32_t)((p.cols + BC - 1) / BC), rt, ct);
  const int64_t r0 = (int64_t)rt * BR, c0 = (int64_t)ct * BC;
  const uint32_t smb = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((mx_lds_void*)sm));

  // ---- loads: 1024 bytes of a tile each.  Offsets of a lane against the tile's first row (plain) or column (turned)
  // stay; the stage moves the base.  Rows past the end repeat the last one, columns past the end the first: they make
  // outputs that are not stored.
  auto offset = [&](auto turned, const MxOperand& o, int64_t first, int64_t count, auto width, int b) MX_INLINE -> uint32_t {
    constexpr int W = decltype(width)::value;
    if constexpr (decltype(turned)::value) {
      const int at = b * 1024 + lane * 16, k = at / (2 * W);
      const int64_t chunk = (at % (2 * W) / 16) ^ mx_swz_turned<2 * W>(k);
      return (uint32_t)(k * o.ld + (first + chunk * 8 < count ? chunk * 16 : 0));
    } else {
      const int row = b * 8 + lane / 8;
      const int64_t i = first + row < count ? row : count - 1 - first;
      return (uint32_t)(i * o.ld + (((lane & 7) ^ mx_swz(row)) << 4));
    }
  };
  using CT = std::bool_constant<T::CT>;
  using RT = std::bool_constant<T::RT>;
  using BCc = std::integral_constant<int, BC>;
  using BRc = std::integral_constant<int, BR>;
  uint32_t off[T::LC + T::LR];
#pragma unroll
  for (int j = 0; j < T::LC; ++j) off[j] = offset(CT{}, p.c, c0, p.cols, BCc{}, j * NW + wave);
#pragma unroll
  for (int j = 0; j < T::LR; ++j) off[T::LC + j] = offset(RT{}, p.r, r0, p.rows, BRc{}, j * NW + wave);
  // bases of the stage to request next: data and scales
  const uint8_t* cb = p.c.p + (T::CT ? c0 * 2 : c0 * p.c.ld);
  const uint8_t* rb = p.r.p + (T::RT ? r0 * 2 : r0 * p.r.ld);
  const uint8_t* csb = p.c.scales + c0 * 8;
  const uint8_t* rsb = p.r.scales + r0 * 8;
  const int cstep = (int)(T::CT ? 64 * p.c.ld : 128), rstep = (int)(T::RT ? 64 * p.r.ld : 128);
  const int csstep = (int)(p.c.scale_rows * 8), rsstep = (int)(p.r.scale_rows * 8);

  const int per = (int)((p.len + T::UNIT - 1) / T::UNIT), total = per * (int)p.planes;  // stages of a plane, of all
  int t0 = 0, t1 = total, it = 0, ik = 0;  // it, ik: the stage to request next, its place in its plane
  if (gridDim.y > 1) {
    t0 = (int)((int64_t)total * blockIdx.y / gridDim.y), t1 = (int)((int64_t)total * (blockIdx.y + 1) / gridDim.y);
    const int ip = t0 / per;
    it = t0, ik = t0 - ip * per;
    cb += (int64_t)ik * cstep, rb += ip * p.plane_bytes + (int64_t)ik * rstep;
    csb += (int64_t)it * csstep, rsb += (int64_t)it * rsstep;
  }
  cb = mx_uniform(cb), rb = mx_uniform(rb), csb = mx_uniform(csb), rsb = mx_uniform(rsb);
  const int64_t cback = (int64_t)per * cstep, rback = p.plane_bytes - (int64_t)per * rstep;
  auto advance = [&]() MX_INLINE {
    ++it;
    cb += cstep, rb += rstep;
    if constexpr (T::FP4) csb += csstep, rsb += rsstep;
    if (++ik == per) ik = 0, cb -= cback, rb += rback;
  };
  const int tail = (int)(p.len - (int64_t)(per - 1) * T::UNIT);  // of UNIT, in the last stage (UNIT with several planes)
  // load j of that stage, a whole one
  auto issue1 = [&](int slot, auto jc) MX_INLINE {
    constexpr int j = decltype(jc)::value;
    const uint32_t at = smb + slot * T::STAGE;
    if constexpr (j < T::LD) {
      mx_dma16(j < T::LC ? cb : rb, off[j], at + (j * NW + wave) * 1024);
    } else if constexpr (j < T::LD + T::LCS) {
      const int b = ((j - T::LD) * NW + wave) % (BC / 32);
      mx_dma4(csb, b * 256 + lane * 4, at + T::DATA + b * 256);
    } else {
      const int b = ((j - T::LD - T::LCS) * NW + wave) % (BR / 32);
      mx_dma4(rsb, b * 256 + lane * 4, at + T::DATA + BC * 8 + b * 256);
    }
  };
  // loads J0 .. J1 - 1 of the next stage into `slot`, if there is one
  auto issue = [&](int slot, auto j0c, auto j1c) MX_INLINE {
    constexpr int J0 = decltype(j0c)::value, J1 = decltype(j1c)::value;
    if (it >= t1) return;
    const bool whole = it + 1 < total || tail == T::UNIT;
    mx_each<J1 - J0>([&](auto i) MX_INLINE {
      constexpr int j = J0 + decltype(i)::value;
      if constexpr (j < T::LD) {
        if (!whole) {  // the reduction ends inside this stage: zeros past it
          constexpr bool c = j < T::LC;
          constexpr int W = c ? BC : BR;
          const int b = (c ? j : j - T::LC) * NW + wave;
          const int k = (c ? T::CT : T::RT) ? (b * 1024 + lane * 16) / (2 * W)
                                            : ((lane & 7) ^ mx_swz(b * 8 + lane / 8)) * (T::UNIT / 8);
          const uint8_t* src = k < tail ? (c ? cb : rb) + off[j] : reinterpret_cast<const uint8_t*>(&kMxZero);
          dma16(src, smb + slot * T::STAGE + (j * NW + wave) * 1024);
          return;
        }
      }
      issue1(slot, std::integral_constant<int, j>{});
    });
  };
  using J0 = std::integral_constant<int, 0>;
  using JH = std::integral_constant<int, (T::LPT + 1) / 2>;
  using JL = std::integral_constant<int, T::LPT>;
  auto wait_stages = [&](int n) MX_INLINE {  // at most n stages of loads still in flight, 0 <= n < S
    mx_each<S>([&](auto ic) MX_INLINE {
      constexpr int I = decltype(ic)::value;
      if (I == n) wait_vmcnt<I * T::LPT>();
    });
  };

  f32x16 acc[RB][CB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  // ---- fragments of step s: 16 bytes a lane.  FP4: block 4 g + s of the stage's 8, so that a lane's four scales are one
  // dword; bf16: elements 16 s + 8 g .. + 7.
  const int q16 = lane & 15, half = (lane >> 4) & 1;
  auto frag = [&](auto turned, auto width, const uint8_t* tile, int blk, int s) MX_INLINE -> uint4 {
    constexpr int W = decltype(width)::value;
    if constexpr (decltype(turned)::value) {
      constexpr int PITCH = 2 * W;
      const int k = 8 * g + (q16 >> 2);
      const int pos = (4 * blk + 2 * half + ((q16 & 3) >> 1)) ^ mx_swz_turned<PITCH>(q16 >> 2);
      const uint8_t* a = tile + k * PITCH + pos * 16 + (q16 & 1) * 8 + s * 16 * PITCH;
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)a));
      const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(a + 4 * PITCH)));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      const int chunk = T::FP4 ? 4 * g + s : 2 * s + g;
      return *reinterpret_cast<const uint4*>(tile + (blk * 32 + col) * 128 + ((chunk ^ mx_swz(col)) << 4));
    }
  };
  uint4 cf[2][CB], rf[2][RB];
  int cs[CB], rs[RB], cn[CB], rn[RB];
  constexpr int P = RB * CB, F = RB + CB;
  // fragment f of step s into buffer b, in the order that the products want them: c0 r0 c1 r1 ...
  auto load1 = [&](int slot, int s, int b, auto fc) MX_INLINE {
    constexpr int f = decltype(fc)::value, lo = RB < CB ? RB : CB;
    constexpr bool c = f < 2 * lo ? f % 2 == 0 : CB > RB;
    constexpr int i = f < 2 * lo ? f / 2 : f - lo;
    const uint8_t* base = sm + slot * T::STAGE;
    if constexpr (c) cf[b][i] = frag(CT{}, BCc{}, base, wc * CB + i, s);
    else rf[b][i] = frag(RT{}, BRc{}, base + BC * 128, wr * RB + i, s);
  };
  auto load = [&](int slot, int s, int b) MX_INLINE { mx_each<F>([&](auto f) MX_INLINE { load1(slot, s, b, f); }); };
  auto load_scales = [&](int slot, int (&c)[CB], int (&r)[RB]) MX_INLINE {
    if constexpr (T::FP4) {
      const uint8_t* base = sm + slot * T::STAGE + T::DATA + col * 8 + g * 4;
#pragma unroll
      for (int j = 0; j < CB; ++j) c[j] = *reinterpret_cast<const int*>(base + (wc * CB + j) * 256);
#pragma unroll
      for (int i = 0; i < RB; ++i) r[i] = *reinterpret_cast<const int*>(base + BC * 8 + (wr * RB + i) * 256);
    }
  };
  // the products of step s; f(n) after the n-th
  auto mma = [&](auto sc, auto&& f) MX_INLINE {
    constexpr int s = decltype(sc)::value, b = s & 1;
    mx_each<P>([&](auto nc) MX_INLINE {
      constexpr int i = decltype(nc)::value / CB, j = decltype(nc)::value % CB;
      if constexpr (T::FP4) {
        const i32x8 x = {(int)cf[b][j].x, (int)cf[b][j].y, (int)cf[b][j].z, (int)cf[b][j].w, 0, 0, 0, 0};
        const i32x8 y = {(int)rf[b][i].x, (int)rf[b][i].y, (int)rf[b][i].z, (int)rf[b][i].w, 0, 0, 0, 0};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, acc[i][j], 4, 4, s, cs[j], s, rs[i]);
      } else {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, cf[b][j]),
                                                            __builtin_bit_cast(bf16x8, rf[b][i]), acc[i][j], 0, 0, 0);
      }
      f(nc);
    });
  };
  auto keep_scales = [&]() MX_INLINE {
    if constexpr (T::FP4) {
#pragma unroll
      for (int j = 0; j < CB; ++j) cs[j] = cn[j];
#pragma unroll
      for (int i = 0; i < RB; ++i) rs[i] = rn[i];
    }
  };
  // step s with the fragments of (slot, s1) read between its products, the first ones first, and loads J0 .. J1 - 1 of the
  // next stage into `into`: neither the LDS nor the memory pipeline holds the wave up while the matrix unit is free.  The
  // scheduling barriers keep this order: without them the products sink into one run behind all the reads.
  auto step = [&](auto sc, int slot, auto s1c, int into, auto j0c, auto j1c) MX_INLINE {
    constexpr int s1 = decltype(s1c)::value, J0 = decltype(j0c)::value, J = decltype(j1c)::value - J0;
    constexpr int R = F < P ? 1 : (F + P - 1) / P;  // reads after a product
    mma(sc, [&](auto nc) MX_INLINE {
      constexpr int n = decltype(nc)::value, a = n * J / P, e = (n + 1) * J / P;
      __builtin_amdgcn_sched_barrier(0);
      mx_each<R>([&](auto i) MX_INLINE {
        constexpr int f = n * R + decltype(i)::value;
        if constexpr (f < F) load1(slot, s1, s1 & 1, std::integral_constant<int, f>{});
      });
      if constexpr (s1 == 0 && n == P - 1) load_scales(slot, cn, rn);
      mx_each<e - a>([&](auto i) MX_INLINE { issue1(into, std::integral_constant<int, J0 + a + decltype(i)::value>{}); });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;
  using S3 = std::integral_constant<int, 3>;

  // ---- main loop: stage t in slot (t - t0) % S.  A step's fragments are read during the step before.  The barrier that
  // publishes stage t stands before the last step of stage t - 1, whose reads are done, so that its slot is free for the
  // stage S ahead, requested during that step and the next.
  if (t0 < t1) {
#pragma unroll
    for (int s = 0; s < S; ++s) issue(s, J0{}, JL{}), advance();
    wait_stages(t1 - t0 - 1 < S - 1 ? t1 - t0 - 1 : S - 1);
    lds_barrier();
    load(0, 0, 0);
    load_scales(0, cs, rs);
    step(S0{}, 0, S1{}, 0, J0{}, J0{});
    step(S1{}, 0, S2{}, 0, J0{}, J0{});
    step(S2{}, 0, S3{}, 0, J0{}, J0{});
    int slot = 0, t = t0 + 1;
    for (const int whole = t1 - (T::UNIT != tail && t1 == total ? 1 : 0); it < whole; ++t) {
      const int next = slot == S - 1 ? 0 : slot + 1;
      wait_vmcnt<(S - 2) * T::LPT>();
      lds_barrier();
      step(S3{}, next, S0{}, slot, J0{}, JH{});
      keep_scales();
      step(S0{}, next, S1{}, slot, JH{}, JL{});
      advance();
      step(S1{}, next, S2{}, 0, J0{}, J0{});
      step(S2{}, next, S3{}, 0, J0{}, J0{});
      slot = next;
    }
    for (; t < t1; ++t) {  // the last stages, and one that the reduction ends in
      const int next = slot == S - 1 ? 0 : slot + 1;
      wait_stages(t1 - 1 - t < S - 2 ? t1 - 1 - t : S - 2);
      lds_barrier();
      issue(slot, J0{}, JL{});
      advance();
      step(S3{}, next, S0{}, 0, J0{}, J0{});
      keep_scales();
      step(S0{}, next, S1{}, 0, J0{}, J0{});
      step(S1{}, next, S2{}, 0, J0{}, J0{});
      step(S2{}, next, S3{}, 0, J0{}, J0{});
      slot = next;
    }
    mma(S3{}, [](auto) MX_INLINE {});
    __syncthreads();  // every wave is done with the ring
  }

  // ---- epilogue: each wave parks 32 rows at a time in its part of the ring and stores them as runs of 8 columns; those
  // of the largest tile pass by the L2, which the operands need (16384 x 8192 -> 8192: 539 us with plain stores, 504 so)
  MxOut o = p.out;
  if (gridDim.y > 1) o.y = static_cast<float*>(o.y) + blockIdx.y * p.partial;
  float* park = reinterpret_cast<float*>(sm) + wave * 32 * CB * 32;
  constexpr int LPR = CB * 4, RPI = 64 / LPR;  // lanes a row, rows a pass
  // chunks of four values; a lane writes one of each of 16 rows: over the 256 bytes that the banks span
  auto place = [&](int row, int chunk) MX_INLINE {
    return row * CB * 32 + ((chunk ^ (CB == 1 ? (row >> 1) & 7 : CB % 2 == 0 ? row & 15 : row & 7)) << 2);
  };
  const int qc = lane % LPR;
  const int64_t n = c0 + wc * CB * 32 + qc * 8;
  float bias[8] = {};
  if (o.bias && n < o.cols) mx_load8(o.bias, o.bias_dtype, n, o.cols - n < 8 ? (int)(o.cols - n) : 8, bias);
  mx_each<RB>([&](auto ic) MX_INLINE {
    constexpr int i = decltype(ic)::value;
#pragma unroll
    for (int j = 0; j < CB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<float4*>(park + place(col, j * 8 + 2 * e + g)) =
            make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]);
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (int u = 0; u < (32 + RPI - 1) / RPI; ++u) {
      const int row = u * RPI + lane / LPR;
      if (64 % LPR != 0 && (lane >= RPI * LPR || row >= 32)) continue;
      const float4 a = *reinterpret_cast<const float4*>(park + place(row, 2 * qc));
      const float4 b = *reinterpret_cast<const float4*>(park + place(row, 2 * qc + 1));
      float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      const int64_t m = r0 + (wr * RB + i) * 32 + row;
      if (m < p.rows && n < o.cols) mx_store8<T::BR == 256>(o, m, n, v, bias);
    }
    __builtin_amdgcn_wave_barrier();
  });
}

// The slices of a split reduction, [splits, rows, pitch] fp32, added in their order.  Two slices of 2304 x 768, 14 MB in and
// 7 MB out, take 6.4 us, of which a launch that moves next to nothing takes 4 in the same trace.
static __global__ __launch_bounds__(256) void mx_reduce_kernel(const float* part, int64_t slice, int splits, int64_t rows,
                                                               int64_t pitch, MxOut o) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= rows * pitch) return;
  const int64_t m = i / pitch, n = i - m * pitch;
  float v[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float4* q = reinterpret_cast<const float4*>(part + s * slice + i);
    const float4 a = q[0], b = q[1];
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
  float bias[8] = {};
  if (n >= o.cols) return;
  if (o.bias) mx_load8(o.bias, o.bias_dtype, n, o.cols - n < 8 ? (int)(o.cols - n) : 8, bias);
  mx_store8<false>(o, m, n, v, bias);
}

// How a product is cut: the tile (0: 256 x 256, 1: 128 x 128, 2: 64 x 64, 3: 256 x 192) and the slices of its reduction.
struct MxPlan {
  int tile, splits;
  double us;  // estimated
};

inline int64_t mx_pad8(int64_t n) { return (n + 7) / 8 * 8; }
// Rows of scales that whole tiles of any size read.
inline int64_t mx_scale_rows(int64_t n) {
  const int64_t a = (n + 255) / 256 * 256, b = (n + 191) / 192 * 192;
  return a > b ? a : b;
}
// Rows and columns of a product at most: a stage of scales, 8 bytes for each of mx_scale_rows, stays below 2^31 bytes, the
// tile kernel's 32-bit step.
constexpr int64_t kMxMaxRows = (1 << 28) - 256;
inline int64_t mx_tiles(int tile, int64_t rows, int64_t cols) {
  const int64_t r = tile == 3 ? 256 : 256 >> tile, c = tile == 3 ? 192 : 256 >> tile;
  return ((rows + r - 1) / r) * ((cols + c - 1) / c);
}
inline int64_t mx_partial_bytes(const MxPlan& pl, int64_t rows, int64_t cols) {
  return pl.splits > 1 ? pl.splits * rows * mx_pad8(cols) * 4 : 0;
}

// Whether the 128 tile takes a ring of four slots, which leaves a CU room for one work-group only: where no CU has two and
// the reduction is long enough to fill it (515 x 4096 summed over 4096, 160 work-groups: 40.9 us with two slots, 29.5 with
// four; 64 x 4096 codes over 4096, 32 of them: 12.2 and 12.8).
inline bool mx_deep(const MxPlan& pl, int64_t rows, int64_t cols, int64_t stages) {
  return mx_tiles(1, rows, cols) * pl.splits <= 256 && stages >= 24 * pl.splits;
}

// The plan of the least estimated time, in us on a card of 256 CUs.  A stage of the two large tiles, one work-group a CU,
// takes a + b times the share of the CUs at work (the clock falls as more of them do); one of the small tiles the larger
// of its latency and its share where n run on a CU.  A tile adds its filling and epilogue; slices add a launch and their
// bytes at 5 TB/s.  Measured on products of 16 to 16,384 rows, bf16 ones in both gradients; over 146 products with 4 to 25
// plans measured each, the choice is 0.5 % slower than the best one in the mean, 20 % at worst (64 rows summed).
inline MxPlan mx_plan(bool fp4, int64_t rows, int64_t cols, int64_t stages) {
  MxPlan best{2, 1, 1e300};
  for (int tile = 0; tile < 4; ++tile) {
    for (const int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (splits > 1 && stages < 4 * splits) break;
      const int64_t groups = mx_tiles(tile, rows, cols) * splits, n = (groups + 255) / 256;
      const double each = (double)((stages + splits - 1) / splits), busy = groups < 256 ? groups / 256.0 : 1.0;
      double us;
      if (tile == 0) {
        us = n * (each * (fp4 ? 1.0 + 1.0 * busy : 0.9 + 0.75 * busy) + 8.0);
      } else if (tile == 3) {
        us = n * (each * (fp4 ? 0.85 + 0.8 * busy : 0.7 + 0.62 * busy) + 7.0);
      } else {
        const bool deep = tile == 1 && mx_deep({1, splits, 0}, rows, cols, stages);
        const double alone = deep ? (fp4 ? 0.55 : 0.42) : tile == 1 ? (fp4 ? 0.73 : 0.60) : (fp4 ? 0.41 : 0.24);
        const double share = n * (tile == 1 ? (fp4 ? 0.60 : 0.465) : (fp4 ? 0.25 : 0.20));
        us = each * (alone > share ? alone : share) + n * (tile == 1 ? 2.8 : 0.8);
      }
      if (splits > 1) us += 4.0 + (double)splits * rows * cols * 8 / 5e6;
      if (us < best.us) best = MxPlan{tile, splits, us};
    }
  }
  return best;
}

// Slices and the kernel's number (include/dimq_hip.h, dimq_mx_linear_route).
inline int mx_route(const MxPlan& pl, int64_t rows, int64_t cols, int64_t stages) {
  const int kernel = pl.tile == 0 ? 1 : pl.tile == 3 ? 2 : pl.tile == 2 ? 5 : mx_deep(pl, rows, cols, stages) ? 4 : 3;
  return pl.splits * 8 + kernel;
}

template <class T>
int mx_mm_launch(const MxMm& p, int splits, hipStream_t s, const char* what) {
  const int64_t tiles = ((p.rows + T::BR - 1) / T::BR) * ((p.cols + T::BC - 1) / T::BC);
  DIMQ_CHECK(tiles < (1ll << 31), "%s: too many outputs", what);
  mx_mm_kernel<T><<<dim3((unsigned)tiles, (unsigned)splits), T::NT, 0, s>>>(p);
  return check_launch(what);
}

template <bool FP4, bool CT, bool RT>
int mx_mm(MxMm p, const MxPlan& pl, float* partial, hipStream_t s, const char* what) {
  // a lane's offsets inside a tile and a stage's step are 32 bits
  DIMQ_CHECK(p.len * p.planes < (1ll << 31) && p.rows <= kMxMaxRows && p.cols <= kMxMaxRows, "%s: too large", what);
  DIMQ_CHECK(p.r.ld < (1 << 23) && p.c.ld < (1 << 23), "%s: rows beyond 8 MB are not supported", what);
  const MxOut out = p.out;
  if (pl.splits > 1) {
    p.partial = p.rows * mx_pad8(p.cols);
    p.out = MxOut{partial, DIMQ_F32, mx_pad8(p.cols), p.cols, nullptr, 0, nullptr, 0, 0};
  }
  const int64_t unit = FP4 ? 8 : 64, stages = (p.len + unit - 1) / unit * p.planes;
  int rc;
  switch (pl.tile) {
    case 0: rc = mx_mm_launch<MxTile<FP4, CT, RT, 4, 2, 2, 4, 2>>(p, pl.splits, s, what); break;
    case 3: rc = mx_mm_launch<MxTile<FP4, CT, RT, 4, 2, 2, 3, 2>>(p, pl.splits, s, what); break;
    case 1:
      if (mx_deep(pl, p.rows, p.cols, stages)) rc = mx_mm_launch<MxTile<FP4, CT, RT, 2, 2, 2, 2, 4>>(p, pl.splits, s, what);
      else rc = mx_mm_launch<MxTile<FP4, CT, RT, 2, 2, 2, 2, 2>>(p, pl.splits, s, what);
      break;
    default: rc = mx_mm_launch<MxTile<FP4, CT, RT, 2, 2, 1, 1, 3>>(p, pl.splits, s, what);
  }
  if (rc != DIMQ_OK || pl.splits == 1) return rc;
  const int64_t pitch = mx_pad8(p.cols), groups = p.rows * pitch / 8;
  DIMQ_CHECK((groups + 255) / 256 < (1ll << 31), "%s: too many outputs", what);
  mx_reduce_kernel<<<dim3((unsigned)((groups + 255) / 256)), 256, 0, s>>>(partial, p.rows * pitch, pl.splits, p.rows, pitch,
                                                                          out);
  return check_launch(what);
}

#endif  // __HIPCC__

}  // namespace dimq
