// Linear layers on 4-bit weights with a scale (and a zero point) per group of a row's elements:
//
//   y[m, n] = act( c[m] sum_g s[n, g] ( sum_{k in g} q[n, k] x[m, k] - z[n, g] sum_{k in g} x[m, k] ) + b[n] + r[m, n] )
//
// q in 0..15, two a byte, the earlier element in the low half, rows padded to whole blocks of 32; z 8 where none are given;
// x in fp32, fp16, bf16, or in e4m3 with a scale c per row.  The products are exact and the sums fp32: the codes go to the
// matrix instructions as integers and a group's scale multiplies its sum, so neither x nor the weights are rounded.
//
// A code's byte 0000qqqq is the e4m3 number q 2^-9 (its subnormals end at 7, and q - 8 is the mantissa from 8 on), so one
// conversion a pair makes bf16 or fp16 numbers of them.  sum x of a group comes from the same instructions against ones.  An
// fp32 x is the sum of three bf16 numbers of 8 bits each; e4m3 rows are converted to bf16 (exactly).  The e4m3 matrix
// instructions would take these rows and the bytes as they are, at twice the rate, but they cut addends off below the
// largest: against 64 bits, sums of 32 products were up to 4,700 2^-24 of their terms' magnitudes off, in bf16 0.1.
//
// Which 32 k of an instruction's share a lane holds is free as long as both operands agree: lane l (column or row l % 16,
// quarter l / 16) takes 2 LB consecutive k of a "span" of 8 LB, whose codes are LB bytes.  A span lies in one group:
// LB 16 for groups of multiples of 128, 8 for other multiples of 64, 4 for other multiples of 32.
#include "decode.h"

#include <type_traits>

namespace dimq {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct GroupArgs {
  const void* x;
  int64_t M, K, ldx;
  const float* xs;        // e4m3: scale per row
  int vec;                // x rows 16-byte aligned
  const uint8_t* codes;   // [N, 16 blocks]
  int64_t pitch, nb;      // bytes and blocks of a row
  const void* scales;     // [N, groups]
  int s_dt;
  const uint8_t* zeros;   // [N, groups], nullable: 8
  int64_t group, groups;
  int64_t N;
  const void* bias;
  int bias_dt;
  void* y;
  int y_dt;
  Epi epi;
  // tiles
  int64_t plane;          // bytes between the planes of x
  int64_t ksteps;         // of 128
  int splits;
  float* part;            // [splits][M][N]
  int64_t tiles_m, tiles_n;
  int64_t span_blocks;    // blocks of 32 spans
  uint32_t prep_first;    // work-groups of the first launch that prepare s z
  const uint8_t* sums;    // the zero points' product
  const uint8_t* szs;
};

constexpr int x_size(int xt) { return xt == DIMQ_F32 ? 4 : xt == DIMQ_E4M3 ? 1 : 2; }
// Type that the matrix instructions take (a lane's share of a span is LB dwords of it), and planes of x in it.
constexpr int mul_type(int xt) { return xt == DIMQ_F16 ? DIMQ_F16 : DIMQ_BF16; }
constexpr int planes_of(int xt) { return xt == DIMQ_F32 ? 3 : 1; }

// Eight codes as bytes in their order.
__device__ __forceinline__ void code_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  lo = perm(odd, even, 0x05010400u);
  hi = perm(odd, even, 0x07030602u);
}

// Two e4m3 bytes (the low or the high pair) times `by`, a power of two, as two MT numbers.
template <int MT, bool HIGH>
__device__ __forceinline__ uint32_t code_pair(uint32_t bytes, float by) {
  if constexpr (MT == DIMQ_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, by, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, by, HIGH));
}

// Eight codes as one step's operand, and a lane's codes of a span.
template <int MT>
__device__ __forceinline__ void decode_step(uint32_t codes, uint32_t (&b)[4]) {
  uint32_t lo, hi;
  code_bytes(codes, lo, hi);
  b[0] = code_pair<MT, false>(lo, 512.0f);
  b[1] = code_pair<MT, true>(lo, 512.0f);
  b[2] = code_pair<MT, false>(hi, 512.0f);
  b[3] = code_pair<MT, true>(hi, 512.0f);
}
template <int MT, int LB>
__device__ __forceinline__ void decode_span(const uint32_t (&codes)[LB / 4], uint32_t (&b)[LB]) {
#pragma unroll
  for (int j = 0; j < LB / 4; ++j) {
    uint32_t s[4];
    decode_step<MT>(codes[j], s);
#pragma unroll
    for (int i = 0; i < 4; ++i) b[4 * j + i] = s[i];
  }
}

// acc + the products of step j of a span, and of all of it.
template <int MT, int LB>
__device__ __forceinline__ floatx4 mul_step(const uint32_t (&a)[LB], const uint32_t (&b)[LB], int j, floatx4 acc) {
  const u32x4 u = {a[4 * j], a[4 * j + 1], a[4 * j + 2], a[4 * j + 3]};
  const u32x4 v = {b[4 * j], b[4 * j + 1], b[4 * j + 2], b[4 * j + 3]};
  if constexpr (MT == DIMQ_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u), __builtin_bit_cast(bf16x8, v), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, u), __builtin_bit_cast(half8, v), acc, 0, 0, 0);
}
template <int MT, int LB>
__device__ __forceinline__ floatx4 mul_span(const uint32_t (&a)[LB], const uint32_t (&b)[LB], floatx4 acc) {
#pragma unroll
  for (int j = 0; j < LB / 4; ++j) acc = mul_step<MT, LB>(a, b, j, acc);
  return acc;
}

// Products against ones.
template <int MT, int LB>
__device__ __forceinline__ floatx4 sum_span(const uint32_t (&a)[LB], floatx4 acc) {
  uint32_t b[LB];
#pragma unroll
  for (int i = 0; i < LB; ++i) b[i] = MT == DIMQ_BF16 ? 0x3f803f80u : 0x3c003c00u;
  return mul_span<MT, LB>(a, b, acc);
}

// Scales without a branch on their type: the aligned dword that holds scale i, and the scale of it.
struct Scales {
  const uint32_t* base;
  uint32_t wide, odd, f16;  // odd: the first 16-bit scale is its dword's second half
  __device__ __forceinline__ Scales(const void* scales, int dt, int64_t first) {
    wide = dt == DIMQ_F32, f16 = dt == DIMQ_F16;
    const uintptr_t at = reinterpret_cast<uintptr_t>(scales) + (first << (1 + wide));
    base = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
    odd = static_cast<uint32_t>(at >> 1) & 1;
  }
  template <class I>
  __device__ __forceinline__ I index(I i) const { return wide ? i : (i + odd) >> 1; }
  template <class I>
  __device__ __forceinline__ uint32_t load(I i) const { return base[index(i)]; }
  // low: the lowest bits of i
  __device__ __forceinline__ float value(uint32_t raw, uint32_t low) const {
    const uint32_t half = ((low + odd) & 1) ? raw >> 16 : raw & 0xffffu;
    return f16 ? f16_bits_to_float(half) : __uint_as_float(wide ? raw : half << 16);
  }
};

// Eight fp32 numbers as three planes of bf16 that add up to them (cut off, not rounded: nothing overflows).  An infinity
// is in the first plane alone; a NaN is in the second, whatever the first plane's cut makes of it.
__device__ __forceinline__ void split3(const uint32_t (&v)[8], uint32_t (&hi)[4], uint32_t (&mid)[4], uint32_t (&lo)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = v[2 * j + i];
      const float x = __uint_as_float(u), r = x - __uint_as_float(u & 0xffff0000u);
      const uint32_t t = (u & 0x7fffffffu) == 0x7f800000u ? 0u : __float_as_uint(r);
      m[i] = t;
      // a NaN stays in the second plane alone
      l[i] = (t & 0x7f800000u) == 0x7f800000u ? 0u : __float_as_uint(__uint_as_float(t) - __uint_as_float(t & 0xffff0000u));
      if ((t & 0x7f800000u) == 0x7f800000u) m[i] = 0x7fc00000u;
    }
    hi[j] = perm(v[2 * j + 1], v[2 * j], 0x07060302u);
    mid[j] = perm(m[1], m[0], 0x07060302u);
    lo[j] = perm(l[1], l[0], 0x07060302u);
  }
}

// The raw bytes of elements k0 .. k0 + 2 LB - 1 of row m; those from K on are 0.
template <int XT, int LB>
struct RawX {
  static constexpr int kDwords = 2 * LB * x_size(XT) / 4;
  uint32_t w[kDwords];
  __device__ __forceinline__ void load(const GroupArgs& p, int64_t m, int64_t k0, bool fast) {
    const char* at = static_cast<const char*>(p.x) + (m * p.ldx + k0) * x_size(XT);
    if (fast) {
      if constexpr (kDwords % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kDwords / 4; ++i) {
          const uint4 t = reinterpret_cast<const uint4*>(at)[i];
          w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
        }
      } else {
        const uint2 t = *reinterpret_cast<const uint2*>(at);
        w[0] = t.x, w[1] = t.y;
      }
      return;
    }
    constexpr int kPer = 4 / x_size(XT);
#pragma unroll
    for (int i = 0; i < kDwords; ++i) {
      uint32_t v = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int64_t k = k0 + i * kPer + e;
        if (k >= p.K) continue;
        const char* q = at + (i * kPer + e) * x_size(XT);
        if constexpr (x_size(XT) == 4) v = *reinterpret_cast<const uint32_t*>(q);
        else if constexpr (x_size(XT) == 2) v |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(q)) << (16 * e);
        else v |= static_cast<uint32_t>(*reinterpret_cast<const uint8_t*>(q)) << (8 * e);
      }
      w[i] = v;
    }
  }
  __device__ __forceinline__ void planes(uint32_t (&a)[planes_of(XT)][LB]) const {
    if constexpr (XT == DIMQ_F32) {
#pragma unroll
      for (int j = 0; j < LB / 4; ++j) {
        uint32_t v[8], o[3][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = w[8 * j + i];
        split3(v, o[0], o[1], o[2]);
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) a[q][4 * j + i] = o[q][i];
      }
    } else if constexpr (XT == DIMQ_E4M3) {
#pragma unroll
      for (int i = 0; i < kDwords; ++i) {
        a[0][2 * i] = code_pair<DIMQ_BF16, false>(w[i], 1.0f);
        a[0][2 * i + 1] = code_pair<DIMQ_BF16, true>(w[i], 1.0f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kDwords; ++i) a[0][i] = w[i];
    }
  }
};

__device__ __forceinline__ uint32_t lds_address(uint8_t* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)p));
}

__device__ __forceinline__ float row_scale(const GroupArgs& p, int64_t m) { return p.xs ? p.xs[m] : 1.0f; }

// Output (m, n) of a complete sum.
__device__ __forceinline__ void put_output(const GroupArgs& p, int64_t m, int64_t n, float v) {
  if (p.bias) v += load_as_float(p.bias, p.bias_dt, n);
  const int64_t off = m * p.N + n;
  store_from_float(p.y, p.y_dt, off, epi1(p.epi, off, v));
}

// Outputs off .. off + left - 1 of one row, their bias in them already.
__device__ __forceinline__ void put8(const GroupArgs& p, int64_t off, int left, float (&v)[8]) {
  if (p.epi.res) {
    for (int j = 0; j < 8; ++j)
      if (j < left) v[j] += load_as_float(p.epi.res, p.epi.res_dt, off + j);
  }
  if (p.epi.act) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = act_apply(v[j], p.epi.act);
  }
  if (left == 8) {  // 16 bytes to a multiple of the element's size
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
    if (p.y_dt == DIMQ_F32) {
      u4* to = reinterpret_cast<u4*>(static_cast<float*>(p.y) + off);
      to[0] = u4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      to[1] = u4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
    } else {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = p.y_dt == DIMQ_F16 ? f16x2_rne(v[2 * j], v[2 * j + 1]) : bf16x2_rne(v[2 * j], v[2 * j + 1]);
      *reinterpret_cast<u4*>(static_cast<uint16_t*>(p.y) + off) = u4{o[0], o[1], o[2], o[3]};
    }
    return;
  }
  for (int j = 0; j < 8; ++j)
    if (j < left) store_from_float(p.y, p.y_dt, off + j, v[j]);
}

// ---- few rows -----------------------------------------------------------------------------------------------------
// 16 MT rows by 16 NC columns a work-group; its 8 waves share out the k in turns of 128, and their sums meet in the LDS.  Codes
// come by 16 bytes a lane whatever the spans; shorter ones are dealt out among a column's four lanes by swaps of their rows.
// A wave takes its turns one after another: what hides their loads is the other waves of the CU (two turns' loads sent out
// together gained nothing at 4096 -> 4096, the next turn loaded ahead lost 2 to 30 %, for its registers; 16 waves are 0 to 3 %
// slower, in fp32 up to 60 %).  16 x 4096 -> 12288, e4m3, groups of 128: 13.7 us (27 MB, 2 TB/s).
// Lanes whose row is past M load no x: their sums are not stored.
constexpr int kFewWaves = 8;

// Rows of 16 lanes: (a0 b0 a2 b2), (a1 b1 a3 b3), and (a0 a1 b0 b1), (a2 a3 b2 b3).
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
// A lane's 16 bytes of a turn's 64, quarter after quarter, to the LB bytes of each of its 16 / LB spans that the lane takes.
template <int LB>
__device__ __forceinline__ void to_spans(uint32_t (&w)[4]) {
  if constexpr (LB == 8) swap32(w[0], w[2]), swap32(w[1], w[3]);
  if constexpr (LB == 4) swap16(w[0], w[1]), swap16(w[2], w[3]), swap32(w[0], w[2]), swap32(w[1], w[3]);
}
// What the quarters hold of a turn's spans (LB 8: of the first span in the first two) to every lane.
template <int LB>
__device__ __forceinline__ void to_lanes(uint32_t v, uint32_t (&o)[16 / LB]) {
#pragma unroll
  for (int i = 0; i < 16 / LB; ++i) o[i] = v;
  if constexpr (LB == 8) swap32(o[0], o[1]);
  if constexpr (LB == 4) swap16(o[0], o[1]), swap16(o[2], o[3]), swap32(o[0], o[2]), swap32(o[1], o[3]);
}

template <int XT, int LB, int MT, int NC>
__global__ __launch_bounds__(64 * kFewWaves) void group_few_kernel(const GroupArgs p) {
  constexpr int ML = mul_type(XT), P = planes_of(XT), SP = 8 * LB, S = 16 / LB;
  __shared__ floatx4 red[kFewWaves][MT * NC][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quarter = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NC), m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const int turns = static_cast<int>((p.nb + 3) / 4), each = (turns + kFewWaves - 1) / kFewWaves;
  const int from = wave * each, to = from + each < turns ? from + each : turns;
  const uint32_t group_spans = static_cast<uint32_t>(p.group / SP), last = static_cast<uint32_t>(p.groups - 1);
  const int mine = LB == 4 ? quarter : LB == 8 ? quarter >> 1 : 0;  // the span whose scale the lane loads
  const int xat = LB == 8 ? (quarter & 1) * 32 + (quarter >> 1) * 16 : quarter * (2 * LB);  // the lane's first k of a span
  const uint8_t* cw[NC];
  int64_t gn[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t n = n0 + 16 * c + col < p.N ? n0 + 16 * c + col : p.N - 1;
    cw[c] = p.codes + n * p.pitch;
    gn[c] = n * p.groups;
  }
  const Scales scales(p.scales, p.s_dt, 0);
  const uint8_t* zeros = p.zeros ? p.zeros : p.codes;  // as long, and not used then
  floatx4 acc[MT][NC];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[t][c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int turn = from; turn < to; ++turn) {
    // a lane's codes past the row's last block are that block's (x is 0 there), scales past the last group that group's
    int64_t at = static_cast<int64_t>(turn) * 64 + quarter * 16;
    if (at + 16 > p.pitch) at = p.pitch - 16;
    uint32_t codes[NC][4], rs[NC], z[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint4 w = *reinterpret_cast<const uint4*>(cw[c] + at);
      codes[c][0] = w.x, codes[c][1] = w.y, codes[c][2] = w.z, codes[c][3] = w.w;
    }
    RawX<XT, LB> rx[MT][S];
    const int64_t k0 = static_cast<int64_t>(turn) * 128 + xat;
    const bool fast = p.vec && static_cast<int64_t>(turn + 1) * 128 <= p.K;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int64_t m = m0 + 16 * t + col;
      if (m < p.M) {
#pragma unroll
        for (int s = 0; s < S; ++s) rx[t][s].load(p, m, k0 + s * SP, fast);
      }
    }
    uint32_t g = (static_cast<uint32_t>(turn) * S + mine) / group_spans;
    g = g < last ? g : last;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      rs[c] = scales.load(gn[c] + g);
      z[c] = zeros[gn[c] + g];
    }
    uint32_t sv[NC][S], zv[NC][S];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      to_spans<LB>(codes[c]);
      to_lanes<LB>(__float_as_uint(scales.value(rs[c], static_cast<uint32_t>(gn[c]) + g)), sv[c]);
      to_lanes<LB>(__float_as_uint(p.zeros ? static_cast<float>(z[c]) : 8.0f), zv[c]);
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      uint32_t b[NC][LB];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t part[LB / 4];
#pragma unroll
        for (int i = 0; i < LB / 4; ++i) part[i] = codes[c][s * (LB / 4) + i];
        decode_span<ML, LB>(part, b[c]);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uint32_t a[P][LB];
        rx[t][s].planes(a);
        floatx4 x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < P; ++i) x = sum_span<ML, LB>(a[i], x);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          floatx4 q = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < P; ++i) q = mul_span<ML, LB>(a[i], b[c], q);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[t][c][i] = fmaf(__uint_as_float(sv[c][s]), fmaf(-__uint_as_float(zv[c][s]), x[i], q[i]), acc[t][c][i]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int c = 0; c < NC; ++c) red[wave][t * NC + c][lane] = acc[t][c];
  __syncthreads();
  for (int tile = wave; tile < MT * NC; tile += kFewWaves) {
    const int64_t n = n0 + 16 * (tile % NC) + col;
    floatx4 v = red[0][tile][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) v += red[w][tile][lane];
    if (n >= p.N) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + 16 * (tile / NC) + 4 * quarter + i;
      if (m < p.M) put_output(p, m, n, v[i] * row_scale(p, m));
    }
  }
}

// ---- many rows ----------------------------------------------------------------------------------------------------
// The zero points' part of the product, sum_g s z sum_{k in g} x, is a product of its own with a reduction 8 LB times
// shorter: a first launch sums x over each span (and copies x where its rows are not whole k steps, aligned and of 16 bits),
// and after the main loop those sums and s z, each as three bf16 parts, go through the matrix instructions once.  Against
// ones in the loop the sums cost a fifth of its matrix instructions, and taken off each span's product half of its fmas.
//
// Then 128 x 256 outputs a work-group of 8 waves of 64 x 64 each.  A k step is 128: x of the 128 rows, the columns' codes and
// scales come into a ring of three slots in the LDS by direct loads, two steps ahead, and the codes are decoded behind the
// LDS.  No other load is in the loop, so the kernel's own counted wait is the only one.  With 128 x 128 tiles, two slots and
// two work-groups a CU the waves stood a third of the time at the barrier.
// Measured at 2048 x 4096 -> 4096, bf16, groups of 128: 85 us with all launches (804 TFLOP/s; the first one 7.4), 150 with the
// smaller tiles; the library's product of bf16 weights of that size takes 62.
constexpr int kTileM = 128, kTileN = 256, kTileK = 128, kTileThreads = 512;
constexpr int kSlots = 3;

// i / per, in 32 bits where they do (a 64-bit division is a hundred instructions).
__device__ __forceinline__ int64_t quotient(int64_t i, uint32_t per) {
  return i <= 0xffffffffll ? static_cast<int64_t>(static_cast<uint32_t>(i) / per) : i / per;
}

// Both operands of the zero points' product: [row][blocks of 32 spans][3 parts][32 spans] in bf16, zeros behind the last span.
constexpr int kPartBytes = 3 * 32 * 2;  // of a block
constexpr int kPrepEach = 4;            // pieces of 8 elements of x a thread

// sums: x's, [M]; szs: -s z, [N]; out (nullable): x padded with zeros to whole k steps, [planes][M][ksteps 128].
template <int XT, int LB>
__global__ __launch_bounds__(256) void group_prep_kernel(const GroupArgs p, uint8_t* out, uint8_t* sums, uint8_t* szs) {
  constexpr int SP = 8 * LB;
  const int64_t blocks = p.span_blocks;
  if (blockIdx.x < p.prep_first) {  // 8 spans a thread
    const Scales scales(p.scales, p.s_dt, 0);
    const uint32_t group_spans = static_cast<uint32_t>(p.group / SP), per = static_cast<uint32_t>(blocks) * 4;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= p.N * per) return;
    const int64_t n = quotient(i, per);
    const uint32_t first = static_cast<uint32_t>(i - n * per) * 8;
    uint32_t v[8], o[3][4];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t g = (first + e) / group_spans;
      const int64_t at = n * p.groups + (g < p.groups ? g : p.groups - 1);
      const float sz = -scales.value(scales.load(at), static_cast<uint32_t>(at)) * static_cast<float>(p.zeros ? p.zeros[at] : 8u);
      v[e] = g < p.groups ? __float_as_uint(sz) : 0u;
    }
    split3(v, o[0], o[1], o[2]);
    uint8_t* to = szs + (n * blocks + first / 32) * kPartBytes + first % 32 * 2;
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(to + q * 64) = make_uint4(o[q][0], o[q][1], o[q][2], o[q][3]);
    return;
  }
  const uint32_t per = static_cast<uint32_t>(blocks) * (32 * SP / 8);  // a multiple of 16: 16 neighbouring lanes share a row
  const int64_t total = p.M * per, kp = p.ksteps * kTileK, base = static_cast<int64_t>(blockIdx.x - p.prep_first) * (256 * kPrepEach);
  RawX<XT, 4> r[kPrepEach];
  int64_t m[kPrepEach], k0[kPrepEach];
#pragma unroll
  for (int e = 0; e < kPrepEach; ++e) {
    const int64_t i = base + e * 256 + threadIdx.x;
    m[e] = i < total ? quotient(i, per) : p.M;
    k0[e] = i - m[e] * per;
    k0[e] *= 8;
    if (m[e] < p.M) r[e].load(p, m[e], k0[e], p.vec && k0[e] + 8 <= p.K);
  }
#pragma unroll
  for (int e = 0; e < kPrepEach; ++e) {
    if (m[e] >= p.M) return;  // with its 16 neighbours
    uint32_t a[planes_of(XT)][4];
    r[e].planes(a);
    if (out && k0[e] < kp) {
#pragma unroll
      for (int q = 0; q < planes_of(XT); ++q)
        *reinterpret_cast<uint4*>(out + q * p.plane + (m[e] * kp + k0[e]) * 2) = make_uint4(a[q][0], a[q][1], a[q][2], a[q][3]);
    }
    float s = 0.0f;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if constexpr (XT == DIMQ_F32) s += __uint_as_float(r[e].w[q]);
      else if constexpr (XT == DIMQ_F16) s += f16_bits_to_float((r[e].w[q >> 1] >> (16 * (q & 1))) & 0xffffu);
      else s += bf16_bits_to_float((a[0][q >> 1] >> (16 * (q & 1))) & 0xffffu);
    }
#pragma unroll
    for (int w = 1; w < LB; w *= 2) s += __shfl_xor(s, w, 64);
    if ((threadIdx.x & (LB - 1)) == 0) {
      const uint32_t v[8] = {__float_as_uint(s), 0, 0, 0, 0, 0, 0, 0};
      uint32_t o[3][4];
      split3(v, o[0], o[1], o[2]);
      const int64_t span = k0[e] / SP;
      uint8_t* to = sums + (m[e] * blocks + span / 32) * kPartBytes + span % 32 * 2;
#pragma unroll
      for (int q = 0; q < 3; ++q) *reinterpret_cast<uint16_t*>(to + q * 64) = static_cast<uint16_t>(o[q][0]);
    }
  }
}

// 16 bytes a lane from base (the same in all lanes) + off into the LDS at lds + 16 lane.  Inline, as dma16 (common.h), so
// that the waits are the kernel's: the load must not follow a vector instruction that wrote its scalar address (a
// readfirstlane, or a spilled register's v_readlane) by fewer than five wait states, which the compiler does not see to here.
__device__ __forceinline__ void group_dma16(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}

__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ void group_dma4(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}

// A span's group, counted up.
struct GroupCount {
  uint32_t g, phase, each, last;
  __device__ __forceinline__ GroupCount(uint32_t span, uint32_t group_spans, uint32_t groups)
      : g(span / group_spans), phase(span % group_spans), each(group_spans), last(groups - 1) {}
  __device__ __forceinline__ uint32_t next() {
    const uint32_t at = g < last ? g : last;  // spans behind the row's end: x is 0 there
    if (++phase == each) phase = 0, ++g;
    return at;
  }
};

// MT: type of x in the LDS; P: its planes, one after another within a k step (each a stage of its own).
template <int MT, int LB, int P>
__global__ __launch_bounds__(kTileThreads) void group_tile_kernel(const GroupArgs p) {
  constexpr int SP = 8 * LB, NS = kTileK / SP;
  constexpr int RowBytes = kTileK * 2, Chunks = RowBytes / 16;
  constexpr int XBytes = kTileM * RowBytes, CodeBytes = kTileN * 64, SlotBytes = XBytes + CodeBytes + NS * kTileN * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kSlots * SlotBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quarter = lane >> 4;
  const int wm = wave & 1, wn = wave >> 1;
  // neighbouring work-groups are on different XCDs: each XCD takes a contiguous part of the tiles, rows fastest, so that its
  // L2 holds a few columns' codes and x
  const uint32_t tiles = static_cast<uint32_t>(p.tiles_m * p.tiles_n), per = tiles / 8, rest = tiles % 8, xcd = blockIdx.x % 8;
  const uint32_t tile = xcd * per + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
  const uint32_t tm = static_cast<uint32_t>(p.tiles_m);
  const int64_t m0 = static_cast<int64_t>(tile % tm) * kTileM, n0 = static_cast<int64_t>(tile / tm) * kTileN;
  const int ksteps = static_cast<int>(p.ksteps), steps_each = (ksteps + p.splits - 1) / p.splits;
  const int step0 = blockIdx.y * steps_each, step1 = step0 + steps_each < ksteps ? step0 + steps_each : ksteps;
  const uint32_t lds0 = lds_address(lds);
  const int rows = p.M - m0 < kTileM ? static_cast<int>(p.M - m0) : kTileM;
  const int cols = p.N - n0 < kTileN ? static_cast<int>(p.N - n0) : kTileN;

  // Stage of x: a wave's load is 1 KB, 4 rows of 16 pieces; piece c of row r lies at slot c ^ (r % 16).  Offsets from the
  // tile's first row stay below 2^32 (checked on the host).  Rows and columns past the end re-read the last one.
  constexpr int kXLoads = XBytes / 1024 / 8, kCodeLoads = CodeBytes / 1024 / 8;
  uint32_t xoff[kXLoads], coff[kCodeLoads];
#pragma unroll
  for (int i = 0; i < kXLoads; ++i) {
    const int r = (wave * kXLoads + i) * 4 + lane / Chunks, c = (lane % Chunks) ^ (r % Chunks);
    xoff[i] = static_cast<uint32_t>(r < rows ? r : rows - 1) * static_cast<uint32_t>(p.ldx * 2) + c * 16;
  }
#pragma unroll
  for (int i = 0; i < kCodeLoads; ++i) {  // 64 bytes a column
    const int r = (wave * kCodeLoads + i) * 16 + lane / 4;
    coff[i] = static_cast<uint32_t>(r < cols ? r : cols - 1) * static_cast<uint32_t>(p.pitch) + lane % 4 * 16;
  }
  const uint8_t* xbase = static_cast<const uint8_t*>(p.x) + m0 * p.ldx * 2;
  const uint8_t* cbase = p.codes + n0 * p.pitch;
  // Scales come as the aligned dwords that hold them, for the 64 columns of the wave.
  const uint32_t groups = static_cast<uint32_t>(p.groups), group_spans = static_cast<uint32_t>(p.group / SP);
  const Scales scaled(p.scales, p.s_dt, n0 * p.groups);
  const uint8_t* sbase = reinterpret_cast<const uint8_t*>(scaled.base);
  const auto column = [&](int n) { return static_cast<uint32_t>(n < cols ? n : cols - 1) * groups; };
  const uint32_t sown = column(wn * 64 + lane);
  uint32_t goff[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) goff[c] = column(wn * 64 + c * 16 + col);
  GroupCount fetched(step0 * NS, group_spans, groups), used = fetched;

  constexpr int kStageLoads = kXLoads + kCodeLoads + NS;  // a wave's
  int fstep = step0, fplane = 0;
  uint32_t at[NS];
  auto fetch = [&](int slot) {
    const uint32_t to = lds0 + slot * SlotBytes;
    const uint8_t* xb = uniform(xbase + fplane * p.plane + static_cast<int64_t>(fstep) * RowBytes);
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) group_dma16(xb, xoff[i], to + (wave * kXLoads + i) * 1024);
    const uint8_t* cb = uniform(cbase + static_cast<int64_t>(fstep) * 64);
    // past the row's last block that block again (x is 0 there)
    const int over = (fstep + 1) * 64 - static_cast<int>(p.pitch), back = over > 0 ? lane % 4 * 16 + over - 48 : 0;
#pragma unroll
    for (int i = 0; i < kCodeLoads; ++i)
      group_dma16(cb, coff[i] - (back > 0 ? back : 0), to + XBytes + (wave * kCodeLoads + i) * 1024);
    if (fplane == 0) {
#pragma unroll
      for (int s = 0; s < NS; ++s) at[s] = fetched.next();
    }
#pragma unroll
    for (int s = 0; s < NS; ++s)
      group_dma4(sbase, scaled.index(sown + at[s]) * 4, to + XBytes + CodeBytes + (s * kTileN + wn * 64) * 4);
    if (++fplane == P) fplane = 0, ++fstep;
  };

  // v: the span's products, added to acc times the scale when the next span begins, so that those fmas and the span's first
  // decoding stand between its first LDS reads and their use; within a span the next step is decoded and read between the
  // matrix instructions of this one.
  constexpr int J = LB / 4;  // steps of 32 k in a span
  floatx4 acc[4][4], v[4][4];
  float scale[4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[t][c] = v[t][c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < 4; ++c) scale[c] = 0.0f;
  auto fold = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][c][i] = fmaf(scale[c], v[t][c][i], acc[t][c][i]);
  };

  const int stages = step1 > step0 ? (step1 - step0) * P : 0;
  if (stages > 0) fetch(0);
  if (stages > 1) fetch(1);
  int slot = 0, uplane = 0;
  for (int stage = 0; stage < stages; ++stage) {
    // this stage is in the LDS for all waves, and the slot of the one before is free
    if (stage + 1 < stages) wait_vmcnt<kStageLoads>();
    else wait_vmcnt<0>();
    lds_barrier();
    if (stage + 2 < stages) fetch(slot == 0 ? 2 : slot - 1);
    GroupCount span = used;
    const uint8_t* st = lds + slot * SlotBytes;
    const uint8_t* ct = st + XBytes + (wn * 64 + col) * 64 + quarter * LB;
    const uint8_t* xt = st + (wm * 64 + col) * RowBytes;
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(st + XBytes + CodeBytes) + wn * 64 + col;
#pragma unroll 1
    for (int s = 0; s < NS; ++s) {
      const uint32_t group_at = span.next();
      uint32_t codes[4][J], a[2][4][4], b[2][4][4], raw[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint8_t* q = ct + c * 1024 + s * (4 * LB);
        if constexpr (LB == 16) {
          const uint4 w = *reinterpret_cast<const uint4*>(q);
          codes[c][0] = w.x, codes[c][1] = w.y, codes[c][2] = w.z, codes[c][3] = w.w;
        } else if constexpr (LB == 8) {
          const uint2 w = *reinterpret_cast<const uint2*>(q);
          codes[c][0] = w.x, codes[c][1] = w.y;
        } else {
          codes[c][0] = *reinterpret_cast<const uint32_t*>(q);
        }
        raw[c] = scales[s * kTileN + c * 16];
      }
      auto read_x = [&](int j) __attribute__((always_inline)) {
        const int piece = ((s * SP + quarter * 2 * LB) / 8 + j) ^ col;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint4 w = *reinterpret_cast<const uint4*>(xt + t * 16 * RowBytes + (piece << 4));
          a[j & 1][t][0] = w.x, a[j & 1][t][1] = w.y, a[j & 1][t][2] = w.z, a[j & 1][t][3] = w.w;
        }
      };
      auto decode = [&](int j) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) decode_step<MT>(codes[c][j], b[j & 1][c]);
      };
      read_x(0);
      fold();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        scale[c] = scaled.value(raw[c], goff[c] + group_at);
      }
      decode(0);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (j + 1 < J) {
          read_x(j + 1);
          decode(j + 1);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            v[t][c] = mul_step<MT, 4>(a[j & 1][t], b[j & 1][c], 0, j == 0 ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : v[t][c]);
      }
    }
    if (++uplane == P) uplane = 0, used = span;
    slot = slot == 2 ? 0 : slot + 1;
  }
  fold();
  // acc -= (sums of x) (s z)^T, the first of the k ranges for all of them; of the parts' products those above 2^-24
  if (blockIdx.y == 0) {
    const int64_t pitch = p.span_blocks * kPartBytes;
    const uint8_t *ap[4], *bp[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int r = wm * 64 + t * 16 + col, n = wn * 64 + t * 16 + col;
      ap[t] = p.sums + (m0 + (r < rows ? r : rows - 1)) * pitch + quarter * 16;
      bp[t] = p.szs + (n0 + (n < cols ? n : cols - 1)) * pitch + quarter * 16;
    }
#pragma unroll 1
    for (int64_t at = 0; at < pitch; at += kPartBytes) {
      uint32_t a[3][4][4], b[3][4][4];
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint4 u = *reinterpret_cast<const uint4*>(ap[t] + at + q * 64), w = *reinterpret_cast<const uint4*>(bp[t] + at + q * 64);
          a[q][t][0] = u.x, a[q][t][1] = u.y, a[q][t][2] = u.z, a[q][t][3] = u.w;
          b[q][t][0] = w.x, b[q][t][1] = w.y, b[q][t][2] = w.z, b[q][t][3] = w.w;
        }
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int j = 0; i + j < 3; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t][c] = mul_step<DIMQ_BF16, 4>(a[i][t], b[j][c], 0, acc[t][c]);
    }
  }
  // 16 rows of the wave at a time through the LDS, so that a lane stores 8 neighbouring columns
  __syncthreads();
  float* mine = reinterpret_cast<float*>(lds) + wave * (16 * 68);
  const int64_t n = n0 + wn * 64 + lane % 8 * 8;
  const int left = p.N - n < 8 ? static_cast<int>(p.N - n) : 8;
  float bias[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = p.bias && p.splits == 1 && j < left ? load_as_float(p.bias, p.bias_dt, n + j) : 0.0f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(quarter * 4 + i) * 68 + c * 16 + col] = acc[t][c][i];
    lds_barrier();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = h * 8 + lane / 8;
      const int64_t m = m0 + wm * 64 + t * 16 + r;
      if (m >= p.M || left <= 0) continue;
      const float4* from = reinterpret_cast<const float4*>(mine + r * 68 + lane % 8 * 8);
      const float4 x = from[0], y = from[1];
      float o[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      const float by = row_scale(p, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(o[j], by, bias[j]);
      if (p.splits > 1) {
        float* to = p.part + (blockIdx.y * p.M + m) * p.N + n;
        if (left == 8) {
          typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
          reinterpret_cast<f4*>(to)[0] = f4{o[0], o[1], o[2], o[3]};
          reinterpret_cast<f4*>(to)[1] = f4{o[4], o[5], o[6], o[7]};
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < left) to[j] = o[j];
        }
      } else {
        put8(p, m * p.N + n, left, o);
      }
    }
    lds_barrier();
  }
}

// Adds the k ranges' sums, 8 neighbouring outputs of a row a thread (fewer at its end).
__global__ __launch_bounds__(256) void group_join_kernel(const GroupArgs p) {
  const uint32_t per = static_cast<uint32_t>((p.N + 7) / 8);
  const int64_t total = p.M * p.N, pieces = p.M * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t m = quotient(i, per), n = (i - m * per) * 8, off = m * p.N + n;
    const int left = p.N - n < 8 ? static_cast<int>(p.N - n) : 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p.bias && j < left ? load_as_float(p.bias, p.bias_dt, n + j) : 0.0f;
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
      const float* from = p.part + s * total + off;
      if (left == 8) {
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
        const f4 x = reinterpret_cast<const f4*>(from)[0], y = reinterpret_cast<const f4*>(from)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += x[j], sum[4 + j] += y[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += j < left ? from[j] : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += sum[j];
    put8(p, off, left, v);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

int span_bytes(int64_t group) { return group % 128 == 0 ? 16 : group % 64 == 0 ? 8 : 4; }

// Products of fewer multiply-adds than this run on the first kernel, larger ones on the tiles, whose three launches cost about
// 20 us before the first product.  In us, bf16, groups of 128 (first kernel / tiles): K 4096, 128 x 4096 24 / 34, 256 x 4096 35 / 35,
// 384 x 4096 66 / 41, 64 x 12288 30 / 36, 128 x 12288 58 / 40, 32 x 28000 46 / 53, 64 x 28000 69 / 56; K 1024, 384 x 8192 33 / 37,
// 512 x 8192 43 / 37; K 2048, 1024 x 2048 38 / 36.  fp32, whose three planes cost the first kernel more: K 4096, 128 x 4096 50 / 50,
// 192 x 4096 73 / 52, 64 x 12288 66 / 68.
// With groups that are no multiple of 64 the tiles decode and scale in spans of 32 and are slower: 256 x 4096 35 / 58,
// 192 x 12288 85 / 98, 256 x 12288 102 / 99, in fp32 192 x 4096 81 / 86, 256 x 4096 106 / 88.
bool few_rows(int xt, int64_t M, int64_t K, int64_t N, int64_t group, int variant) {
  // row and column blocks of one launch
  if (variant == DIMQ_VARIANT_MFMA || M > int64_t{65535} * 16 || N > (int64_t{1} << 23) * 16 - 16) return false;
  const bool fp32 = xt == DIMQ_F32, shorter = span_bytes(group) == 4;
  const double most = fp32 ? (shorter ? 3.5e9 : 2.1e9) : (shorter ? 8e9 : 4e9);
  return variant == DIMQ_VARIANT_SMALL_M || static_cast<double>(M) * static_cast<double>(K) * static_cast<double>(N) < most;
}
// One group a row, however large: the longest spans.
int64_t group_of(int64_t group, int64_t K) { return group >= K ? (K + 127) / 128 * 128 : group; }

int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

struct TilePlan {
  int64_t ksteps, tm, tn, copy_bytes, sum_bytes, sz_bytes, part_bytes;
  int splits;
  int64_t bytes() const { return copy_bytes + sum_bytes + sz_bytes + part_bytes; }
};
// Tiles that leave CUs idle are cut along k, into parts of at least four steps.
TilePlan tile_plan(int xt, int64_t M, int64_t K, int64_t N, bool in_place) {
  TilePlan t;
  t.ksteps = (K + kTileK - 1) / kTileK;
  t.tm = (M + kTileM - 1) / kTileM, t.tn = (N + kTileN - 1) / kTileN;
  const int64_t tiles = t.tm * t.tn, cus = device_cus();
  int64_t s = cus / tiles;
  if (s > t.ksteps / 4) s = t.ksteps / 4;
  t.splits = static_cast<int>(s < 1 ? 1 : s);
  t.splits = static_cast<int>((t.ksteps + (t.ksteps + t.splits - 1) / t.splits - 1) / ((t.ksteps + t.splits - 1) / t.splits));
  t.copy_bytes = in_place ? 0 : up256(M * t.ksteps * kTileK * 2) * planes_of(xt);
  const int64_t blocks = (t.ksteps * (kTileK / 32) + 31) / 32;  // spans of 32 at the least
  t.sum_bytes = up256(M * blocks * kPartBytes);
  t.sz_bytes = up256(N * blocks * kPartBytes);
  t.part_bytes = t.splits > 1 ? t.splits * M * N * 4 : 0;
  return t;
}

int64_t span_blocks(const TilePlan& t, int lb) { return (t.ksteps * (kTileK / (8 * lb)) + 31) / 32; }

bool rows_aligned(const void* x, int xt, int64_t M, int64_t ldx) {
  return aligned(x, 16) && (M <= 1 || ldx * x_size(xt) % 16 == 0);
}
constexpr int64_t kMostApart = 1 << 23;  // elements between rows that the tiles read: 128 of them stay below 2^32 bytes
bool rows_in_place(const void* x, int xt, int64_t M, int64_t K, int64_t ldx) {
  return x_size(xt) == 2 && K % kTileK == 0 && rows_aligned(x, xt, M, ldx) && ldx < kMostApart;
}

// Blocks of 16 rows (MT) and of 16 columns (NC) a work-group.  Its time goes as the loads and conversions of a turn, MT + NC (fp32,
// with three planes of x, 4 MT + NC), whatever MT NC products they feed, and one CU's work-groups add up: the plan is the one of
// least work-groups a CU times that.  Over 150 calls of 1 to 256 rows, K 1000 to 4096, N 1030 to 28000 and groups of 32, 64 and 128,
// each measured on all plans, the choice is 0.4 % slower than the best in the mean, 6 % at worst.  In us, bf16, K 4096, groups of
// 128 (MT x NC): 16 x 12288 1x1 22.1, 1x2 21.9, 1x3 16.0, 1x4 19.4; 64 x 12288 1x1 77, 2x2 42, 4x3 30.5; 256 x 4096 1x1 101, 4x4
// 34.9; groups of 32: 1 x 4096 1x1 7.6, 64 x 12288 1x1 81, 4x3 30.3 (with codes loaded by 4 bytes 14.5 and 52.8).
template <int XT, int LB>
constexpr bool few_plan(int mt, int nc) {
  return XT != DIMQ_F32 || (mt <= 2 && mt * nc < (LB == 4 ? 6 : 8));  // more would spill registers
}

template <int XT, int LB>
void launch_few(const GroupArgs& p, hipStream_t s) {
  constexpr int kXCost = XT == DIMQ_F32 ? 4 : 1;
  const int64_t gm = (p.M + 15) / 16, gn = (p.N + 15) / 16, cus = device_cus();
  int64_t least = INT64_MAX;
  int plan = 0;
  const auto each_plan = [](auto f) {
    const auto columns = [&](auto mt) {
      f(mt, std::integral_constant<int, 1>()), f(mt, std::integral_constant<int, 2>());
      f(mt, std::integral_constant<int, 3>()), f(mt, std::integral_constant<int, 4>());
    };
    columns(std::integral_constant<int, 1>()), columns(std::integral_constant<int, 2>()), columns(std::integral_constant<int, 4>());
  };
  each_plan([&](auto mt, auto nc) {
    if (!few_plan<XT, LB>(mt, nc)) return;
    const int64_t groups = ((gm + mt - 1) / mt) * ((gn + nc - 1) / nc), cost = kXCost * mt + nc;
    const int64_t all = ((groups + cus - 1) / cus * cost) << 8 | cost;  // among equals the smaller work-group
    if (all < least) least = all, plan = mt * 8 + nc;
  });
  each_plan([&](auto mt, auto nc) {
    if constexpr (few_plan<XT, LB>(mt, nc)) {
      if (plan != mt * 8 + nc) return;
      const dim3 grid(static_cast<unsigned>((gn + nc - 1) / nc), static_cast<unsigned>((gm + mt - 1) / mt));
      hipLaunchKernelGGL((group_few_kernel<XT, LB, mt, nc>), grid, dim3(64 * kFewWaves), 0, s, p);
    }
  });
}

template <int XT, int LB>
void launch_tile(GroupArgs p, const TilePlan& t, uint8_t* ws, hipStream_t s) {
  constexpr int ML = mul_type(XT), P = planes_of(XT);
  p.ksteps = t.ksteps, p.tiles_m = t.tm, p.tiles_n = t.tn, p.splits = t.splits;
  uint8_t *sums = ws + t.copy_bytes, *szs = sums + t.sum_bytes;
  p.plane = t.copy_bytes / P;
  p.span_blocks = span_blocks(t, LB);
  p.prep_first = static_cast<uint32_t>((p.N * p.span_blocks * 4 + 255) / 256);
  const int64_t blocks = (p.M * p.span_blocks * (32 * LB) + 256 * kPrepEach - 1) / (256 * kPrepEach);
  hipLaunchKernelGGL((group_prep_kernel<XT, LB>), dim3(static_cast<unsigned>(p.prep_first + blocks)), dim3(256), 0, s, p,
                     t.copy_bytes ? ws : nullptr, sums, szs);
  if (t.copy_bytes) {
    p.x = ws;
    p.ldx = t.ksteps * kTileK;
  }
  p.sums = sums, p.szs = szs;
  p.part = reinterpret_cast<float*>(szs + t.sz_bytes);
  const dim3 grid(static_cast<unsigned>(t.tm * t.tn), static_cast<unsigned>(t.splits));
  hipLaunchKernelGGL((group_tile_kernel<ML, LB, P>), grid, dim3(kTileThreads), 0, s, p);
  if (t.splits > 1) {
    const int64_t pieces = (p.M * ((p.N + 7) / 8) + 255) / 256;
    hipLaunchKernelGGL(group_join_kernel, dim3(static_cast<unsigned>(pieces < 4096 ? pieces : 4096)), dim3(256), 0, s, p);
  }
}

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_linear_grouped_workspace_bytes(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                                                       int64_t group, int64_t N, int variant) {
  if (M <= 0 || K <= 0 || N <= 0 || few_rows(x_dtype, M, K, N, group_of(group, K), variant)) return 0;
  if (x_dtype != DIMQ_F32 && x_dtype != DIMQ_F16 && x_dtype != DIMQ_BF16 && x_dtype != DIMQ_E4M3) return 0;
  const TilePlan t = tile_plan(x_dtype, M, K, N, rows_in_place(x, x_dtype, M, K, ldx));
  return t.bytes();
}

extern "C" int dimq_linear_grouped(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const float* x_scales,
                                   const uint8_t* codes, const void* scales, int scales_dtype, const uint8_t* zeros,
                                   int64_t group, const void* bias, int bias_dtype, int64_t N, void* y, int y_dtype,
                                   const void* residual, int residual_dtype, int activation, int variant,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  DIMQ_CHECK(x_dtype == DIMQ_F32 || x_dtype == DIMQ_F16 || x_dtype == DIMQ_BF16 || x_dtype == DIMQ_E4M3,
             "linear_grouped: input must be fp32, fp16, bf16 or e4m3");
  DIMQ_CHECK((x_dtype == DIMQ_E4M3) == (x_scales != nullptr) || M == 0, "linear_grouped: e4m3 rows, and no others, have scales");
  DIMQ_CHECK(scales_dtype == DIMQ_F32 || scales_dtype == DIMQ_F16 || scales_dtype == DIMQ_BF16,
             "linear_grouped: scales must be fp32, fp16 or bf16");
  DIMQ_CHECK(y_dtype == DIMQ_F32 || y_dtype == DIMQ_F16 || y_dtype == DIMQ_BF16,
             "linear_grouped: output must be fp32, fp16 or bf16");
  DIMQ_CHECK(M >= 0 && K > 0 && N > 0, "linear dimensions must be positive");
  DIMQ_CHECK(K < (int64_t)1 << 31 && N < (int64_t)1 << 31 && M < (int64_t)1 << 31,
             "linear_grouped: dimensions of 2^31 or more are not supported");
  DIMQ_CHECK(group > 0 && group % 32 == 0, "linear_grouped: the group size must be a positive multiple of 32");
  DIMQ_CHECK(M <= 1 || ldx >= K, "linear_grouped: row stride is below the row length");
  DIMQ_CHECK(activation >= DIMQ_ACT_NONE && activation <= DIMQ_ACT_GELU, "unknown activation %d", activation);
  DIMQ_CHECK(variant >= DIMQ_VARIANT_AUTO && variant <= DIMQ_VARIANT_MFMA, "unknown variant %d", variant);
  DIMQ_CHECK(!bias || is_float_dtype(bias_dtype), "linear_grouped: bias must be a float type");
  DIMQ_CHECK(!residual || is_float_dtype(residual_dtype), "linear_grouped: residual must be a float type");
  if (M == 0) return DIMQ_OK;
  DIMQ_CHECK(x && codes && scales && y, "linear_grouped: null pointer");
  DIMQ_CHECK(aligned(codes, 16), "linear_grouped: codes must be 16-byte aligned");
  DIMQ_CHECK(aligned(scales, dtype_size(scales_dtype)), "linear_grouped: misaligned scales");
  DIMQ_CHECK(aligned(x, x_dtype == DIMQ_E4M3 ? 1 : dtype_size(x_dtype)), "linear_grouped: misaligned input");
  group = group_of(group, K);
  GroupArgs p{};
  p.x = x, p.M = M, p.K = K, p.ldx = ldx, p.xs = x_scales, p.vec = rows_aligned(x, x_dtype, M, ldx);
  p.nb = (K + 31) / 32, p.codes = codes, p.pitch = p.nb * 16, p.scales = scales, p.s_dt = scales_dtype, p.zeros = zeros;
  p.group = group, p.groups = (K + group - 1) / group;
  p.N = N, p.bias = bias, p.bias_dt = bias_dtype, p.y = y, p.y_dt = y_dtype;
  p.epi = Epi{};
  p.epi.res = residual, p.epi.res_dt = residual_dtype, p.epi.act = activation;
  const hipStream_t s = as_stream(stream);
  const int lb = span_bytes(group);
#define DIMQ_GROUP_LB(F, XT, ...)               \
  if (lb == 16) F<XT, 16>(__VA_ARGS__);         \
  else if (lb == 8) F<XT, 8>(__VA_ARGS__);      \
  else F<XT, 4>(__VA_ARGS__);
#define DIMQ_GROUP_XT(F, ...)                                          \
  switch (x_dtype) {                                                   \
    case DIMQ_F32: DIMQ_GROUP_LB(F, DIMQ_F32, __VA_ARGS__) break;      \
    case DIMQ_F16: DIMQ_GROUP_LB(F, DIMQ_F16, __VA_ARGS__) break;      \
    case DIMQ_BF16: DIMQ_GROUP_LB(F, DIMQ_BF16, __VA_ARGS__) break;    \
    default: DIMQ_GROUP_LB(F, DIMQ_E4M3, __VA_ARGS__)                  \
  }
  if (few_rows(x_dtype, M, K, N, group, variant)) {
    DIMQ_GROUP_XT(launch_few, p, s)
  } else {
    const TilePlan t = tile_plan(x_dtype, M, K, N, rows_in_place(x, x_dtype, M, K, ldx));
    DIMQ_CHECK(workspace_bytes >= t.bytes() && aligned(workspace, 16),
               "linear_grouped: the workspace is too small or not 16-byte aligned");
    // a launch has less than 2^32 threads
    const int64_t prepared = span_blocks(t, lb) * (N * 4 + M * 32 * lb / kPrepEach);
    DIMQ_CHECK(t.tm * t.tn < (int64_t)1 << 23 && prepared < ((int64_t)1 << 32) - 4096, "linear_grouped: too many outputs for one launch");
    DIMQ_CHECK(t.ksteps * kTileK < kMostApart, "linear_grouped: rows of 2^23 elements or more take fewer rows");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    DIMQ_GROUP_XT(launch_tile, p, t, ws, s)
  }
#undef DIMQ_GROUP_XT
#undef DIMQ_GROUP_LB
  return check_launch("linear_grouped");
}
