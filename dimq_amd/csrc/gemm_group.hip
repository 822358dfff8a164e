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
// quarter l / 16) takes 2 LB consecutive k of a "span" of 8 LB, its codes one load of LB bytes.  A span lies in one group:
// LB 16 for groups of multiples of 128, 8 for other multiples of 64, 4 for other multiples of 32.
#include "decode.h"

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
  const float* sums;      // [M][spans of whole k steps]
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

// A lane's codes of a span as the instructions' operand.
template <int MT, int LB>
__device__ __forceinline__ void decode_span(const uint32_t (&codes)[LB / 4], uint32_t (&b)[LB]) {
#pragma unroll
  for (int j = 0; j < LB / 4; ++j) {
    uint32_t lo, hi;
    code_bytes(codes[j], lo, hi);
    b[4 * j] = code_pair<MT, false>(lo, 512.0f);
    b[4 * j + 1] = code_pair<MT, true>(lo, 512.0f);
    b[4 * j + 2] = code_pair<MT, false>(hi, 512.0f);
    b[4 * j + 3] = code_pair<MT, true>(hi, 512.0f);
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

// Scale i without a branch on its type: its first and last two bytes, which a 16-bit one has in common.
struct RawScale {
  uint32_t lo, hi;
};
__device__ __forceinline__ RawScale load_scale(const GroupArgs& p, int64_t i) {
  const uint16_t* s = static_cast<const uint16_t*>(p.scales);
  const int wide = p.s_dt == DIMQ_F32;
  return {s[i << wide], s[(i << wide) + wide]};
}
__device__ __forceinline__ float scale_of(const GroupArgs& p, const RawScale& r) {
  const float wide = __uint_as_float(r.hi << 16 | (p.s_dt == DIMQ_F32 ? r.lo : 0u));  // fp32, and bf16's bits
  return p.s_dt == DIMQ_F16 ? f16_bits_to_float(r.lo) : wide;
}

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

// ---- few rows -----------------------------------------------------------------------------------------------------
// 16 MT rows by 16 columns a work-group; its 8 waves share out the spans, and their sums meet in the LDS.  A wave's loads
// of U spans go out together.  Rows past M re-read the last one; they are not stored.
constexpr int kFewWaves = 8;

template <int XT, int LB, int MT, int U>
__global__ __launch_bounds__(64 * kFewWaves) void group_few_kernel(const GroupArgs p) {
  constexpr int ML = mul_type(XT), P = planes_of(XT), SP = 8 * LB;
  __shared__ floatx4 red[kFewWaves][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quarter = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16, m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const int64_t n = n0 + col < p.N ? n0 + col : p.N - 1;
  const int spans = static_cast<int>((p.nb * 32 + SP - 1) / SP), each = (spans + kFewWaves - 1) / kFewWaves;
  const int from = wave * each, to = from + each < spans ? from + each : spans;
  const uint8_t* cw = p.codes + n * p.pitch;
  const int group_spans = static_cast<int>(p.group / SP);  // a group is a whole number of spans
  floatx4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = from; s0 < to; s0 += U) {
    uint32_t codes[U][LB / 4];
    RawScale rs[U];
    uint32_t z[U];
    RawX<XT, LB> rx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int sp = s0 + u < to ? s0 + u : to - 1;
      // a lane's codes past the row's last block read that block's (x is 0 there)
      int64_t at = static_cast<int64_t>(sp) * (4 * LB) + quarter * LB;
      if (at + LB > p.pitch) at = p.pitch - LB < 0 ? 0 : p.pitch - LB;
      if constexpr (LB == 16) {
        const uint4 c = *reinterpret_cast<const uint4*>(cw + at);
        codes[u][0] = c.x, codes[u][1] = c.y, codes[u][2] = c.z, codes[u][3] = c.w;
      } else if constexpr (LB == 8) {
        const uint2 c = *reinterpret_cast<const uint2*>(cw + at);
        codes[u][0] = c.x, codes[u][1] = c.y;
      } else {
        codes[u][0] = *reinterpret_cast<const uint32_t*>(cw + at);
      }
      const int64_t gi = n * p.groups + sp / group_spans;
      rs[u] = load_scale(p, gi);
      z[u] = p.zeros ? p.zeros[gi] : 8u;
      const int64_t k0 = static_cast<int64_t>(sp) * SP + quarter * (2 * LB);
      const bool fast = p.vec && static_cast<int64_t>(sp + 1) * SP <= p.K;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int64_t m = m0 + 16 * t + col;
        rx[u][t].load(p, m < p.M ? m : p.M - 1, k0, fast);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= to) break;
      uint32_t b[LB];
      decode_span<ML, LB>(codes[u], b);
      const float s = scale_of(p, rs[u]), zf = static_cast<float>(z[u]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uint32_t a[P][LB];
        rx[u][t].planes(a);
        floatx4 q = floatx4{0.0f, 0.0f, 0.0f, 0.0f}, x = q;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          q = mul_span<ML, LB>(a[i], b, q);
          x = sum_span<ML, LB>(a[i], x);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(s, fmaf(-zf, x[i], q[i]), acc[t][i]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave >= MT) return;
  floatx4 v = red[0][wave][lane];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) v += red[w][wave][lane];
  if (n0 + col >= p.N) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + 16 * wave + 4 * quarter + i;
    if (m < p.M) put_output(p, m, n0 + col, v[i] * row_scale(p, m));
  }
}

// ---- many rows ----------------------------------------------------------------------------------------------------
// The zero points' part of the product, sum_g s z sum_{k in g} x, is a product of its own with a reduction 8 LB times
// shorter: a first launch sums x over each span (and copies x where its rows are not whole k steps, aligned and of 16 bits),
// and after the main loop those sums and s z, each as three bf16 parts, go through the matrix instructions once.  Against
// ones in the loop the sums cost a fifth of its matrix instructions, and taken off each span's product half of its fmas.
//
// Then 128 x 128 outputs a work-group of 4 waves of 64 x 64 each.  A k step is 128: x of all 128 rows and the columns' codes
// come into the LDS by direct loads, a step ahead, and the codes are decoded behind the LDS.
constexpr int kTile = 128, kTileK = 128, kTileThreads = 256;

// sums [M][spans of whole k steps]; out (nullable): x padded with zeros to whole k steps, [planes][M][ksteps 128].
template <int XT, int LB>
__global__ __launch_bounds__(256) void group_prep_kernel(const GroupArgs p, uint8_t* out, float* sums) {
  const uint32_t per = static_cast<uint32_t>(p.ksteps) * (kTileK / 8);  // a multiple of 16: 16 neighbouring lanes share a row
  const int64_t total = p.M * per, kp = p.ksteps * kTileK;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t m = i / per, k0 = (i - m * per) * 8;
    RawX<XT, 4> r;
    r.load(p, m, k0, p.vec && k0 + 8 <= p.K);
    uint32_t a[planes_of(XT)][4];
    r.planes(a);
    if (out) {
#pragma unroll
      for (int q = 0; q < planes_of(XT); ++q)
        *reinterpret_cast<uint4*>(out + q * p.plane + (m * kp + k0) * 2) = make_uint4(a[q][0], a[q][1], a[q][2], a[q][3]);
    }
    float s = 0.0f;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if constexpr (XT == DIMQ_F32) s += __uint_as_float(r.w[q]);
      else if constexpr (XT == DIMQ_F16) s += f16_bits_to_float((r.w[q >> 1] >> (16 * (q & 1))) & 0xffffu);
      else s += bf16_bits_to_float((a[0][q >> 1] >> (16 * (q & 1))) & 0xffffu);
    }
#pragma unroll
    for (int w = 1; w < LB; w *= 2) s += __shfl_xor(s, w, 64);
    if ((threadIdx.x & (LB - 1)) == 0) sums[(m * kp + k0) / (8 * LB)] = s;
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

// MT: type of x in the LDS; P: its planes, one after another within a k step.
template <int MT, int LB, int P>
__global__ __launch_bounds__(kTileThreads, 2) void group_tile_kernel(const GroupArgs p) {
  constexpr int SP = 8 * LB, NS = kTileK / SP;
  constexpr int RowBytes = kTileK * 2, Chunks = RowBytes / 16, StageBytes = kTile * RowBytes, CodeBytes = kTile * 64;
  __shared__ __attribute__((aligned(1024))) uint8_t xs[2][StageBytes];
  __shared__ __attribute__((aligned(1024))) uint8_t cs[2][CodeBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quarter = lane >> 4;
  const int wm = wave & 1, wn = wave >> 1;
  // neighbouring work-groups are on different XCDs: each XCD takes a contiguous part of the tiles, rows fastest, so that its
  // L2 holds a few columns' codes and x
  const uint32_t tiles = static_cast<uint32_t>(p.tiles_m * p.tiles_n), per = tiles / 8, rest = tiles % 8, xcd = blockIdx.x % 8;
  const uint32_t tile = xcd * per + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
  const uint32_t tm = static_cast<uint32_t>(p.tiles_m);
  const int64_t m0 = static_cast<int64_t>(tile % tm) * kTile, n0 = static_cast<int64_t>(tile / tm) * kTile;
  const int ksteps = static_cast<int>(p.ksteps), steps_each = (ksteps + p.splits - 1) / p.splits;
  const int step0 = blockIdx.y * steps_each, step1 = step0 + steps_each < ksteps ? step0 + steps_each : ksteps;
  const uint32_t ldsx = lds_address(&xs[0][0]), ldsc = lds_address(&cs[0][0]);
  const int rows = p.M - m0 < kTile ? static_cast<int>(p.M - m0) : kTile, cols = p.N - n0 < kTile ? static_cast<int>(p.N - n0) : kTile;

  // Stage of x: a wave's load is 1 KB, 4 rows of 16 pieces; piece c of row r lies at slot c ^ (r % 16).  Offsets from the
  // tile's first row stay below 2^32 (checked on the host).
  constexpr int kLoads = StageBytes / 1024 / 4;
  uint32_t xoff[kLoads], coff[2];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = (wave * kLoads + i) * 4 + lane / Chunks, c = (lane % Chunks) ^ (r % Chunks);
    xoff[i] = static_cast<uint32_t>(r < rows ? r : rows - 1) * static_cast<uint32_t>(p.ldx * 2) + c * 16;
  }
  // stage of codes: 64 bytes a column
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (wave * 2 + i) * 16 + lane / 4;
    coff[i] = static_cast<uint32_t>(r < cols ? r : cols - 1) * static_cast<uint32_t>(p.pitch) + lane % 4 * 16;
  }
  const uint8_t* xbase = static_cast<const uint8_t*>(p.x) + m0 * p.ldx * 2;
  const uint8_t* cbase = p.codes + n0 * p.pitch;
  auto fetch_x = [&](int step, int plane, int slot) {
    const uint8_t* base = uniform(xbase + plane * p.plane + static_cast<int64_t>(step) * RowBytes);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) group_dma16(base, xoff[i], ldsx + slot * StageBytes + (wave * kLoads + i) * 1024);
  };
  auto fetch_codes = [&](int step, int slot) {
    const uint8_t* base = uniform(cbase + static_cast<int64_t>(step) * 64);
    // past the row's last block that block again (x is 0 there)
    const int over = (step + 1) * 64 - static_cast<int>(p.pitch), back = over > 0 ? lane % 4 * 16 + over - 48 : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      group_dma16(base, coff[i] - (back > 0 ? back : 0), ldsc + slot * CodeBytes + (wave * 2 + i) * 1024);
  };
  // scales of 4 blocks of 16 columns in a step (their bits; load_scale); the spans' groups are counted up
  const int wide = p.s_dt == DIMQ_F32, group_spans = static_cast<int>(p.group / SP);
  uint32_t goff[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int n = wn * 64 + c * 16 + col;
    goff[c] = static_cast<uint32_t>(n < cols ? n : cols - 1) * static_cast<uint32_t>(p.groups);
  }
  const uint16_t* sbase = static_cast<const uint16_t*>(p.scales) + ((n0 * p.groups) << wide);
  const uint32_t groups = static_cast<uint32_t>(p.groups);
  auto raw_scale = [&](int c, uint32_t at) -> RawScale {
    const uint32_t i = (goff[c] + at) << wide;
    return {sbase[i], sbase[i + wide]};
  };
  RawScale rs[4][NS];
  uint32_t g = static_cast<uint32_t>(step0) * NS / group_spans, phase = static_cast<uint32_t>(step0) * NS % group_spans;
  auto fetch_scales = [&]() {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int c = 0; c < 4; ++c) rs[c][s] = raw_scale(c, g < groups ? g : groups - 1);
      if (++phase == static_cast<uint32_t>(group_spans)) phase = 0, ++g;
    }
  };

  floatx4 acc[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[t][c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  if (step0 < step1) {
    fetch_scales();
    fetch_codes(step0, 0);
    fetch_x(step0, 0, 0);
  }
  int slot = 0, cslot = 0;
  for (int step = step0; step < step1; ++step) {
    float sc[4][NS];
#pragma unroll 1  // unrolled, the planes would keep their codes decoded and spill
    for (int plane = 0; plane < P; ++plane) {
      wait_vmcnt<0>();
      __syncthreads();  // this stage is in the LDS, and the other one is free
      if (plane == 0) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[c][s] = scale_of(p, rs[c][s]);
      }
      if (plane + 1 < P) {
        fetch_x(step, plane + 1, slot ^ 1);
      } else if (step + 1 < step1) {
        fetch_scales();
        fetch_codes(step + 1, cslot ^ 1);
        fetch_x(step + 1, 0, slot ^ 1);
      }
      const uint8_t *st = xs[slot], *ct = cs[cslot] + (wn * 64 + col) * 64;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        uint32_t a[4][LB];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int r = wm * 64 + t * 16 + col, c0 = (s * SP + quarter * 2 * LB) / 8;  // piece of the row
#pragma unroll
          for (int i = 0; i < LB / 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(st + r * RowBytes + (((c0 + i) ^ (r % Chunks)) << 4));
            a[t][4 * i] = v.x, a[t][4 * i + 1] = v.y, a[t][4 * i + 2] = v.z, a[t][4 * i + 3] = v.w;
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[LB / 4], b[LB];
          const uint8_t* q = ct + c * 1024 + s * (4 * LB) + quarter * LB;
          if constexpr (LB == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(q);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
          } else if constexpr (LB == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(q);
            w[0] = v.x, w[1] = v.y;
          } else {
            w[0] = *reinterpret_cast<const uint32_t*>(q);
          }
          decode_span<MT, LB>(w, b);
          floatx4 v[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) v[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < LB / 4; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = mul_step<MT, LB>(a[t], b, j, v[t]);
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][c][i] = fmaf(sc[c][s], v[t][i], acc[t][c][i]);
        }
      }
      slot ^= 1;
    }
    cslot ^= 1;
  }
  // acc -= (sums of x) (s z)^T, the first of the k ranges for all of them; of the parts' products those above 2^-24
  if (blockIdx.y == 0) {
    const uint8_t* zbase = p.zeros ? p.zeros + n0 * p.groups : nullptr;
    const int spans = ksteps * NS;
    const float* sums = p.sums + m0 * spans;
#pragma unroll 1
    for (int g0 = 0; g0 < spans; g0 += 32) {
      const int mine = g0 + quarter * 8;
      uint32_t a[4][3][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int r = wm * 64 + t * 16 + col;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = sums[static_cast<int64_t>(r < rows ? r : rows - 1) * spans + (mine + e < spans ? mine + e : spans - 1)];
          v[e] = mine + e < spans ? __float_as_uint(f) : 0u;
        }
        split3(v, a[t][0], a[t][1], a[t][2]);
      }
      uint32_t at[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        at[e] = static_cast<uint32_t>(mine + e) / static_cast<uint32_t>(group_spans);
        if (at[e] >= groups) at[e] = groups - 1;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t v[8], b[3][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = static_cast<float>(zbase ? zbase[goff[c] + at[e]] : 8u);
          v[e] = __float_as_uint(-scale_of(p, raw_scale(c, at[e])) * z);
        }
        split3(v, b[0], b[1], b[2]);
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int j = 0; i + j < 3; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t][c] = mul_step<DIMQ_BF16, 4>(a[t][i], b[j], 0, acc[t][c]);
      }
    }
  }
  // 16 rows of the wave at a time through the LDS, so that a store is 64 neighbouring columns
  __syncthreads();
  float* mine = reinterpret_cast<float*>(&xs[0][0]) + wave * (16 * 65);
  const int64_t n = n0 + wn * 64 + lane;
  const float bias = p.bias && n < p.N && p.splits == 1 ? load_as_float(p.bias, p.bias_dt, n) : 0.0f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(quarter * 4 + i) * 65 + c * 16 + col] = acc[t][c][i];
    lds_barrier();
    const int64_t first = m0 + wm * 64 + t * 16;
    if (n < p.N) {
#pragma unroll 4
      for (int r = 0; r < 16; ++r) {
        const int64_t m = first + r;
        if (m >= p.M) break;
        const float v = mine[r * 65 + lane] * row_scale(p, m);
        if (p.splits > 1) {
          p.part[(blockIdx.y * p.M + m) * p.N + n] = v;
        } else {
          const int64_t off = m * p.N + n;
          store_from_float(p.y, p.y_dt, off, epi1(p.epi, off, v + bias));
        }
      }
    }
    lds_barrier();
  }
}

__global__ __launch_bounds__(256) void group_join_kernel(const GroupArgs p) {
  const int64_t total = p.M * p.N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    float v = p.part[i];
    for (int s = 1; s < p.splits; ++s) v += p.part[s * total + i];
    const int64_t m = i / p.N;
    put_output(p, m, i - m * p.N, v);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

int span_bytes(int64_t group) { return group % 128 == 0 ? 16 : group % 64 == 0 ? 8 : 4; }

constexpr int64_t kFewRows = 64;  // rows of the first kernel

int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

struct TilePlan {
  int64_t ksteps, tm, tn, copy_bytes, sum_bytes, part_bytes;
  int splits;
  int64_t bytes() const { return copy_bytes + sum_bytes + part_bytes; }
};
// Tiles that leave CUs idle are cut along k, into parts of at least four steps.
TilePlan tile_plan(int xt, int64_t M, int64_t K, int64_t N, bool in_place) {
  TilePlan t;
  t.ksteps = (K + kTileK - 1) / kTileK;
  t.tm = (M + kTile - 1) / kTile, t.tn = (N + kTile - 1) / kTile;
  const int64_t tiles = t.tm * t.tn, cus = device_cus();
  int64_t s = cus / tiles;
  if (s > t.ksteps / 4) s = t.ksteps / 4;
  t.splits = static_cast<int>(s < 1 ? 1 : s);
  t.splits = static_cast<int>((t.ksteps + (t.ksteps + t.splits - 1) / t.splits - 1) / ((t.ksteps + t.splits - 1) / t.splits));
  t.copy_bytes = in_place ? 0 : up256(M * t.ksteps * kTileK * 2) * planes_of(xt);
  t.sum_bytes = up256(M * t.ksteps * (kTileK / 32) * 4);  // spans of 32 at the least
  t.part_bytes = t.splits > 1 ? t.splits * M * N * 4 : 0;
  return t;
}

bool rows_aligned(const void* x, int xt, int64_t M, int64_t ldx) {
  return aligned(x, 16) && (M <= 1 || ldx * x_size(xt) % 16 == 0);
}
constexpr int64_t kMostApart = 1 << 23;  // elements between rows that the tiles read: 128 of them stay below 2^32 bytes
bool rows_in_place(const void* x, int xt, int64_t M, int64_t K, int64_t ldx) {
  return x_size(xt) == 2 && K % kTileK == 0 && rows_aligned(x, xt, M, ldx) && ldx < kMostApart;
}

template <int XT, int LB>
void launch_few(const GroupArgs& p, hipStream_t s) {
  const unsigned gx = static_cast<unsigned>((p.N + 15) / 16);
  const dim3 threads(64 * kFewWaves);
  if (p.M <= 16) hipLaunchKernelGGL((group_few_kernel<XT, LB, 1, 4>), dim3(gx), threads, 0, s, p);
  else if (p.M <= 32) hipLaunchKernelGGL((group_few_kernel<XT, LB, 2, 2>), dim3(gx), threads, 0, s, p);
  else hipLaunchKernelGGL((group_few_kernel<XT, LB, 4, 1>), dim3(gx, static_cast<unsigned>((p.M + 63) / 64)), threads, 0, s, p);
}

template <int XT, int LB>
void launch_tile(GroupArgs p, const TilePlan& t, uint8_t* ws, hipStream_t s) {
  constexpr int ML = mul_type(XT), P = planes_of(XT);
  p.ksteps = t.ksteps, p.tiles_m = t.tm, p.tiles_n = t.tn, p.splits = t.splits;
  float* sums = reinterpret_cast<float*>(ws + t.copy_bytes);
  p.plane = t.copy_bytes / P;
  const int64_t blocks = (p.M * t.ksteps * (kTileK / 8) + 255) / 256;
  hipLaunchKernelGGL((group_prep_kernel<XT, LB>), dim3(static_cast<unsigned>(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, p,
                     t.copy_bytes ? ws : nullptr, sums);
  if (t.copy_bytes) {
    p.x = ws;
    p.ldx = t.ksteps * kTileK;
  }
  p.sums = sums;
  p.part = reinterpret_cast<float*>(ws + t.copy_bytes + t.sum_bytes);
  const dim3 grid(static_cast<unsigned>(t.tm * t.tn), static_cast<unsigned>(t.splits));
  hipLaunchKernelGGL((group_tile_kernel<ML, LB, P>), grid, dim3(kTileThreads), 0, s, p);
  if (t.splits > 1) {
    const int64_t blocks = (p.M * p.N + 255) / 256;
    hipLaunchKernelGGL(group_join_kernel, dim3(static_cast<unsigned>(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, p);
  }
}

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_linear_grouped_workspace_bytes(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int64_t N) {
  if (M <= kFewRows || K <= 0 || N <= 0) return 0;
  if (x_dtype != DIMQ_F32 && x_dtype != DIMQ_F16 && x_dtype != DIMQ_BF16 && x_dtype != DIMQ_E4M3) return 0;
  const TilePlan t = tile_plan(x_dtype, M, K, N, rows_in_place(x, x_dtype, M, K, ldx));
  return t.bytes();
}

extern "C" int dimq_linear_grouped(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const float* x_scales,
                                   const uint8_t* codes, const void* scales, int scales_dtype, const uint8_t* zeros,
                                   int64_t group, const void* bias, int bias_dtype, int64_t N, void* y, int y_dtype,
                                   const void* residual, int residual_dtype, int activation, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
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
  DIMQ_CHECK(!bias || is_float_dtype(bias_dtype), "linear_grouped: bias must be a float type");
  DIMQ_CHECK(!residual || is_float_dtype(residual_dtype), "linear_grouped: residual must be a float type");
  if (M == 0) return DIMQ_OK;
  DIMQ_CHECK(x && codes && scales && y, "linear_grouped: null pointer");
  DIMQ_CHECK(aligned(codes, 16), "linear_grouped: codes must be 16-byte aligned");
  DIMQ_CHECK(aligned(x, x_dtype == DIMQ_E4M3 ? 1 : dtype_size(x_dtype)), "linear_grouped: misaligned input");
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
  if (M <= kFewRows) {
    DIMQ_GROUP_XT(launch_few, p, s)
  } else {
    const TilePlan t = tile_plan(x_dtype, M, K, N, rows_in_place(x, x_dtype, M, K, ldx));
    DIMQ_CHECK(workspace_bytes >= t.bytes() && aligned(workspace, 16),
               "linear_grouped: the workspace is too small or not 16-byte aligned");
    DIMQ_CHECK(t.tm * t.tn < (int64_t)1 << 24, "linear_grouped: too many outputs for one launch");
    DIMQ_CHECK(t.ksteps * kTileK < kMostApart, "linear_grouped: more than 64 rows must be shorter than 2^23 elements");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    DIMQ_GROUP_XT(launch_tile, p, t, ws, s)
  }
#undef DIMQ_GROUP_XT
#undef DIMQ_GROUP_LB
  return check_launch("linear_grouped");
}
