// Rows of logits x: log probabilities of given tokens, entropy and the largest alternatives, the distillation loss of a
// teacher's top logits, and the gradients of both.
//
//   m = max x,  s = sum 2^(k x - i),  u = sum 2^(k x - i) (k x - i)      one pass, kept as a running (m, s, u)
//   k = log2 e (over the temperature),  i = k m rounded to an integer
//   log p = (x - m) / t - l,  l = log s - (k m - i) log 2,  entropy = -sum p log p = log s - (u / s) log 2
//
// so that an element costs an fma, an exponential and an addition, nothing but the fma rounds an exponent, and a larger
// maximum scales s by a power of two.  From |k m| = 2^20 on, where k m's own rounding would count (a row of masks at the type's
// lowest number), the exponent is k (x - m) instead.
//
// A row that holds a NaN or +infinity, or nothing above -infinity, has no distribution: its values are NaN and its
// alternatives' tokens -1.  -infinity in a row has p = 0 and adds nothing; the type's lowest finite number is a number.
//
// Alternatives, in the same pass: of each thread's running maxima (256 to a work-group) the k-th largest is a lower bound of
// the k-th largest logit, and only the threads whose maximum reaches it, little more than k of them, read their logits
// again and hand on those that reach it.  Those few are ranked by counting.  Equal logits rank by token, lower first.
//
// Bound by bytes: a row is read once (the gradients read it once more and write theirs).  A row is cut over several
// work-groups where there are few of them; a second launch then joins their (m, s, u) and candidates.
//
// Measured (large reads reach 6.0 to 6.8 TB/s, copies 5.07): distillation of 2048 x 128000 bf16 103 us forward (5.1 TB/s) and
// 209 backward (5.0 TB/s); scores of 4096 x 32768 fp16 with 32 alternatives 74 us (3.6 TB/s; 45 of them are the pass), of one
// row of 128000 12 us, where the two launches' latencies count.
#include "common.h"
#include "rows.h"

namespace dimq {
namespace {

constexpr int kLgThreads = 256;
constexpr int kLgCand = 1024;      // candidates a work-group holds: more fall back to one pass per alternative
constexpr int kLgTop = 128;        // most alternatives
constexpr int kLgSplits = 32;      // most work-groups to a row
constexpr int64_t kMostEntries = 4096;  // of a teacher's row: the gradient looks for equal tokens by comparing all pairs
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;

struct LogitArgs {
  const void* x;
  int64_t ldx, rows, V;
  int splits;
  int64_t chunk;  // elements of a split, a multiple of 8
  float tau_inv;  // distillation: 1 / temperature
  // scoring
  const void* tokens;
  int tokens64;
  int top;
  float* logp;
  float* entropy;
  float* norm;     // [rows][2] m and log s, kept for the gradients (the pair: a large lse alone would lose digits)
  float* top_logp;
  int64_t* top_ids;
  // distillation
  const void* values;
  int values_dt;
  const void* ids;
  int ids64;
  int k;
  float* loss;     // [rows]
  float* p;        // [rows][k] the teacher's probabilities
  // partial results of splits
  float* stats;    // [rows][splits][4]: m, s, u
  uint64_t* cand;  // [rows][splits][top]
};

constexpr float kLn2 = 0.69314718055994530942f;

// 2^d, d no larger than 1.
__device__ __forceinline__ float exp2_of(float d) { return __builtin_amdgcn_exp2f(d); }
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// Where the exponents of a running maximum m are counted from.
struct Origin {
  float m, i;
  bool far;
  __device__ __forceinline__ Origin(float max, float k) : m(max) {
    const float x = max * k;
    far = !(fabsf(x) < 0x1p20f);
    i = far ? 0.0f : __builtin_rintf(x);
  }
  __device__ __forceinline__ float exponent(float x, float k) const { return far ? (x - m) * k : fmaf(x, k, -i); }
  // from this origin to another
  __device__ __forceinline__ float to(const Origin& o, float k) const {
    return far ? (o.far ? (m - o.m) * k : fmaf(m, k, -o.i)) : (o.far ? fmaf(-o.m, k, i) : i - o.i);
  }
};

struct Stats {
  float m, s, u;
};

// (m, s, u) from its own maximum's origin to a larger one's.  Exponents are held above -300, whose power is 0, so that no
// 0 * infinity arises.
template <bool U>
__device__ __forceinline__ void raise(Stats& a, const Origin& from, const Origin& o, float k) {
  const float d = fmaxf(from.to(o, k), -300.0f), e = exp2_of(d);
  if constexpr (U) a.u = e * fmaf(a.s, d, a.u);
  a.s *= e;
  a.m = o.m;
}

// Two sums over the work-group behind one barrier.
__device__ __forceinline__ void block_add2(float& a, float& b, float (*red)[4]) {
  a = wave_add(a);
  b = wave_add(b);
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = a, red[1][threadIdx.x >> 6] = b;
  __syncthreads();
  a = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
  b = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
}

// Every thread's to the common maximum, then plain sums.
template <bool U>
__device__ __forceinline__ Stats block_stats(Stats a, float k, float (*red)[4]) {
  const float m = row_reduce<kLgThreads, true>(a.m, red[0]);
  raise<U>(a, Origin(a.m, k), Origin(m, k), k);
  block_add2(a.s, a.u, red + 1);
  return a;
}

// Order of the logits as unsigned numbers, NaN above all, -0 equal to 0; 0 is below every logit.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 + 0 = 0
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Unique keys: the larger logit first, then the lower token.
__device__ __forceinline__ uint64_t key_of(float v, int64_t at) {
  return static_cast<uint64_t>(order_of(v)) << 32 | (0xffffffffu - static_cast<uint32_t>(at));
}

template <int XT>
__device__ __forceinline__ float logit(const void* row, int64_t i) {
  return load_as_float(row, XT, i);
}

template <int XT>
constexpr int pack_of() {
  return XT == DIMQ_F32 ? 4 : 8;
}

// 16 aligned bytes of a row as floats.
template <int XT>
__device__ __forceinline__ void unpack16(const uint4& t, float (&v)[pack_of<XT>()]) {
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
  if constexpr (XT == DIMQ_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = XT == DIMQ_F16 ? f16_bits_to_float(w[j] & 0xffffu) : bf16_bits_to_float(w[j] & 0xffffu);
      v[2 * j + 1] = XT == DIMQ_F16 ? f16_bits_to_float(w[j] >> 16) : bf16_bits_to_float(w[j] >> 16);
    }
  }
}

// Elements [a, b) of a row in three parts: single ones up to the first 16-byte boundary, whole 16-byte pieces, the rest.
struct Span {
  int64_t a, body, b;  // body: first element of the pieces
  int64_t pieces;
  template <int XT>
  __device__ __forceinline__ static Span of(const void* row, int64_t a, int64_t b) {
    constexpr int kSize = XT == DIMQ_F32 ? 4 : 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(row) + a * kSize;
    int64_t head = static_cast<int64_t>((16 - (at & 15)) & 15) / kSize;
    if (head > b - a) head = b - a;
    return {a, a + head, b, (b - a - head) / pack_of<XT>()};
  }
  __device__ __forceinline__ int singles(int pack) const {
    return static_cast<int>((body - a) + (b - body - pieces * pack));
  }
  __device__ __forceinline__ int64_t single(int i, int pack) const {
    return i < body - a ? a + i : body + pieces * pack + (i - (body - a));
  }
};

__device__ __forceinline__ float max3(float a, float b, float c) {  // not of fmaxf: it would quiet each operand first
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Adds N elements; NaN and +infinity make s NaN.
template <int N, bool U>
__device__ __forceinline__ void add_to(Stats& st, Origin& o, const float (&v)[N], float k) {
  float cm;
  if constexpr (N == 8) cm = max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), max3(v[6], v[7], v[7]));
  else if constexpr (N == 4) cm = max3(max3(v[0], v[1], v[2]), v[3], v[3]);
  else cm = v[0];
  if (cm > st.m) {
    const Origin n(cm, k);
    raise<U>(st, o, n, k);
    o = n;
  }
  float d[N];
  if (__builtin_expect(o.far, 0)) {
#pragma unroll
    for (int j = 0; j < N; ++j) d[j] = (v[j] - o.m) * k;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) d[j] = fmaf(v[j], k, -o.i);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float e = exp2_of(d[j]);
    st.s += e;
    if constexpr (U) st.u = fmaf(e, fmaxf(d[j], -300.0f), st.u);
  }
}

// The calling thread's part of [a, b): pieces tid, tid + 256, ..., and one of the single elements.
template <int XT, bool U>
__device__ __forceinline__ Stats stream_stats(const void* row, const Span& sp, float k) {
  constexpr int P = pack_of<XT>();
  Stats st{kLowest, 0.0f, 0.0f};
  Origin o(kLowest, k);
  const uint4* body = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + sp.body * (16 / P));
  int64_t i = threadIdx.x;
  for (; i + 3 * kLgThreads < sp.pieces; i += 4 * kLgThreads) {
    uint4 t[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) t[q] = body[i + q * kLgThreads];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[P];
      unpack16<XT>(t[q], v);
      add_to<P, U>(st, o, v, k);
    }
  }
  for (; i < sp.pieces; i += kLgThreads) {
    float v[P];
    unpack16<XT>(body[i], v);
    add_to<P, U>(st, o, v, k);
  }
  if (static_cast<int>(threadIdx.x) < sp.singles(P)) {
    const float v[1] = {logit<XT>(row, sp.single(threadIdx.x, P))};
    add_to<1, U>(st, o, v, k);
  }
  return st;
}

// Calls f(element, index) for the calling thread's part, as stream_stats goes through it.
template <int XT, class F>
__device__ __forceinline__ void each_of_mine(const void* row, const Span& sp, F f) {
  constexpr int P = pack_of<XT>();
  const uint4* body = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + sp.body * (16 / P));
  for (int64_t i = threadIdx.x; i < sp.pieces; i += kLgThreads) {
    float v[P];
    unpack16<XT>(body[i], v);
#pragma unroll
    for (int j = 0; j < P; ++j) f(v[j], sp.body + i * P + j);
  }
  if (static_cast<int>(threadIdx.x) < sp.singles(P)) {
    const int64_t at = sp.single(threadIdx.x, P);
    f(logit<XT>(row, at), at);
  }
}

struct TopShared {
  alignas(16) uint32_t maxima[kLgThreads];
  uint64_t cand[kLgCand];
  uint8_t owners[kLgThreads];
  int count, nowners;
  uint32_t bound;
};

// A lower bound of the top-th largest logit's order, from the largest order each thread knows of (0: none): the top-th
// largest of these, found by counting.  Their last 8 bits give way to a number, so that no two are alike and a comparison is
// all it takes; the bound is only lower for it.  Up to 48 alternatives the maxima of four threads each do: 64 of them, which
// every wave counts by itself in a quarter of the time, for a third more candidates at the most.
constexpr int kFewTop = 48;

__device__ __forceinline__ uint32_t bound_of(uint32_t mine, int top, TopShared& sh) {
  if (threadIdx.x == 0) sh.count = 0, sh.nowners = 0;
  if (top <= kFewTop) {
    sh.maxima[threadIdx.x] = mine;
    __syncthreads();
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t a = sh.maxima[lane], b = sh.maxima[lane + 64], c = sh.maxima[lane + 128], d = sh.maxima[lane + 192];
    const uint32_t ab = a > b ? a : b, cd = c > d ? c : d, key = ((ab > cd ? ab : cd) & ~0xffu) | (63u - lane);
    int before = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) before += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), i)) > key;
    const uint64_t at = __ballot(before == top - 1);
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), __builtin_ctzll(at))) & ~0xffu;
  }
  const uint32_t key = (mine & ~0xffu) | (255u - threadIdx.x);
  sh.maxima[threadIdx.x] = key;
  __syncthreads();
  int before = 0;
#pragma unroll 16
  for (int i = 0; i < kLgThreads; i += 4) {
    const uint4 o = *reinterpret_cast<const uint4*>(&sh.maxima[i]);
    before += (o.x > key) + (o.y > key) + (o.z > key) + (o.w > key);
  }
  if (before == top - 1) sh.bound = mine & ~0xffu;
  __syncthreads();
  return sh.bound;
}

// The bound as a number to compare with: every logit but a NaN of that order or a higher one is no smaller.
__device__ __forceinline__ float bound_value(uint32_t bound) {
  return bound <= 0x007fffffu ? __uint_as_float(0xff800000u) : of_order(bound);
}

__device__ __forceinline__ void push(TopShared& sh, uint64_t key) {
  const int i = atomicAdd(&sh.count, 1);  // the order of the list does not matter: its keys are ranked
  if (i < kLgCand) sh.cand[i] = key;
}

// Ranks n unique keys and hands the first `top`, which there are, to out(rank, key).
template <class Out>
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, int top, Out out) {
  for (int c = threadIdx.x; c < n; c += kLgThreads) {
    const uint64_t key = keys[c];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += keys[i] > key;
    if (rank < top) out(rank, key);
  }
}

// The `top` largest keys of the work-group's span, or all of a shorter one with keys 0 behind them.  `mine`: the largest
// order_of() of the thread's elements, or less.
template <int XT, class Out>
__device__ __forceinline__ void span_top(const void* row, const Span& sp, uint32_t mine, int top, TopShared& sh, Out out) {
  const uint32_t bound = bound_of(mine, top, sh);
  if (mine >= bound) sh.owners[atomicAdd(&sh.nowners, 1)] = static_cast<uint8_t>(threadIdx.x);
  __syncthreads();
  // the owners' elements once more, shared out over the whole work-group so that their loads go out together
  constexpr int P = pack_of<XT>();
  const int no = sh.nowners;
  const int items = no * static_cast<int>((sp.pieces + kLgThreads - 1) / kLgThreads);  // at most 2^29 + 2^8
  const uint4* body = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + sp.body * (16 / P));
  const float least = bound_value(bound), per_owner = 1.0f / static_cast<float>(no);
  auto test = [&](float v, int64_t at) {
    if (!(v < least)) push(sh, key_of(v, at));  // with a NaN the row's alternatives are not used
  };
  for (int base = threadIdx.x; base < items; base += 4 * kLgThreads) {
    uint4 t[4];
    int64_t at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // turn and owner of an item; up to 2^22 items the product is off by less than the half that keeps it from the next
      const int item = base + q * kLgThreads;
      const int turn = items < 1 << 22 ? static_cast<int>((static_cast<float>(item) + 0.5f) * per_owner) : item / no;
      const int64_t i = item < items ? sh.owners[item - turn * no] + turn * static_cast<int64_t>(kLgThreads) : sp.pieces;
      at[q] = i < sp.pieces ? i : -1;
      t[q] = body[at[q] < 0 ? 0 : at[q]];  // there is a piece: items > 0
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (at[q] < 0) continue;
      float v[P];
      unpack16<XT>(t[q], v);
#pragma unroll
      for (int j = 0; j < P; ++j) test(v[j], sp.body + at[q] * P + j);
    }
  }
  if (static_cast<int>(threadIdx.x) < sp.singles(P)) {
    const int64_t at = sp.single(threadIdx.x, P);
    test(logit<XT>(row, at), at);
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= kLgCand) {
    rank_keys(sh.cand, n, top, out);
    for (int r = n + threadIdx.x; r < top; r += kLgThreads) out(r, 0);
    return;
  }
  // many equal to the bound: one pass for each alternative, the largest key below the last
  uint64_t last = ~0ull;
  for (int r = 0; r < top; ++r) {
    uint64_t best = 0;
    if (mine >= bound) {
      each_of_mine<XT>(row, sp, [&](float v, int64_t at) {
        const uint64_t key = key_of(v, at);
        if (key < last && key > best) best = key;
      });
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
      const uint64_t o = __shfl_xor(best, s, 64);
      best = o > best ? o : best;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.cand[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kLgThreads / 64; ++w) best = sh.cand[w] > best ? sh.cand[w] : best;
    last = best;
    if (threadIdx.x == 0) out(r, best);
  }
}

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ float nan32() { return __uint_as_float(0x7fc00000u); }

// Whether (m, s) is a distribution's: no NaN, no +infinity, something above -infinity.
__device__ __forceinline__ bool proper(const Stats& st) { return st.s > 0.0f && st.s < __uint_as_float(0x7f800000u); }

// A row's token and its logit, loaded ahead of the pass over the row.
struct TokenLogit {
  int64_t token;
  float x;
  template <int XT>
  __device__ __forceinline__ static TokenLogit of(const LogitArgs& a, int64_t row, const void* xr) {
    const int64_t t = index_at(a.tokens, a.tokens64, row);
    return {t, logit<XT>(xr, t >= 0 && t < a.V ? t : 0)};
  }
};

// log sum exp((x - m) / t) of complete statistics.
__device__ __forceinline__ float log_sum(const Stats& st, float k) {
  const Origin o(st.m, k);
  return logf(st.s) - o.exponent(st.m, k) * kLn2;
}

__device__ __forceinline__ void finish_score(const LogitArgs& a, int64_t row, const TokenLogit& t, const Stats& st) {
  if (threadIdx.x != 0) return;
  const bool ok = proper(st);
  const float ls = ok ? log_sum(st, kLog2e) : nan32();
  a.logp[row] = t.token < 0 ? 0.0f : ok && t.token < a.V ? (t.x - st.m) - ls : nan32();
  a.entropy[row] = ok ? logf(st.s) - st.u / st.s * kLn2 : nan32();
  if (a.norm) a.norm[2 * row] = st.m, a.norm[2 * row + 1] = ls;
}

// ls: log_sum of the row
__device__ __forceinline__ void put_top(const LogitArgs& a, int64_t row, int r, uint64_t key, float m, float ls, bool ok) {
  const float v = of_order(static_cast<uint32_t>(key >> 32));
  a.top_logp[row * a.top + r] = ok ? (v - m) - ls : nan32();
  a.top_ids[row * a.top + r] = ok ? static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key)) : -1;
}

// Whether a teacher entry counts: its token is given and its value is not -infinity.
__device__ __forceinline__ bool kept(int64_t id, float value) { return id >= 0 && value != __uint_as_float(0xff800000u); }

// A teacher's entry: value (-infinity: left out), token and the student's logit there.
struct Entry {
  float v, x;
  bool beyond;
  template <int XT>
  __device__ __forceinline__ static Entry of(const LogitArgs& a, int64_t row, const void* xr, int64_t j) {
    if (j >= a.k) return {__uint_as_float(0xff800000u), 0.0f, false};
    const int64_t id = index_at(a.ids, a.ids64, row * a.k + j);
    const float v = load_as_float(a.values, a.values_dt, row * a.k + j);
    const bool in = id >= 0 && id < a.V;
    return {kept(id, v) ? v : __uint_as_float(0xff800000u), logit<XT>(xr, in ? id : 0), id >= a.V};
  }
  __device__ __forceinline__ bool counts() const { return v != __uint_as_float(0xff800000u); }
};

// The teacher's softmax over a row's kept entries, and the row's loss.  With e_j = exp((v_j - m) / t) and s their sum,
// sum_j p_j (log p_j - log q_j) = sum_j e_j ((v_j - m) / t - log q_j) / s - log s: two reductions.  `first`: the thread's
// first entry, loaded ahead of the pass over the row (the others are loaded where they are used).
template <int XT>
__device__ __forceinline__ void finish_distill(const LogitArgs& a, int64_t row, const void* xr, const Entry& first,
                                               const Stats& st, float (*red)[4]) {
  const float ls = log_sum(st, a.tau_inv * kLog2e), tau = 1.0f / a.tau_inv;
  const float none = __uint_as_float(0xff800000u);
  float m = none;
  auto each = [&](auto f) {
    f(first, static_cast<int64_t>(threadIdx.x));
    for (int64_t j = threadIdx.x + kLgThreads; j < a.k; j += kLgThreads) f(Entry::of<XT>(a, row, xr, j), j);
  };
  each([&](const Entry& e, int64_t) {
    if (e.counts()) m = fmaxf(m, e.v == e.v ? e.v : kLowest);
  });
  m = row_reduce<kLgThreads, true>(m, red[0]);
  float s = 0.0f, w = 0.0f;
  each([&](const Entry& e, int64_t) {
    if (!e.counts()) return;
    const float d = (e.v - m) * a.tau_inv, p = exp_of(d);
    s += p;
    if (p != 0.0f) w += p * (d - (e.beyond ? nan32() : (e.x - st.m) * a.tau_inv - ls));
  });
  block_add2(s, w, red + 1);
  const float r = 1.0f / s;
  each([&](const Entry& e, int64_t j) {
    if (j < a.k) a.p[row * a.k + j] = e.counts() ? exp_of((e.v - m) * a.tau_inv) * r : 0.0f;
  });
  if (threadIdx.x == 0) {
    // a row without entries has no loss, whatever its logits: log s of +infinity marks it.  One whose loss is NaN (its
    // logits', its values' or a token's beyond the vocabulary) has NaN gradients.
    const float loss = proper(st) ? w / s - logf(s) : nan32();
    a.loss[row] = m == none ? 0.0f : loss * tau * tau;
    a.norm[2 * row] = st.m;
    a.norm[2 * row + 1] = m == none ? __uint_as_float(0x7f800000u) : loss == loss ? ls : nan32();
  }
}

// One split of one row: grid (splits, rows).
template <int XT, bool DISTILL>
__global__ __launch_bounds__(kLgThreads) void logits_kernel(const LogitArgs a) {
  __shared__ float red[6][4];
  __shared__ TopShared sh;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const char* xr = static_cast<const char*>(a.x) + row * a.ldx * (XT == DIMQ_F32 ? 4 : 2);
    const int64_t from = blockIdx.x * a.chunk, to = from + a.chunk < a.V ? from + a.chunk : a.V;
    const Span sp = Span::of<XT>(xr, from, to);
    const float k = DISTILL ? a.tau_inv * kLog2e : kLog2e;
    TokenLogit token;
    Entry entry;
    if (a.splits == 1) {
      if constexpr (DISTILL) entry = Entry::of<XT>(a, row, xr, threadIdx.x);
      else token = TokenLogit::of<XT>(a, row, xr);
    }
    const Stats mine = stream_stats<XT, !DISTILL>(xr, sp, k);
    const Stats st = block_stats<!DISTILL>(mine, k, red);
    if (a.splits > 1) {
      if (threadIdx.x == 0) {
        float* to_stats = a.stats + (row * a.splits + blockIdx.x) * 4;
        to_stats[0] = st.m, to_stats[1] = st.s, to_stats[2] = st.u;
      }
    } else if constexpr (DISTILL) {
      finish_distill<XT>(a, row, xr, entry, st, red + 3);
    } else {
      finish_score(a, row, token, st);
    }
    if constexpr (!DISTILL) {
      if (a.top > 0) {
        // the thread's maximum, 0 where it saw nothing above -infinity: a lower bound needs no more, but with fewer than
        // `top` such threads every element is a candidate
        const uint32_t m = mine.s > 0.0f ? order_of(mine.m) : 1u;
        uint64_t* cand = a.cand + (row * a.splits + blockIdx.x) * a.top;
        const bool ok = proper(st);
        if (a.splits > 1) {
          span_top<XT>(xr, sp, m, a.top, sh, [&](int r, uint64_t key) { cand[r] = key; });
        } else if (ok) {
          const float ls = log_sum(st, k);
          span_top<XT>(xr, sp, m, a.top, sh, [&](int r, uint64_t key) { put_top(a, row, r, key, st.m, ls, true); });
        } else {
          for (int r = threadIdx.x; r < a.top; r += kLgThreads) put_top(a, row, r, 0, 0.0f, 0.0f, false);
        }
      }
    }
    __syncthreads();
  }
}

// Joins the splits of a row.
template <int XT, bool DISTILL>
__global__ __launch_bounds__(kLgThreads) void logits_join_kernel(const LogitArgs a) {
  __shared__ float red[6][4];
  __shared__ uint64_t keys[DISTILL ? 1 : kLgSplits * kLgTop];
  __shared__ TopShared sh;
  const int64_t row = blockIdx.x;
  const char* xr = static_cast<const char*>(a.x) + row * a.ldx * (XT == DIMQ_F32 ? 4 : 2);
  Stats st{kLowest, 0.0f, 0.0f};
  if (static_cast<int>(threadIdx.x) < a.splits) {
    const float* from = a.stats + (row * a.splits + threadIdx.x) * 4;
    st = {from[0], from[1], from[2]};
  }
  if constexpr (DISTILL) {
    const Entry entry = Entry::of<XT>(a, row, xr, threadIdx.x);
    st = block_stats<false>(st, a.tau_inv * kLog2e, red);
    finish_distill<XT>(a, row, xr, entry, st, red + 3);
  } else {
    const TokenLogit token = TokenLogit::of<XT>(a, row, xr);
    const int n = a.splits * a.top;
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < n; i += kLgThreads) {
      const uint64_t key = a.cand[row * n + i];
      keys[i] = key;
      mine = key > mine ? key : mine;
    }
    st = block_stats<true>(st, kLog2e, red);
    finish_score(a, row, token, st);
    if (a.top == 0) return;
    if (!proper(st)) {
      for (int r = threadIdx.x; r < a.top; r += kLgThreads) put_top(a, row, r, 0, 0.0f, 0.0f, false);
      return;
    }
    // as in span_top, over the splits' keys: there are at least `top` of them that are not 0
    const uint32_t bound = bound_of(static_cast<uint32_t>(mine >> 32), a.top, sh);
    for (int i = threadIdx.x; i < n; i += kLgThreads) {
      const uint64_t key = keys[i];
      if (key != 0 && static_cast<uint32_t>(key >> 32) >= bound) push(sh, key);
    }
    __syncthreads();
    const float ls = log_sum(st, kLog2e);
    auto put = [&](int r, uint64_t key) { put_top(a, row, r, key, st.m, ls, true); };
    if (sh.count <= kLgCand) rank_keys(sh.cand, sh.count, a.top, put);
    else rank_keys(keys, n, a.top, put);  // zeros rank behind all others
  }
}

// The sum of the rows' losses, or their mean over the rows that keep an entry (0 without any), and what that divides by.  One work-group, a fixed order.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ loss, const float* __restrict__ norm,
                                                           int64_t rows, int mean, float* out, float* divisor) {
  __shared__ float red[2][16];
  float s = 0.0f, n = 0.0f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    s += loss[i];
    n += norm[2 * i + 1] != __uint_as_float(0x7f800000u) ? 1.0f : 0.0f;
  }
  s = row_reduce<1024>(s, red[0]);
  n = row_reduce<1024>(n, red[1]);
  if (threadIdx.x == 0) {
    const float by = mean ? fmaxf(n, 1.0f) : 1.0f;
    out[0] = s / by;
    divisor[0] = by;
  }
}

struct GradArgs {
  const void* x;
  int64_t ldx, rows, V, chunk;
  const float* norm;
  void* gx;
  // scoring
  const void* tokens;
  int tokens64;
  const float* entropy;
  const float* ga;  // [rows], nullable; strides 0 or 1
  const float* gb;
  int64_t sa, sb;
  // distillation
  float tau, tau_inv;
  const void* ids;
  int ids64;
  int k;
  const float* p;
  const float* by;  // nullable
};

// grid (chunks, rows): the gradient of one chunk of a row.
//   scoring        a ([v = token] - p) - b p (log p + H)
//   distillation   tau c (q - p_teacher), the teacher's entries subtracted after the chunk is written
template <int XT, bool DISTILL>
__global__ __launch_bounds__(kLgThreads, 8) void logits_grad_kernel(const GradArgs a) {
  constexpr int P = pack_of<XT>(), kSize = XT == DIMQ_F32 ? 4 : 2;
  for (int64_t turn = blockIdx.y; turn < a.rows; turn += gridDim.y) {
    // The forward pass's last rows first, which may still be in the cache, and gradients stored past it: forward and backward
    // of 2048 x 128000 bf16 take 313 us, in the rows' order 338, with cached stores as well 364.
    const int64_t row = a.rows - 1 - turn;
    const char* xr = static_cast<const char*>(a.x) + row * a.ldx * kSize;
    char* gr = static_cast<char*>(a.gx) + row * a.V * kSize;
    const int64_t from = blockIdx.x * a.chunk, to = from + a.chunk < a.V ? from + a.chunk : a.V;
    const float m = a.norm[2 * row], ls = a.norm[2 * row + 1];
    float ca = a.ga ? a.ga[row * a.sa] : 0.0f, cb = 0.0f, H = 0.0f;
    int64_t token = -1;
    bool none;  // nothing reaches this row, whatever it holds
    if constexpr (DISTILL) {
      ca *= a.tau / (a.by ? a.by[0] : 1.0f);
      none = ls == __uint_as_float(0x7f800000u) || ca == 0.0f;
    } else {
      token = index_at(a.tokens, a.tokens64, row);
      if (token < 0) ca = 0.0f;
      cb = a.gb ? a.gb[row * a.sb] : 0.0f;
      none = ca == 0.0f && cb == 0.0f;
      H = a.entropy[row];
      if (cb == 0.0f) H = 0.0f;
      if (token >= a.V && ca != 0.0f) ca = nan32();
    }
    auto grad = [&](float x, int64_t at) {
      float g;
      if constexpr (DISTILL) {
        g = ca * exp_of(fmaf(x - m, a.tau_inv, -ls));
      } else {
        const float lp = (x - m) - ls, p = exp_of(lp);
        const float t = fmaf(cb, fmaxf(lp, -200.0f) + H, ca);  // p = 0: no 0 * infinity
        g = (at == token ? ca : 0.0f) - p * t;
      }
      return none ? 0.0f : g;
    };
    Span sp = Span::of<XT>(xr, from, to);
    // pieces are written whole only where both rows reach a 16-byte boundary together
    if (((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(gr)) & 15) != 0) {
      for (int64_t i = from + threadIdx.x; i < to; i += kLgThreads)
        store_from_float(gr, XT, i, grad(logit<XT>(xr, i), i));
    } else {
      const uint4* body = reinterpret_cast<const uint4*>(xr + sp.body * kSize);
      uint4* out = reinterpret_cast<uint4*>(gr + sp.body * kSize);
      auto put = [&](int64_t i, const uint4& t) {
        float v[P];
        unpack16<XT>(t, v);
#pragma unroll
        for (int j = 0; j < P; ++j) v[j] = grad(v[j], sp.body + i * P + j);
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (XT == DIMQ_F32) o[j] = __float_as_uint(v[j]);
          else o[j] = XT == DIMQ_F16 ? f16x2_rne(v[2 * j], v[2 * j + 1]) : bf16x2_rne(v[2 * j], v[2 * j + 1]);
        }
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(u4{o[0], o[1], o[2], o[3]}, reinterpret_cast<u4*>(out) + i);
      };
      int64_t i = threadIdx.x;
      for (; i + 3 * kLgThreads < sp.pieces; i += 4 * kLgThreads) {
        uint4 t[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) t[q] = body[i + q * kLgThreads];
#pragma unroll
        for (int q = 0; q < 4; ++q) put(i + q * kLgThreads, t[q]);
      }
      for (; i < sp.pieces; i += kLgThreads) put(i, body[i]);
      if (static_cast<int>(threadIdx.x) < sp.singles(P)) {
        const int64_t at = sp.single(threadIdx.x, P);
        store_from_float(gr, XT, at, grad(logit<XT>(xr, at), at));
      }
    }
    if constexpr (DISTILL) {
      if (none) continue;
      __syncthreads();  // the chunk is written before its entries are written again
      for (int j = threadIdx.x; j < a.k; j += kLgThreads) {
        const int64_t id = index_at(a.ids, a.ids64, row * a.k + j);
        if (id < from || id >= to) continue;
        // the first of equal tokens takes all of their probability
        bool first = true;
        float p = 0.0f;
        for (int i = 0; i < a.k; ++i) {
          if (index_at(a.ids, a.ids64, row * a.k + i) != id) continue;
          if (i < j) first = false;
          p += a.p[row * a.k + i];
        }
        if (first) store_from_float(gr, XT, id, ca * (exp_of(fmaf(logit<XT>(xr, id) - m, a.tau_inv, -ls)) - p));
      }
    }
  }
}

// Splits of a row: one where the rows alone fill the chip (four work-groups a CU), else as many as do, of at least 4,096
// elements.
int row_splits(int64_t rows, int64_t V) {
  const int64_t want = (4 * static_cast<int64_t>(device_cus()) + rows - 1) / rows, most = (V + 4095) / 4096;
  const int64_t n = want < most ? want : most;
  return static_cast<int>(n < 1 ? 1 : n > kLgSplits ? kLgSplits : n);
}
int64_t split_chunk(int64_t V, int splits) { return ((V + splits - 1) / splits + 7) / 8 * 8; }

int64_t up16(int64_t b) { return (b + 15) / 16 * 16; }

bool float_logits(int dt) { return dt == DIMQ_F32 || dt == DIMQ_F16 || dt == DIMQ_BF16; }

int check_logits(const char* what, const void* x, int dtype, int64_t rows, int64_t V, int64_t ldx) {
  DIMQ_CHECK(float_logits(dtype), "%s: logits must be fp32, fp16 or bf16", what);
  DIMQ_CHECK(rows >= 0 && V > 0, "%s: there must be at least one logit a row", what);
  DIMQ_CHECK(V < (int64_t)1 << 31, "%s: rows of 2^31 logits or more are not supported", what);
  DIMQ_CHECK(rows <= 1 || ldx >= V, "%s: row stride is below the row length", what);
  DIMQ_CHECK(rows == 0 || x, "%s: null pointer", what);
  DIMQ_CHECK(aligned(x, dtype_size(dtype)), "%s: misaligned logits", what);
  return DIMQ_OK;
}

template <bool DISTILL>
int launch_rows(const LogitArgs& a, int dtype, hipStream_t s) {
  // a grid's second dimension ends at 65,535: more rows are taken in turn
  const dim3 grid(a.splits, static_cast<unsigned>(a.rows < 65535 ? a.rows : 65535));
  switch (dtype) {
    case DIMQ_F32: hipLaunchKernelGGL((logits_kernel<DIMQ_F32, DISTILL>), grid, dim3(kLgThreads), 0, s, a); break;
    case DIMQ_F16: hipLaunchKernelGGL((logits_kernel<DIMQ_F16, DISTILL>), grid, dim3(kLgThreads), 0, s, a); break;
    default: hipLaunchKernelGGL((logits_kernel<DIMQ_BF16, DISTILL>), grid, dim3(kLgThreads), 0, s, a);
  }
  if (a.splits > 1) {
    const dim3 one(static_cast<unsigned>(a.rows));
    switch (dtype) {
      case DIMQ_F32: hipLaunchKernelGGL((logits_join_kernel<DIMQ_F32, DISTILL>), one, dim3(kLgThreads), 0, s, a); break;
      case DIMQ_F16: hipLaunchKernelGGL((logits_join_kernel<DIMQ_F16, DISTILL>), one, dim3(kLgThreads), 0, s, a); break;
      default: hipLaunchKernelGGL((logits_join_kernel<DIMQ_BF16, DISTILL>), one, dim3(kLgThreads), 0, s, a);
    }
  }
  return check_launch(DISTILL ? "top_logits_distillation_loss" : "token_logprobs");
}

template <bool DISTILL>
int launch_grad(GradArgs& a, int dtype, hipStream_t s) {
  // chunks of at least 8,192 elements, and enough of them for four work-groups a CU
  const int64_t want = (4 * static_cast<int64_t>(device_cus()) + a.rows - 1) / a.rows, most = (a.V + 8191) / 8192;
  const int64_t n = want < 1 ? 1 : want < most ? want : most;
  a.chunk = split_chunk(a.V, static_cast<int>(n));
  const dim3 grid(static_cast<unsigned>((a.V + a.chunk - 1) / a.chunk), static_cast<unsigned>(a.rows < 65535 ? a.rows : 65535));
  switch (dtype) {
    case DIMQ_F32: hipLaunchKernelGGL((logits_grad_kernel<DIMQ_F32, DISTILL>), grid, dim3(kLgThreads), 0, s, a); break;
    case DIMQ_F16: hipLaunchKernelGGL((logits_grad_kernel<DIMQ_F16, DISTILL>), grid, dim3(kLgThreads), 0, s, a); break;
    default: hipLaunchKernelGGL((logits_grad_kernel<DIMQ_BF16, DISTILL>), grid, dim3(kLgThreads), 0, s, a);
  }
  return check_launch(DISTILL ? "top_logits_distillation_loss backward" : "token_logprobs backward");
}

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int64_t dimq_logits_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0) return 0;
  const int splits = row_splits(rows, vocab);
  return splits == 1 ? 0 : up16(rows * splits * 16) + up16(rows * splits * static_cast<int64_t>(top) * 8);
}

extern "C" int dimq_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ldx, const void* tokens,
                                   int tokens64, int top, float* logprobs, float* entropy, float* norm, float* top_logprobs,
                                   int64_t* top_ids, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_logits("token_logprobs", logits, dtype, rows, vocab, ldx);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(top >= 0 && top <= kLgTop && top <= vocab, "token_logprobs: top must be in [0, %d] and not above the vocabulary",
             kLgTop);
  if (rows == 0) return DIMQ_OK;
  DIMQ_CHECK(tokens && logprobs && entropy && (top == 0 || (top_logprobs && top_ids)), "token_logprobs: null pointer");
  DIMQ_CHECK(workspace_bytes >= dimq_logits_workspace_bytes(rows, vocab, top) && aligned(workspace, 16),
             "token_logprobs: the workspace is too small or not 16-byte aligned");
  LogitArgs a{};
  a.x = logits, a.ldx = ldx, a.rows = rows, a.V = vocab;
  a.splits = row_splits(rows, vocab);
  a.chunk = split_chunk(vocab, a.splits);
  a.tau_inv = 1.0f, a.tokens = tokens, a.tokens64 = tokens64, a.top = top;
  a.logp = logprobs, a.entropy = entropy, a.norm = norm, a.top_logp = top_logprobs, a.top_ids = top_ids;
  a.stats = static_cast<float*>(workspace);
  a.cand = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + up16(rows * a.splits * 16));
  return launch_rows<false>(a, dtype, as_stream(stream));
}

extern "C" int dimq_token_logprobs_backward(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ldx,
                                            const void* tokens, int tokens64, const float* norm, const float* entropy,
                                            const float* grad_logprobs, int64_t stride_logprobs, const float* grad_entropy,
                                            int64_t stride_entropy, void* grad_logits, void* stream) {
  const int rc = check_logits("token_logprobs backward", logits, dtype, rows, vocab, ldx);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0) return DIMQ_OK;
  DIMQ_CHECK(tokens && norm && entropy && grad_logits, "token_logprobs backward: null pointer");
  GradArgs a{};
  a.x = logits, a.ldx = ldx, a.rows = rows, a.V = vocab, a.norm = norm, a.gx = grad_logits;
  a.tokens = tokens, a.tokens64 = tokens64, a.entropy = entropy;
  a.ga = grad_logprobs, a.sa = stride_logprobs, a.gb = grad_entropy, a.sb = stride_entropy;
  return launch_grad<false>(a, dtype, as_stream(stream));
}

extern "C" int dimq_distill_loss(const void* student, int dtype, int64_t rows, int64_t vocab, int64_t ldx, const void* values,
                                 int values_dtype, const void* ids, int ids64, int64_t k, double temperature, int reduction,
                                 float* row_loss, float* loss, float* divisor, float* norm, float* p,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_logits("top_logits_distillation_loss", student, dtype, rows, vocab, ldx);
  if (rc != DIMQ_OK) return rc;
  DIMQ_CHECK(float_logits(values_dtype), "top_logits_distillation_loss: teacher values must be fp32, fp16 or bf16");
  DIMQ_CHECK(k >= 0 && k <= kMostEntries, "top_logits_distillation_loss: at most %d teacher entries a row",
             static_cast<int>(kMostEntries));
  // t^2 multiplies what fp32 leaves of a difference of logarithms
  DIMQ_CHECK(temperature >= 1e-3 && temperature <= 1e3,
             "top_logits_distillation_loss: the temperature must be in [0.001, 1000]");
  DIMQ_CHECK(reduction >= 0 && reduction <= 2, "top_logits_distillation_loss: unknown reduction");
  const hipStream_t s = as_stream(stream);
  if (rows > 0) {
    DIMQ_CHECK(row_loss && norm && (k == 0 || (values && ids && p)), "top_logits_distillation_loss: null pointer");
    DIMQ_CHECK(workspace_bytes >= dimq_logits_workspace_bytes(rows, vocab, 0) && aligned(workspace, 16),
               "top_logits_distillation_loss: the workspace is too small or not 16-byte aligned");
    LogitArgs a{};
    a.x = student, a.ldx = ldx, a.rows = rows, a.V = vocab;
    a.splits = row_splits(rows, vocab);
    a.chunk = split_chunk(vocab, a.splits);
    a.tau_inv = static_cast<float>(1.0 / temperature);
    a.values = values, a.values_dt = values_dtype, a.ids = ids, a.ids64 = ids64, a.k = static_cast<int>(k);
    a.loss = row_loss, a.norm = norm, a.p = p, a.stats = static_cast<float*>(workspace);
    const int r = launch_rows<true>(a, dtype, s);
    if (r != DIMQ_OK) return r;
  }
  if (reduction != 0) {
    DIMQ_CHECK(loss && divisor, "top_logits_distillation_loss: null pointer");
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, s, row_loss, norm, rows, reduction == 1, loss, divisor);
  }
  return check_launch("top_logits_distillation_loss");
}

extern "C" int dimq_distill_loss_backward(const void* student, int dtype, int64_t rows, int64_t vocab, int64_t ldx,
                                          const void* ids, int ids64, int64_t k, const float* p, const float* norm,
                                          double temperature, const float* grad, int64_t grad_stride, const float* divisor,
                                          void* grad_student, void* stream) {
  const int rc = check_logits("top_logits_distillation_loss backward", student, dtype, rows, vocab, ldx);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0) return DIMQ_OK;
  DIMQ_CHECK(k >= 0 && k <= kMostEntries && (k == 0 || (ids && p)) && norm && grad && grad_student,
             "top_logits_distillation_loss backward: null pointer or too many entries");
  GradArgs a{};
  a.x = student, a.ldx = ldx, a.rows = rows, a.V = vocab, a.norm = norm, a.gx = grad_student;
  a.ga = grad, a.sa = grad_stride, a.tau = static_cast<float>(temperature), a.tau_inv = static_cast<float>(1.0 / temperature);
  a.ids = ids, a.ids64 = ids64, a.k = static_cast<int>(k), a.p = p, a.by = divisor;
  return launch_grad<true>(a, dtype, as_stream(stream));
}
