// The next token of each row of logits, from a given random number.
//
//   w_i = exp((x_i - max x) / t); ordered by x descending, ties to the lower index, the first top_k
//   are kept, of these the shortest run whose sum reaches top_p of theirs, of these w_i >= min_p;
//   the draw is the lowest index i at which the running sum of the kept weights, in the vocabulary's
//   order, exceeds u times their sum.  t = 0: the largest logit's lowest index.
//
// Every cut keeps a run of that order, so the kept set is "x above a border, and the first m of those at
// it": top_k and top_p each give a border (a logit and a number), min_p a logit; the tightest holds.
//
// A workgroup a row.  The first pass takes each thread's two largest.  top_k <= 2048 gets a lower bound of
// its border from those; top_p alone gets one from a histogram of the row's weights over the distance from
// the maximum, which gives their sum as well; min_p is one.  The logits above the bound, usually few, are
// gathered into LDS, and all else is done there: up to 256 by comparing each with each.  Where more than
// 8192 are above it, top_p's border comes from the logits of its bin; where there is no bound, the same
// code reads the row again.
//
// A border is found by a radix search, 11 bits a round, in a histogram in LDS of how many keys, or how much
// weight, each value of the bits has; a draw from what was gathered is the same search over the
// indices, one from the row takes the sums of 256 tokens each.  Weights are summed as whole numbers of 2^-40:
// sums do not depend on their order, so neither does the token.
//
// What bounds it: a row's passes by one CU's vector work, not the card's memory.  Of 73448 float32 logits, 2.4
// GHz: the largest ones 13 thousand cycles (5 us), the histogram 44 (a weight is some 25 instructions in 64
// bits, and an addition in LDS), a gather 16, all of up to 256 by comparison 16, the draw from the row 60.  One
// row with top-k 50 and top-p takes 24 us, 16 rows of bf16 with top-p and min-p 40, 256 rows of mixed
// settings 93 (0.8 TB/s); a greedy row 15, 256 of them 24 (3.1 TB/s).  Several workgroups a row would
// have to join their sums through memory, a launch or a wait at each of the cuts; a row stays with one.
//
// The reference draws with torch's multinomial on the host's settings; it has no such kernel.
#include <algorithm>
#include <type_traits>

#include "ls_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 8192;
constexpr int kFew = 256;
constexpr int kBounded = 2048;   // the largest top_k that gets a bound from the threads' two largest
constexpr int kSlot = 4 * kThreads;  // tokens of a round over the row
constexpr int kIndexBits = 19;
constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;
static_assert((1 << kIndexBits) / kSlot * kWaves <= kBins, "a bin for what a wave takes in each round");
constexpr int kShift = 40;       // weights are whole numbers of 2^-40: a row's sum is 2^59 at most
static_assert(kBounded <= 2 * kThreads, "");

struct SaArgs {
  const void* x;
  int64_t rs;
  int64_t rows;
  int vocab;
  const float* u;
  double t, top_p, min_p;
  int top_k;
  const float* ts;  // per row, or NULL
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  int32_t* tokens;
  float* logprobs;
};

// Logits in their order as whole numbers (-0 as 0).
__device__ __forceinline__ uint32_t sa_key(float x) { return ls_order_key32(__float_as_uint(x == 0.f ? 0.f : x)); }
__device__ __forceinline__ float sa_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// The next smaller logit (-inf: itself).  Below 0 stands the largest negative one: the key between them is -0's.
__device__ __forceinline__ float sa_below(float x) {
  const uint32_t key = sa_key(x);
  return x > -INFINITY ? sa_value(key - (key == 0x80000000u ? 2 : 1)) : x;
}

__device__ __forceinline__ uint64_t sa_lane64(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32;
}
// Inclusive sum over the lanes up to this one, by shifts within rows of 16 and broadcasts of their last.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t sa_dpp64(uint64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, true);
  return (uint64_t)lo | (uint64_t)hi << 32;
}
__device__ __forceinline__ uint64_t sa_upto64(uint64_t x) {
  x += sa_dpp64<0x111, 0xf>(x);
  x += sa_dpp64<0x112, 0xf>(x);
  x += sa_dpp64<0x114, 0xf>(x);
  x += sa_dpp64<0x118, 0xf>(x);
  x += sa_dpp64<0x142, 0xa>(x);
  x += sa_dpp64<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ uint64_t sa_add64(uint64_t x) { return sa_lane64(sa_upto64(x), 63); }

struct SaShared {
  unsigned long long bins[kBins];
  unsigned long long part[kWaves];
  double table[64];
  unsigned long long found;
  uint32_t at;
  uint32_t n;
  uint32_t word[kWaves];
  float x[kList];
  uint32_t index[kList];
};

// A row in memory.  f(index, logit) for this thread's; NaN as -inf, which is also what lies beyond the last.
template <int DT>
struct SaRow {
  typedef typename LsElem<DT>::T T;
  typedef typename std::conditional<DT == LS_F32, ls_f32x4, uint2>::type T4;
  const T* x;
  int vocab;
  bool wide;  // four may be read at once

  __device__ __forceinline__ float one(int i) const { return i < vocab ? LsElem<DT>::to_f(x[i]) : -INFINITY; }
  __device__ __forceinline__ ls_f32x4 load4(int i) const {
    ls_f32x4 v;
    if (wide && i + 4 <= vocab) {
      const T4 w = *reinterpret_cast<const T4*>(x + i);
      if constexpr (DT == LS_F32)
        v = w;
      else
        v = ls_f32x4{LsElem<DT>::to_f((T)(w.x & 0xffffu)), LsElem<DT>::to_f((T)(w.x >> 16)),
                     LsElem<DT>::to_f((T)(w.y & 0xffffu)), LsElem<DT>::to_f((T)(w.y >> 16))};
    } else {
      v = ls_f32x4{one(i), one(i + 1), one(i + 2), one(i + 3)};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaxf(v[e], -INFINITY);
    return v;
  }
  // Two rounds' loads ahead of the one in hand.
  template <class F>
  __device__ __forceinline__ void each4(F f) const {
    int i = 4 * (int)threadIdx.x;
    ls_f32x4 a = load4(i), b = load4(i + kSlot);
#pragma unroll 2
    for (int i0 = 0; i0 < vocab; i0 += kSlot, i += kSlot) {
      const ls_f32x4 c = load4(i + 2 * kSlot);
      f(i, a);
      a = b;
      b = c;
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    each4([&](int i, const ls_f32x4& v) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(i + e, v[e]);
    });
  }
};

// What was gathered.
struct SaList {
  const float* x;
  const uint32_t* index;
  int n;
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const int i = i0 + (int)threadIdx.x;
      const bool in = i < n;
      f(in ? (int)index[i] : 0x7fffffff, in ? x[i] : -INFINITY);
    }
  }
};

__device__ __forceinline__ uint32_t sa_max(uint32_t x, SaShared& s) {
  x = ls_wave_max_u32(x);
  __syncthreads();
  if (ls_lane() == 0) s.word[threadIdx.x >> 6] = x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) x = max(x, s.word[i]);
  return x;
}
__device__ __forceinline__ uint64_t sa_sum(uint64_t x, SaShared& s) {
  x = sa_add64(x);
  __syncthreads();
  if (ls_lane() == 0) s.part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) x += s.part[i];
  return x;
}

__device__ __forceinline__ void sa_clear(SaShared& s) {
  __syncthreads();
  s.bins[threadIdx.x] = s.bins[threadIdx.x + kThreads] = 0;
  __syncthreads();
}
// The bin, from the top one, at which the running sum reaches `want` (0 < want <= all); `before`: the sum
// of those above it.
__device__ __forceinline__ uint32_t sa_find(SaShared& s, uint64_t want, uint64_t& before) {
  const int tid = threadIdx.x, wave = tid >> 6;
  __syncthreads();
  const int hi = kBins - 1 - 2 * tid;
  const uint64_t b0 = s.bins[hi], b1 = s.bins[hi - 1], upto = sa_upto64(b0 + b1);
  if (ls_lane() == 63) s.part[wave] = upto;
  __syncthreads();
  uint64_t x = upto - (b0 + b1);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) x += i < wave ? s.part[i] : 0;
  if (x < want && x + b0 + b1 >= want) {
    const bool first = x + b0 >= want;
    s.at = first ? hi : hi - 1;
    s.found = first ? x : x + b0;
  }
  __syncthreads();
  before = s.found;
  return s.at;
}

// The largest c such that the measures of the entries with order(index, logit) >= c sum up to `need` at least
// (0 < need <= all; a measure of 0 does not count); `above`: the sum of those > c.
template <int BITS, class Row, class Order, class Measure>
__device__ __forceinline__ uint32_t sa_border(const Row& row, SaShared& s, uint64_t need, uint64_t& above,
                                              Order order, Measure measure) {
  uint32_t prefix = 0;
  above = 0;
#pragma unroll 1
  for (int left = BITS; left > 0;) {
    const int bits = min(left, 11), low = left - bits;
    const uint32_t mask = left == 32 ? 0u : ~0u << left;
    sa_clear(s);
    row.each([&](int i, float x) {
      const uint32_t o = order(i, x);
      const uint64_t w = measure(i, x);
      if (w != 0 && (o & mask) == prefix) atomicAdd(&s.bins[o >> low & ((1u << bits) - 1)], (unsigned long long)w);
    });
    uint64_t before;
    prefix |= sa_find(s, need - above, before) << low;
    above += before;
    left = low;
  }
  return prefix;
}

// A row's settings, and what a logit weighs.
struct SaRule {
  float top;
  double inv;         // 1 / temperature
  double scale;       // a weight's base-2 exponent: scale (x - top)
  int k;          // 0: none
  double p;
  float min_cut;  // logits above it pass min_p
  const double* table;

  // 2^y in whole numbers of 2^-40, y = m / 64 + f: a table of 2^(k / 64), and 2^f to the fourth power (|f| <
  // 2^-7: 2^-44).  Rounding to m, and of the result, by adding a number that leaves no smaller bits.  The
  // difference is formed first (exact, or off by 2^-53 of itself): scale x and scale top would each round by
  // 2^-53 of what a common offset makes of them.
  __device__ __forceinline__ uint64_t weight(float x) const {
    const double y = fmax(((double)x - (double)top) * scale, -60.0);
    const double m = y + 0x1.8p46, f = y - (m - 0x1.8p46);
    const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, m);  // 64 y, rounded
    double q = fma(f, 0.0096181291076284771619, 0.055504108664821579953);
    q = fma(f, q, 0.24022650695910071233);
    q = fma(f, q, 0.69314718055994530942);
    q = fma(f, q, 1.0);
    const double w = ldexp(q * table[k & 63], (k >> 6) + kShift) + 0x1p52;
    const uint64_t whole = __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull;
    return x == top ? 1ull << kShift : top < INFINITY ? whole : 0;
  }
  // ln of the weight.
  __device__ __forceinline__ double log_weight(float x) const {
    return x == top ? 0.0 : ((double)x - (double)top) * inv;
  }
  // ln of its share of a sum.
  __device__ __forceinline__ float share(float x, uint64_t sum) const {
    return (float)(log_weight(x) - log(ldexp((double)sum, -kShift)));
  }
  __device__ __forceinline__ uint64_t need(uint64_t total) const {
    return max((uint64_t)ceil(p * (double)total), (uint64_t)1);
  }
  // u sum < a running sum  <=>  floor(u sum) < it, a whole number.
  __device__ __forceinline__ static uint64_t goal(double u, uint64_t sum) {
    const uint64_t g = u > 0.0 ? (uint64_t)(u * (double)sum) : 0;
    return g < sum ? g : sum - 1;
  }
};

// Kept are the logits above `cut`, and the first `ties` of those at it: with an index up to `last`.
struct SaKept {
  float cut;
  uint32_t last;
  uint64_t ties;
  __device__ __forceinline__ bool operator()(int i, float x) const {
    return x > cut || (ties != 0 && x == cut && (uint32_t)i <= last);
  }
  __device__ __forceinline__ void above(float c) {
    if (c >= cut) cut = c, ties = 0;
  }
};

__device__ __forceinline__ uint32_t sa_by_index(int i, float) { return ~(uint32_t)i & kIndexMask; }  // lowest first
__device__ __forceinline__ uint32_t sa_by_logit(int, float x) { return sa_key(x); }

// `last`, from a row or list that has all logits at the border.
template <class Row>
__device__ __forceinline__ void sa_last(const Row& row, SaShared& s, SaKept& kept) {
  kept.last = 0x7fffffff;
  if (kept.ties == 0) return;
  uint64_t n = 0, above;
  row.each([&](int, float x) { n += x == kept.cut; });
  n = sa_sum(n, s);
  if (n > kept.ties)
    kept.last = ~sa_border<kIndexBits>(row, s, kept.ties, above, sa_by_index,
                                       [&](int, float x) -> uint64_t { return x == kept.cut ? 1 : 0; }) &
                kIndexMask;
}

// What top_p keeps: the logits from a border, found in a row or list of which `counts` says what is summed
// up; the sum of all larger ones is `front`.
template <class Row, class Counts>
__device__ __forceinline__ void sa_top_p(const Row& row, SaShared& s, const SaRule& rule, uint64_t need, uint64_t front,
                                         SaKept& kept, Counts counts) {
  uint64_t above;
  const float c = sa_value(sa_border<32>(row, s, need - front, above, sa_by_logit, [&](int, float x) -> uint64_t {
    const uint64_t w = rule.weight(x);
    return counts(x) ? w : 0;
  }));
  const uint64_t w = rule.weight(c), n = (need - front - above + w - 1) / w;
  if (c > kept.cut || n < kept.ties) kept.cut = c, kept.ties = n;
}

// The cuts over the row or what was gathered of it.  `total`: the weights of the whole row, for top_p without
// top_k.
template <class Row>
__device__ __forceinline__ SaKept sa_cuts(const Row& row, SaShared& s, const SaRule& rule, uint64_t total) {
  SaKept kept{-INFINITY, 0x7fffffff, 0};
  if (rule.k > 0) {
    uint64_t n = 0, above;
    row.each([&](int, float x) { n += x > -INFINITY; });
    n = sa_sum(n, s);
    if (n > (uint64_t)rule.k) {
      kept.cut = sa_value(sa_border<32>(row, s, rule.k, above, sa_by_logit,
                                        [&](int, float x) -> uint64_t { return x > -INFINITY ? 1 : 0; }));
      kept.ties = rule.k - above;
    }
  }
  if (rule.p < 1.0) {
    const uint64_t at_cut = rule.weight(kept.cut);
    uint64_t here = 0;
    row.each([&](int, float x) {
      const uint64_t w = rule.weight(x);
      here += x > kept.cut ? w : 0;
    });
    here = sa_sum(here, s) + kept.ties * at_cut;
    const uint64_t need = rule.need(rule.k > 0 ? here : total);
    if (need <= here)  // (else more than what is here is kept)
      sa_top_p(row, s, rule, need, 0, kept, [&](float x) { return x > kept.cut || (x == kept.cut && kept.ties); });
  }
  kept.above(rule.min_cut);
  sa_last(row, s, kept);
  return kept;
}

// The draw.
template <class Row>
__device__ __forceinline__ void sa_draw(const Row& row, SaShared& s, const SaRule& rule, const SaKept& kept, double u,
                                        int32_t* token, float* logprob) {
  uint64_t above;
  auto measure = [&](int i, float x) -> uint64_t {
    const bool k = kept(i, x);
    return __any(k) ? (k ? rule.weight(x) : 0) : 0;
  };
  auto answer = [&](uint32_t i, float x, uint64_t sum) {
    *token = (int32_t)i;
    if (logprob) *logprob = rule.share(x, sum);
  };
  if (std::is_same<Row, SaList>::value || !(u > 0.0)) {
    uint64_t sum = 0;
    row.each([&](int i, float x) { sum += measure(i, x); });
    sum = sa_sum(sum, s);
    // (u = 0: the lowest index with any weight, however small)
    auto any = [&](int i, float x) -> uint64_t { return kept(i, x) && rule.log_weight(x) > -745.0 ? 1 : 0; };
    const uint32_t i = ~(u > 0.0 ? sa_border<kIndexBits>(row, s, rule.goal(u, sum) + 1, above, sa_by_index, measure)
                                 : sa_border<kIndexBits>(row, s, 1, above, sa_by_index, any)) &
                       kIndexMask;
    row.each([&](int j, float x) {
      if ((uint32_t)j == i) answer(i, x, sum);
    });
    return;
  }
  if constexpr (!std::is_same<Row, SaList>::value) {
    // The sums of what a wave takes in each round, 256 tokens in a row; then the one in which u falls.
    const int tid = threadIdx.x, wave = tid >> 6, rounds = (row.vocab + kSlot - 1) / kSlot;
    sa_clear(s);
    row.each4([&](int i, const ls_f32x4& x) {
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += measure(i + e, x[e]);
      sum = sa_add64(sum);
      if (ls_lane() == 0) s.bins[kBins - 1 - (i / kSlot * kWaves + wave)] = sum;
    });
    __syncthreads();
    const uint64_t sum = sa_sum(s.bins[tid] + s.bins[tid + kThreads], s);
    const uint64_t goal = rule.goal(u, sum);
    const uint32_t bin = kBins - 1 - sa_find(s, goal + 1, above);
    if ((int)(bin % kWaves) != wave || (int)(bin / kWaves) >= rounds) return;
    const int i = (int)(bin / kWaves) * kSlot + 4 * tid;
    const ls_f32x4 x = row.load4(i);
    uint64_t w[4], mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) mine += w[e] = measure(i + e, x[e]);
    uint64_t before = above + sa_upto64(mine) - mine;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (before <= goal && goal < before + w[e]) answer(i + e, x[e], sum);
      before += w[e];
    }
  }
}

// All of it for at most kFew gathered logits, one a thread: what is in front of it in either order is found
// by looking at each of the others.  WAVE: at most 64, by the first wave from its lanes.
template <bool WAVE>
__device__ __forceinline__ void sa_draw_few(int n, SaShared& s, const SaRule& rule, uint64_t total, double u,
                                            int32_t* token, float* logprob) {
  const int tid = threadIdx.x;
  if (WAVE && tid >= 64) return;
  const bool in = tid < n;
  const float x = in ? s.x[tid] : -INFINITY;
  const uint32_t i = in ? s.index[tid] : 0x7fffffffu;
  const uint64_t w = WAVE || tid < kFew ? rule.weight(x) : 0;
  if (!WAVE) {
    if (tid < kFew) s.bins[tid] = w;
    __syncthreads();
  }
  auto add = [&](uint64_t v) { return WAVE ? sa_add64(v) : sa_sum(v, s); };
  uint32_t rank = 0;
  uint64_t before = 0;
  if (WAVE || in) {
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const float xj = WAVE ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), j)) : s.x[j];
      const uint32_t ij = WAVE ? (uint32_t)__builtin_amdgcn_readlane((int)i, j) : s.index[j];
      const bool first = xj > x || (xj == x && ij < i);
      rank += first;
      before += first ? (WAVE ? sa_lane64(w, j) : s.bins[j]) : 0;
    }
  }
  bool kept = in && x > -INFINITY && (rule.k == 0 || rank < (uint32_t)rule.k);
  if (rule.p < 1.0) {
    if (rule.k > 0) total = add(kept ? w : 0);
    kept = kept && before < rule.need(total);
  }
  kept = kept && x > rule.min_cut;
  const uint64_t sum = add(kept ? w : 0);
  // u = 0: the lowest index with any weight, however small.
  const uint64_t m = !kept ? 0 : u > 0.0 ? w : rule.log_weight(x) > -745.0 ? 1 : 0;
  if (!WAVE) {
    if (tid < kFew) s.bins[tid] = m;
    __syncthreads();
    if (m == 0) return;
  }
  const uint64_t goal = u > 0.0 ? rule.goal(u, sum) : 0;
  before = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const uint32_t ij = WAVE ? (uint32_t)__builtin_amdgcn_readlane((int)i, j) : s.index[j];
    before += ij < i ? (WAVE ? sa_lane64(m, j) : s.bins[j]) : 0;
  }
  if (before <= goal && goal < before + m) {
    *token = (int32_t)i;
    if (logprob) *logprob = rule.share(x, sum);
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void ls_sample_kernel(const SaArgs a) {
  __shared__ SaShared s;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  SaRow<DT> row;
  row.x = (const typename LsElem<DT>::T*)a.x + r * a.rs;
  row.vocab = a.vocab;
  row.wide = ((uintptr_t)row.x & (DT == LS_F32 ? 15 : 7)) == 0;
  if (tid < 64) s.table[tid] = exp2((double)tid / 64.0);
  float best[2] = {-INFINITY, -INFINITY};
  row.each([&](int, float x) {
    best[1] = __builtin_amdgcn_fmed3f(best[0], best[1], x);
    best[0] = fmaxf(best[0], x);
  });
  SaRule rule;
  rule.top = sa_value(sa_max(sa_key(best[0]), s));
  const double t = a.ts ? (double)a.ts[r] : a.t;
  int32_t* token = a.tokens + r;
  float* logprob = a.logprobs ? a.logprobs + r : nullptr;
  if (!(rule.top > -INFINITY) || !(t > 0.0)) {
    // Nothing to draw from, or the lowest index of the largest.
    uint32_t first = 0;
    if (rule.top > -INFINITY)
      row.each([&](int i, float x) { first = x == rule.top ? max(first, ~(uint32_t)i) : first; });
    first = sa_max(first, s);
    if (tid == 0) {
      *token = (int32_t)~first;  // (0: -1)
      if (logprob) *logprob = first ? 0.f : -INFINITY;
    }
    return;
  }
  rule.inv = 1.0 / t;
  rule.scale = 1.4426950408889634074 / t;
  rule.table = s.table;
  rule.k = a.top_ks ? a.top_ks[r] : a.top_k;
  if (rule.k <= 0 || rule.k >= a.vocab) rule.k = 0;
  rule.p = a.top_ps ? (double)a.top_ps[r] : a.top_p;
  rule.min_cut = -INFINITY;
  const double min_p = a.min_ps ? (double)a.min_ps[r] : a.min_p;
  if (min_p > 0.0) {
    // exp((x - max) / t) >= min_p  <=>  x >= max + t ln min_p; the next logit below passes not.
    const double border = (double)rule.top + log(min_p) * t;
    const float f = fminf((float)border, rule.top);
    if (f > -INFINITY) rule.min_cut = (double)f < border && f < rule.top ? f : sa_below(f);
  }
  const double u = (double)a.u[r];
  // What is kept, or has to be summed up, is among the logits above `low`.
  float low = -INFINITY;
  uint64_t total = 0, need = 0, front = 0;
  float to_bins = 0.f;
  int border = 0;  // the bin in which top_p's border lies; `front`: the weights of those before it
  auto bin_of = [&](float x) {  // (falls as x rises)
    const float d = (rule.top - x) * to_bins;
    return d < kBins - 1 ? (int)d : kBins - 1;
  };
  bool bounded = false;
  if (rule.k > 0 && rule.k <= kBounded) {
    // Each thread's largest (and second) are top_k or more in all; the border among them, by bins, is a bound.
    const float least = sa_value(~sa_max(~sa_key(rule.k <= kThreads ? best[0] : best[1]), s));
    const float range = rule.top - least;
    bounded = true;
    low = sa_below(least);
    to_bins = (kBins - 2) / range;
    // (else one value, infinities, or a range so small that its bins' width is none: the least alone is the bound)
    if (range < INFINITY && to_bins < INFINITY) {
      sa_clear(s);
#pragma unroll
      for (int m = 0; m < 2; ++m)
        if (best[m] >= least) atomicAdd(&s.bins[kBins - 1 - bin_of(best[m])], 1ull);
      uint64_t before;
      const uint32_t bin = kBins - 1 - sa_find(s, rule.k, before);
      // (two bins and a step more: theirs are rounded products, and the difference may be rounded up to a logit)
      low = fmaxf(low, sa_below(rule.top - (bin + 2) / to_bins));
    }
  } else if (rule.k == 0 && rule.p < 1.0) {
    // Bins of 1/64 of a temperature, or more where float32 does not hold so large a factor (the largest logit's
    // distance, 0, times infinity would be none): beyond the last no logit has any weight.
    to_bins = (float)fmin(64.0 / t, 0x1.fffffep127);
    sa_clear(s);
    row.each([&](int, float x) {
      const uint64_t w = rule.weight(x);
      if (w != 0) atomicAdd(&s.bins[kBins - 1 - bin_of(x)], (unsigned long long)w);
    });
    __syncthreads();
    total = sa_sum(s.bins[tid] + s.bins[tid + kThreads], s);
    need = min(rule.need(total), total);
    border = kBins - 1 - (int)sa_find(s, need, front);
    // (two bins and a step more: theirs are rounded products; the last is open)
    const float f = border < kBins - 1 ? rule.top - (border + 2) / to_bins : -INFINITY;
    low = sa_below(f);
    bounded = true;
  }
  // (What top_p sums up is more than what min_p leaves.)
  if (!(rule.k > 0 && rule.p < 1.0)) {
    low = fmaxf(low, rule.min_cut);
    bounded = bounded || rule.min_cut > -INFINITY;
  }
  low = fminf(low, sa_below(rule.top));  // (the largest are kept whatever the settings hold)
  // Logits into LDS, a wave's in one go.
  auto gather = [&](auto take) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    bool full = false;
    row.each4([&](int i, const ls_f32x4& x) {
      bool t4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) t4[e] = take(x[e]);
      if (!__any(t4[0] | t4[1] | t4[2] | t4[3]) || full) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t mask = __ballot(t4[e]);
        uint32_t n = 0;
        if (ls_lane() == 0 && mask != 0) n = atomicAdd(&s.n, (uint32_t)__popcll(mask));
        n = __builtin_amdgcn_readfirstlane(n);
        full = n > kList;  // (one more than fits is all that matters)
        n += ls_lanes_below(mask);
        if (t4[e] && n < kList) s.x[n] = x[e], s.index[n] = (uint32_t)(i + e);
      }
    });
    __syncthreads();
    return (int)s.n;
  };
  if (bounded) {
    const int n = gather([&](float x) { return x > low; });
    if (n <= 64) {
      sa_draw_few<true>(n, s, rule, total, u, token, logprob);
      return;
    }
    if (n <= kFew) {
      sa_draw_few<false>(n, s, rule, total, u, token, logprob);
      return;
    }
    if (n <= kList) {
      const SaList list{s.x, s.index, n};
      sa_draw(list, s, rule, sa_cuts(list, s, rule, total), u, token, logprob);
      return;
    }
  }
  if (need > 0) {
    // Only the border's bin; where too many logits are in it, in bins of 1/2048 of it.
    const float from = (float)border, to = border < kBins - 1 ? from + 1.f : INFINITY;
    auto in_bin = [&](float x) {  // bin_of(x) == border
      const float d = (rule.top - x) * to_bins;
      return !(d < from) && !(d >= to) && x > -INFINITY;
    };
    int n = gather(in_bin), sub = -1;
    auto sub_of = [&](float x) {
      const float d = ((rule.top - x) * to_bins - from) * kBins;
      return d < kBins - 1 ? max((int)d, 0) : kBins - 1;
    };
    if (n > kList) {
      sa_clear(s);
      row.each([&](int, float x) {
        const uint64_t w = rule.weight(x);
        if (w != 0 && in_bin(x)) atomicAdd(&s.bins[kBins - 1 - sub_of(x)], (unsigned long long)w);
      });
      uint64_t before;
      sub = kBins - 1 - (int)sa_find(s, need - front, before);
      front += before;
      n = gather([&](float x) { return in_bin(x) && sub_of(x) == sub; });
    }
    if (n <= kList) {
      const SaList list{s.x, s.index, n};
      SaKept kept{-INFINITY, 0x7fffffff, 0};
      sa_top_p(list, s, rule, need, front, kept, [](float) { return true; });
      kept.above(rule.min_cut);
      sa_last(list, s, kept);
      sa_draw(row, s, rule, kept, u, token, logprob);
      return;
    }
  }
  sa_draw(row, s, rule, sa_cuts(row, s, rule, total), u, token, logprob);
}

}  // namespace

extern "C" int ls_sample_logits(const void* logits, int64_t row_stride, int64_t rows, int64_t vocab,
                                int32_t dtype, const float* u, double temperature, int32_t top_k,
                                double top_p, double min_p, const float* temperatures, const int32_t* top_ks,
                                const float* top_ps, const float* min_ps, int32_t* tokens, float* logprobs,
                                void* stream) {
  const char* who = "ls_sample_logits";
  LS_REQUIRE(rows >= 0 && vocab >= 1, LS_ERR_INVALID, "%s: bad sizes", who);
  LS_REQUIRE(vocab <= (1 << kIndexBits) && rows < (1 << 22), LS_ERR_UNSUPPORTED,
             "%s: at most 2^19 tokens, fewer than 2^22 rows", who);
  LS_REQUIRE(dtype == LS_F32 || dtype == LS_BF16 || dtype == LS_F16, LS_ERR_UNSUPPORTED,
             "%s: float32, bf16 or fp16", who);
  LS_REQUIRE(temperature >= 0.0 && temperature < INFINITY && top_p > 0.0 && min_p >= 0.0 && min_p <= 1.0, LS_ERR_INVALID,
             "%s: temperature >= 0, top_p > 0 and 0 <= min_p <= 1", who);
  if (rows == 0) return LS_OK;
  LS_REQUIRE(logits && u && tokens, LS_ERR_INVALID, "%s: null pointer", who);
  SaArgs a;
  a.x = logits;
  a.rs = row_stride;
  a.rows = rows;
  a.vocab = (int)vocab;
  a.u = u;
  a.t = temperature;
  a.top_p = top_p;
  a.min_p = min_p;
  a.top_k = top_k;
  a.ts = temperatures;
  a.top_ks = top_ks;
  a.top_ps = top_ps;
  a.min_ps = min_ps;
  a.tokens = tokens;
  a.logprobs = logprobs;
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(kThreads), 0, s, a); };
  if (dtype == LS_F32) go(ls_sample_kernel<LS_F32>);
  else if (dtype == LS_BF16) go(ls_sample_kernel<LS_BF16>);
  else go(ls_sample_kernel<LS_F16>);
  return ls_check_launch("ls_sample_kernel");
}
