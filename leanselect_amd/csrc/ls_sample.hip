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
// A workgroup a row.  The first pass takes each thread's four largest.  top_k <= 2048 gets a lower bound of
// its border from those; top_p alone gets one from the row's sum S: all logits of a weight below (1 - top_p)
// S / vocab are in the rest that it leaves.  The logits above the bound, usually few, are gathered into
// LDS, and all else is done there: up to 256 by comparing each with each.  Where more than 8192 are
// above it, top_p's border comes from a histogram of the weights over the distance from the maximum and
// the logits of its bin; where there is no bound, the same code reads the row again.
//
// A border is found by a radix search, 11 bits a round, in a histogram in LDS of how many keys, or how much
// weight, each value of the bits has; a draw from what was gathered is the same search over the
// indices, one from the row takes the sums of 256 tokens each.  Weights are summed as whole numbers of 2^-s, s
// such that a row's sum stays under 2^62 (2^-45 for 73448 tokens): sums do not depend on their order, so
// neither does the token.
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
constexpr int kMaxima = 4;  // of each thread
constexpr int kBounded = 2048;  // the largest top_k that gets a bound from them
constexpr int kSlot = 4 * kThreads;  // tokens of a round over the row
constexpr int kIndexBits = 19;
constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;
static_assert((1 << kIndexBits) / kSlot * kWaves <= kBins, "a bin for what a wave takes in each round");

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
  int shift;  // weights are whole numbers of 2^-shift
  int32_t* tokens;
  float* logprobs;
};


// 2^y, y = (x - x_max) log2(e) / t, in whole numbers of 2^-shift.  The power of y's fraction: below 2^-12 in
// float32 (1.5e-7 of it); above, where that would show, from a table of 2^(k / 16) and exp(g) to the
// seventh power (|g| < 0.022: 2^-54).
__device__ __forceinline__ uint64_t sa_exp(float x, float x_max, double scale2, int shift, const double* table) {
  const double y = fmax(((double)x - (double)x_max) * scale2, -200.0);
  const double n = rint(y), f = y - n;
  uint64_t w = (uint64_t)rintf(ldexpf(__builtin_amdgcn_exp2f((float)f), (int)n + shift));
  if (__any(y > -12.0)) {
    const double m = rint(16.0 * y), g = fma(m, -1.0 / 16.0, y) * 0.69314718055994530942;
    double p = fma(g, 1.0 / 720.0, 1.0 / 120.0);
    p = fma(g, p, 1.0 / 24.0);
    p = fma(g, p, 1.0 / 6.0);
    p = fma(g, p, 0.5);
    p = fma(g, p, 1.0);
    p = fma(g, p, 1.0);
    const int k = (int)m;
    const uint64_t exact = (uint64_t)rint(ldexp(p * table[k & 15], (k >> 4) + shift));
    w = y > -12.0 ? exact : w;
  }
  return w;
}

// A logit's key: their order is that of the logits, NaN as -inf.
template <int DT>
__device__ __forceinline__ uint32_t sa_key(typename LsElem<DT>::T v) {
  const float x = LsElem<DT>::to_f(v);
  return ls_order_key32(__float_as_uint(x != x ? -INFINITY : x == 0.f ? 0.f : x));
}
__device__ __forceinline__ float sa_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ uint64_t sa_add64(uint64_t x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor((unsigned long long)x, o, 64);
  return x;
}
// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ uint64_t sa_upto64(uint64_t x) {
  const int lane = ls_lane();
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up((unsigned long long)x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

struct SaShared {
  unsigned long long bins[kBins];
  unsigned long long part[kWaves];
  double table[16];
  unsigned long long found;
  uint32_t at;
  uint32_t n;
  uint32_t key[kList];
  uint32_t index[kList];
};

// A row in memory.  f(index, key) for this thread's logits; 0 (below every key) beyond the last.
template <int DT>
struct SaRow {
  typedef typename LsElem<DT>::T T;
  const T* x;
  int vocab;
  bool wide;  // four may be read at once

  __device__ __forceinline__ void load4(int i, uint32_t (&k)[4]) const {
    if (wide && i + 4 <= vocab) {
      if constexpr (DT == LS_F32) {
        const ls_f32x4 v = *reinterpret_cast<const ls_f32x4*>(x + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = sa_key<DT>(v[e]);
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(x + i);
        k[0] = sa_key<DT>((T)(v.x & 0xffffu));
        k[1] = sa_key<DT>((T)(v.x >> 16));
        k[2] = sa_key<DT>((T)(v.y & 0xffffu));
        k[3] = sa_key<DT>((T)(v.y >> 16));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = i + e < vocab ? sa_key<DT>(x[i + e]) : 0u;
    }
  }
  // (nine rounds' loads are under way at once: 73448 tokens are two times that)
  template <class F>
  __device__ __forceinline__ void each4(F f) const {
#pragma unroll 9
    for (int i0 = 0; i0 < vocab; i0 += kSlot) {
      const int i = i0 + 4 * (int)threadIdx.x;
      uint32_t k[4];
      load4(i, k);
      f(i, k);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    each4([&](int i, const uint32_t(&k)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(i + e, k[e]);
    });
  }
};

// What was gathered.  (Every lane runs every round: the weights are formed by whole waves.)
struct SaList {
  const uint32_t* key;
  const uint32_t* index;
  int n;
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const int i = i0 + (int)threadIdx.x;
      const bool in = i < n;
      f(in ? (int)index[i] : 0x7fffffff, in ? key[i] : 0u);
    }
  }
};

__device__ __forceinline__ uint64_t sa_max(uint64_t x, SaShared& s) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t y = __shfl_xor((unsigned long long)x, o, 64);
    x = y > x ? y : x;
  }
  __syncthreads();
  if (ls_lane() == 0) s.part[threadIdx.x >> 6] = x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) x = s.part[i] > x ? s.part[i] : x;
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

// The largest c such that the measures of the entries with order(index, key) >= c sum up to `need` at least
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
    row.each([&](int i, uint32_t key) {
      const uint32_t o = order(i, key);
      const uint64_t w = measure(i, key);
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
  uint32_t top, least;
  float x_max;
  double scale, scale2;  // 1 / temperature, log2(e) / temperature
  int shift;
  int k;          // 0: none
  double p;
  uint32_t min_cut;  // keys from here on pass min_p
  const double* table;

  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    const uint64_t w = sa_exp(sa_value(key), x_max, scale2, shift, table);
    return key == top ? 1ull << shift : key > least && x_max < INFINITY ? w : 0;
  }
};

// Kept are the keys above `cut`, and the first `ties` of those at it: with an index up to `last`.
struct SaKept {
  uint32_t cut, last;
  uint64_t ties;
  __device__ __forceinline__ bool operator()(int i, uint32_t key) const {
    return key > cut || (ties != 0 && key == cut && (uint32_t)i <= last);
  }
};

__device__ __forceinline__ uint32_t sa_by_index(int i, uint32_t) { return ~(uint32_t)i & kIndexMask; }  // lowest first
__device__ __forceinline__ uint32_t sa_by_key(int, uint32_t key) { return key; }

// `last`, from a row or list that has all keys at the border.
template <class Row>
__device__ __forceinline__ void sa_last(const Row& row, SaShared& s, SaKept& kept) {
  kept.last = 0x7fffffff;
  if (kept.ties == 0) return;
  uint64_t n = 0, above;
  row.each([&](int, uint32_t key) { n += key == kept.cut; });
  n = sa_sum(n, s);
  if (n > kept.ties)
    kept.last = ~sa_border<kIndexBits>(row, s, kept.ties, above, sa_by_index,
                                       [&](int, uint32_t key) -> uint64_t { return key == kept.cut ? 1 : 0; }) &
                kIndexMask;
}

// What top_p keeps: the keys from a border, found in a row or list of which `counts` says what is summed up; the
// sum of all larger ones is `front`.
template <class Row, class Counts>
__device__ __forceinline__ void sa_top_p(const Row& row, SaShared& s, const SaRule& rule, uint64_t need, uint64_t front,
                                         SaKept& kept, Counts counts) {
  uint64_t above;
  const uint32_t c = sa_border<32>(row, s, need - front, above, sa_by_key, [&](int, uint32_t key) -> uint64_t {
    const uint64_t w = rule.weight(key);
    return counts(key) ? w : 0;
  });
  const uint64_t w = rule.weight(c), n = (need - front - above + w - 1) / w;
  if (c > kept.cut || n < kept.ties) kept.cut = c, kept.ties = n;
}

// The cuts over the row or what was gathered of it.  `total`: the weights of the whole row, for top_p without
// top_k.
template <class Row>
__device__ __forceinline__ SaKept sa_cuts(const Row& row, SaShared& s, const SaRule& rule, uint64_t total) {
  SaKept kept{rule.least, 0x7fffffff, 0};
  if (rule.k > 0) {
    uint64_t n = 0, above;
    row.each([&](int, uint32_t key) { n += key > rule.least; });
    n = sa_sum(n, s);
    if (n > (uint64_t)rule.k) {
      kept.cut = sa_border<32>(row, s, rule.k, above, sa_by_key,
                               [&](int, uint32_t key) -> uint64_t { return key > rule.least ? 1 : 0; });
      kept.ties = rule.k - above;
    }
  }
  if (rule.p < 1.0) {
    const uint64_t at_cut = rule.weight(kept.cut);
    uint64_t here = 0;
    row.each([&](int, uint32_t key) {
      const uint64_t w = rule.weight(key);
      here += key > kept.cut ? w : 0;
    });
    here = sa_sum(here, s) + kept.ties * at_cut;
    if (rule.k > 0) total = here;
    const uint64_t need = max((uint64_t)ceil(rule.p * (double)total), (uint64_t)1);
    if (need <= here)  // (else more than what is here is kept)
      sa_top_p(row, s, rule, need, 0, kept,
               [&](uint32_t key) { return key > kept.cut || (key == kept.cut && kept.ties); });
  }
  if (rule.min_cut > kept.cut) kept.cut = rule.min_cut - 1, kept.ties = 0;
  sa_last(row, s, kept);
  return kept;
}

// The draw.
template <class Row>
__device__ __forceinline__ void sa_draw(const Row& row, SaShared& s, const SaRule& rule, const SaKept& kept, double u,
                                        int32_t* token, float* logprob) {
  uint64_t above;
  auto any = [&](int i, uint32_t key) {  // whether there is a weight at all, however small
    return kept(i, key) && (key == rule.top ||
                            (key > rule.least && ((double)sa_value(key) - rule.x_max) * rule.scale > -745.0));
  };
  auto measure = [&](int i, uint32_t key) -> uint64_t {
    const bool k = kept(i, key);
    if (!__any(k)) return 0;
    const uint64_t w = rule.weight(key);
    return k ? w : 0;
  };
  // u sum < a running sum  <=>  floor(u sum) < it, a whole number.
  auto goal_of = [&](uint64_t sum) {
    const uint64_t goal = u > 0.0 ? (uint64_t)(u * (double)sum) : 0;
    return goal < sum ? goal : sum - 1;
  };
  auto answer = [&](uint32_t i, uint32_t key, uint64_t sum) {
    *token = (int32_t)i;
    if (logprob) {
      const double y = key == rule.top ? 0.0 : ((double)sa_value(key) - rule.x_max) * rule.scale;
      *logprob = (float)(y - log(ldexp((double)sum, -rule.shift)));
    }
  };
  if (std::is_same<Row, SaList>::value || !(u > 0.0)) {
    uint64_t sum = 0;
    row.each([&](int i, uint32_t key) { sum += measure(i, key); });
    sum = sa_sum(sum, s);
    const uint32_t i =
        ~(u > 0.0 ? sa_border<kIndexBits>(row, s, goal_of(sum) + 1, above, sa_by_index, measure)
                  : sa_border<kIndexBits>(row, s, 1, above, sa_by_index,
                                          [&](int i, uint32_t key) -> uint64_t { return any(i, key) ? 1 : 0; })) &
        kIndexMask;
    row.each([&](int j, uint32_t key) {
      if ((uint32_t)j == i && key != 0) answer(i, key, sum);
    });
    return;
  }
  if constexpr (!std::is_same<Row, SaList>::value) {
    // The sums of what a wave takes in each round, 256 tokens in a row; then the one in which u falls.
    const int tid = threadIdx.x, wave = tid >> 6, rounds = (row.vocab + kSlot - 1) / kSlot;
    sa_clear(s);
    row.each4([&](int i, const uint32_t(&key)[4]) {
      uint64_t x = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) x += measure(i + e, key[e]);
      x = sa_add64(x);
      if (ls_lane() == 0) s.bins[kBins - 1 - (i / kSlot * kWaves + wave)] = x;
    });
    uint64_t sum = 0;
    __syncthreads();
    sum = sa_sum(s.bins[tid] + s.bins[tid + kThreads], s);
    const uint64_t goal = goal_of(sum);
    const uint32_t bin = kBins - 1 - sa_find(s, goal + 1, above);
    if ((int)(bin % kWaves) != wave || (int)(bin / kWaves) >= rounds) return;
    const int i = (int)(bin / kWaves) * kSlot + 4 * tid;
    uint32_t key[4];
    uint64_t w[4], x = 0;
    row.load4(i, key);
#pragma unroll
    for (int e = 0; e < 4; ++e) x += w[e] = measure(i + e, key[e]);
    uint64_t before = above + sa_upto64(x) - x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (before <= goal && goal < before + w[e]) answer(i + e, key[e], sum);
      before += w[e];
    }
  }
}

// The same for at most kFew gathered logits, one a thread: what is in front of it in either order is found by
// looking at each of the others, without a search or a histogram.
__device__ __forceinline__ void sa_draw_few(int n, SaShared& s, const SaRule& rule, uint64_t total, double u,
                                            int32_t* token, float* logprob) {
  const int tid = threadIdx.x;
  const bool in = tid < n;
  const uint32_t key = in ? s.key[tid] : 0u, i = in ? s.index[tid] : 0u;
  uint64_t w = 0;
  if (tid < kFew) {
    w = rule.weight(key);
    s.bins[tid] = w;
  }
  __syncthreads();
  uint32_t rank = 0;
  uint64_t before = 0;
  if (in) {
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const bool first = s.key[j] > key || (s.key[j] == key && s.index[j] < i);
      rank += first;
      before += first ? s.bins[j] : 0;
    }
  }
  bool kept = in && key > rule.least && (rule.k == 0 || rank < (uint32_t)rule.k);
  if (rule.p < 1.0) {
    if (rule.k > 0) total = sa_sum(kept ? w : 0, s);
    const double goal = ceil(rule.p * (double)total);
    kept = kept && before < max((uint64_t)goal, (uint64_t)1);
  }
  kept = kept && key >= rule.min_cut;
  const uint64_t sum = sa_sum(kept ? w : 0, s);
  const double y = key == rule.top ? 0.0 : ((double)sa_value(key) - rule.x_max) * rule.scale;
  // u = 0: the lowest index with any weight, however small.
  const uint64_t m = !kept ? 0 : u > 0.0 ? w : y > -745.0 ? 1 : 0;
  if (tid < kFew) s.bins[tid] = m;
  __syncthreads();
  if (m == 0) return;
  uint64_t goal = u > 0.0 ? (uint64_t)(u * (double)sum) : 0;
  goal = goal < sum ? goal : sum - 1;
  before = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) before += s.index[j] < i ? s.bins[j] : 0;
  if (before <= goal && goal < before + m) {
    *token = (int32_t)i;
    if (logprob) *logprob = (float)(y - log(ldexp((double)sum, -rule.shift)));
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
  if (tid < 16) s.table[tid] = exp2((double)tid / 16.0);
  uint32_t best[kMaxima] = {}, at = 0;
  row.each([&](int i, uint32_t key) {
    at = key > best[0] ? (uint32_t)i : at;
#pragma unroll
    for (int m = kMaxima - 1; m > 0; --m) best[m] = max(best[m], min(best[m - 1], key));
    best[0] = max(best[0], key);
  });
  const uint64_t first = sa_max((uint64_t)best[0] << 32 | (uint32_t)~at, s);
  SaRule rule;
  rule.top = (uint32_t)(first >> 32);
  rule.least = ls_order_key32(0xff800000u);  // -inf: no weight
  rule.x_max = sa_value(rule.top);
  const double t = a.ts ? (double)a.ts[r] : a.t;
  float* logprob = a.logprobs ? a.logprobs + r : nullptr;
  if (rule.top <= rule.least || !(t > 0.0)) {
    // Nothing to draw from, or the largest alone.
    if (tid == 0) {
      const bool none = rule.top <= rule.least;
      a.tokens[r] = none ? -1 : (int32_t)~(uint32_t)first;
      if (logprob) *logprob = none ? -INFINITY : 0.f;
    }
    return;
  }
  rule.scale = 1.0 / t;
  rule.scale2 = 1.4426950408889634074 / t;
  rule.shift = a.shift;
  rule.k = a.top_ks ? a.top_ks[r] : a.top_k;
  if (rule.k <= 0 || rule.k >= a.vocab) rule.k = 0;
  rule.p = a.top_ps ? (double)a.top_ps[r] : a.top_p;
  rule.table = s.table;
  rule.min_cut = 0;
  const double min_p = a.min_ps ? (double)a.min_ps[r] : a.min_p;
  if (min_p > 0.0) {
    // exp((x - max) / t) >= min_p  <=>  x >= max + t ln min_p.
    const double border = (double)rule.x_max + log(min_p) * t;
    const float f = (float)border;
    uint32_t c = ls_order_key32(__float_as_uint(f == 0.f ? 0.f : f));
    if ((double)f < border) ++c;  // the least logit that is not below it
    rule.min_cut = min(c, rule.top);
  }
  const double u = (double)a.u[r];
  // What is kept, or has to be summed up, is among the keys from `low` that are no more than `far` bins of
  // 1 / `to_bins` from the maximum.
  uint32_t low = rule.least + 1;
  float to_bins = 0.f;
  int far = 0;
  auto bin_of = [&](uint32_t key) {  // (falls as the key rises)
    const float d = (rule.x_max - sa_value(key)) * to_bins;
    return d < kBins - 1 ? (int)d : kBins - 1;
  };
  uint64_t total = 0, need = 0;
  bool bounded = false;
  if (rule.k > 0 && rule.k <= kBounded) {
    // Some of the threads' largest are the k-th largest or more; their k-th largest is a bound.
    static_assert(kBounded <= 2 * kThreads && kMaxima >= 2, "");
    const uint32_t mine = rule.k <= kThreads ? best[0] : best[1];
    const uint32_t least = ~(uint32_t)sa_max(~mine, s);
    const float range = rule.x_max - sa_value(least);
    bounded = true;
    if (least > rule.least && range > 0.f && range < INFINITY) {
      to_bins = (kBins - 2) / range;
      sa_clear(s);
#pragma unroll
      for (int m = 0; m < kMaxima; ++m)
        if (best[m] >= least) atomicAdd(&s.bins[kBins - 1 - bin_of(best[m])], 1ull);
      uint64_t before;
      far = kBins - 1 - (int)sa_find(s, rule.k, before);
    } else if (least > rule.least) {
      low = least;
    }
  } else if (rule.k == 0 && rule.p < 1.0) {
    row.each([&](int, uint32_t key) { total += rule.weight(key); });
    total = sa_sum(total, s);
    need = min(max((uint64_t)ceil(rule.p * (double)total), (uint64_t)1), total);
    // (a hundredth below it: the bound is rounded)
    const double least = (1.0 - rule.p) * ldexp((double)total, -rule.shift) / a.vocab;
    const float f = (float)((double)rule.x_max + t * (log(least) - 0.01));
    low = max(low, ls_order_key32(__float_as_uint(f == 0.f ? 0.f : f)));
    bounded = true;
  }
  // (What top_p sums up is more than what min_p leaves.)
  if (!(rule.k > 0 && rule.p < 1.0)) {
    low = max(low, rule.min_cut);
    bounded = bounded || rule.min_cut > rule.least + 1;
  }
  // Logits into LDS, a wave's in one go.
  auto gather = [&](auto take) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    row.each([&](int i, uint32_t key) {
      const uint64_t mask = __ballot(take(key));
      if (mask == 0) return;
      uint32_t n = 0;
      if (ls_lane() == 0) n = atomicAdd(&s.n, (uint32_t)__popcll(mask));
      n = __builtin_amdgcn_readfirstlane(n) + ls_lanes_below(mask);
      if (take(key) && n < kList) s.key[n] = key, s.index[n] = (uint32_t)i;
    });
    __syncthreads();
    return (int)s.n;
  };
  int32_t* token = a.tokens + r;
  if (bounded) {
    const int n = gather([&](uint32_t key) { return key >= low && (to_bins == 0.f || bin_of(key) <= far); });
    if (n <= kFew) {
      sa_draw_few(n, s, rule, total, u, token, logprob);
      return;
    }
    if (n <= kList) {
      const SaList list{s.key, s.index, n};
      sa_draw(list, s, rule, sa_cuts(list, s, rule, total), u, token, logprob);
      return;
    }
  }
  if (need > 0) {
    // Bins of 1/32 of a temperature; then, where too many logits are in the border's, of 1/65536.
    to_bins = (float)(32.0 / t);
    sa_clear(s);
    row.each([&](int, uint32_t key) {
      const uint64_t w = rule.weight(key);
      if (w != 0) atomicAdd(&s.bins[kBins - 1 - bin_of(key)], (unsigned long long)w);
    });
    uint64_t front;
    const int bin = kBins - 1 - (int)sa_find(s, need, front);
    auto in_bin = [&](uint32_t key) { return key > rule.least && bin_of(key) == bin; };
    int n = gather(in_bin), sub = -1;
    auto sub_of = [&](uint32_t key) {
      const float d = ((rule.x_max - sa_value(key)) * to_bins - (float)bin) * kBins;
      return d < kBins - 1 ? max((int)d, 0) : kBins - 1;
    };
    if (n > kList) {
      sa_clear(s);
      row.each([&](int, uint32_t key) {
        const uint64_t w = rule.weight(key);
        if (w != 0 && in_bin(key)) atomicAdd(&s.bins[kBins - 1 - sub_of(key)], (unsigned long long)w);
      });
      uint64_t before;
      sub = kBins - 1 - (int)sa_find(s, need - front, before);
      front += before;
      n = gather([&](uint32_t key) { return in_bin(key) && sub_of(key) == sub; });
    }
    if (n <= kList) {
      const SaList list{s.key, s.index, n};
      SaKept kept{rule.least, 0x7fffffff, 0};
      sa_top_p(list, s, rule, need, front, kept, [](uint32_t) { return true; });
      if (rule.min_cut > kept.cut) kept.cut = rule.min_cut - 1, kept.ties = 0;
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
  LS_REQUIRE(temperature >= 0.0 && temperature < 1e30 && top_p > 0.0 && min_p >= 0.0 && min_p <= 1.0, LS_ERR_INVALID,
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
  a.shift = 62;
  while (a.shift > 40 && (int64_t)1 << (62 - a.shift) < vocab) --a.shift;
  a.tokens = tokens;
  a.logprobs = logprobs;
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(kThreads), 0, s, a); };
  if (dtype == LS_F32) go(ls_sample_kernel<LS_F32>);
  else if (dtype == LS_BF16) go(ls_sample_kernel<LS_BF16>);
  else go(ls_sample_kernel<LS_F16>);
  return ls_check_launch("ls_sample_kernel");
}
