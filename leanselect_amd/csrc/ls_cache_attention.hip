// Attention over a dense 16-bit KV cache with capped, biased and windowed scores, and the same for
// a batch whose sequences share a prefix that is kept once.
//
//   row i of sequence b (n_b rows, len_b own keys, P prefix keys) stands at p = P + len_b - n_b + i;
//   key j of P + len_b is visible where  causal: j <= p,  left >= 0: j >= p - left,  right >= 0:
//   j <= p + right;  x = scale q.k,  cap > 0: x = cap tanh(x / cap),  slopes: x -= slope_h |p - j|;
//   out = softmax(x) v, lse = ln sum exp x;  nothing visible: zeros and lse = +inf.
//
// A tile is R query tokens with the heads of one KV group, its columns (token, head); one pass over
// its keys with a running maximum and sum.  Keys are the rows of S^T = K Q^T, so a lane (r, q) =
// (lane & 15, lane >> 4) holds the scores of column r and keys 16 t + 4 q + i, the running values
// are a lane's own, and P^T is the right operand of O^T = V^T P^T as it stands when the left one
// holds the keys in the same order, which the transposing LDS read of V gives.
//
// The prefix is one more sequence that every row attends: its tiles take rows of any sequence, so its
// keys are read once for a tile of them rather than once for each.  What the slices of the prefix
// and of a row's own keys give (O, maximum, sum) is joined by a second kernel.
//
// Extends ls_dense_attn_kvcache (options that infllmv2_attn_with_kvcache takes:
// third_party/infllmv2/paper1.patch:2511-2615).
#include <algorithm>
#include <type_traits>

#include "ls_common.h"

namespace {

constexpr int kDim = 128;
constexpr int kRowB = 2 * kDim;         // a key's bytes
constexpr int kSub = 32;                // keys of a wave's step
constexpr int kSubB = kSub * kRowB;     // their bytes
constexpr int kWaves = 4;
constexpr int kUnit = kWaves * kSub;    // keys of a workgroup's step
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

typedef short CaS4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) CaS4* CaLdsS4;

#define CA_WAIT_VM(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")
#define CA_WAIT_LDS() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")

struct CaArgs {
  const uint16_t* q;
  int64_t q_rs;
  const int32_t* cu_q;
  int64_t total_q;
  const uint16_t* kp;  // prefix
  const uint16_t* vp;
  int64_t p_rs;
  int p_len;
  const uint16_t* kc;  // own keys
  const uint16_t* vc;
  int64_t c_bs;
  int64_t c_rs;
  int capacity;
  const int32_t* lens;
  int batch;
  int G;
  int gs;
  float scale2;        // scale log2(e)
  float cap_a;         // cap log2(e)
  float cap_b;         // 2 scale log2(e) / cap
  const float* slopes;
  int64_t slopes_bs;
  int causal;
  int left;
  int right;
  int tokens;          // of a tile
  int prefix_tiles;
  int prefix_slices;
  int own_tiles;
  int own_slices;
  float* part;         // [rows][heads][slices][128], or NULL: one slice
  float* ml;           // [rows][heads][slices][2]
  uint16_t* out;
  float* lse;
};

// Over the four lanes that hold a column.
__device__ __forceinline__ float ca_max4(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float ca_sum4(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ int ca_min64(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = min(x, __shfl_xor(x, d, 64));
  return x;
}
__device__ __forceinline__ int ca_max64(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = max(x, __shfl_xor(x, d, 64));
  return x;
}

// Softmax weights are held as a 16-bit head and its remainder, a product each (2^-17 of a weight in
// bf16; in fp16, whose range is small, 2^kBias times the weight, 2^-22 of it or 2^-35 of the largest),
// so that the output's rounding is the one that shows: one bf16 a weight would add as much error again.
template <int DT> struct CaBias { static constexpr float value = 0.f; };
template <> struct CaBias<LS_F16> { static constexpr float value = 10.f; };
// The maximum follows once it is this far behind (base-2 units): weights reach 2^(kLazy + kBias).
constexpr float kLazy = 5.f;

// What a tile's columns see, and what is carried over its keys.
template <int NC>
struct CaState {
  ls_u32x4 qf[NC][4];
  ls_f32x4 o[8][NC];
  float m[NC], l[NC];
  float slope2[NC], pos[NC];  // position among the source's keys
  int lo[NC], hi[NC];         // visible keys, among the source's
};

// One step: 32 keys from key0, K rows at sk and V rows at sv (LDS, swizzled), `v_ready` waits for V.
// FULL: every column sees all of them.
template <int DT, int NC, bool CAP, bool ALIBI, bool FULL, class VReady>
__device__ __forceinline__ void ca_step(const uint8_t* sk, const uint8_t* sv, int key0, CaState<NC>& st,
                                        const CaArgs& a, VReady v_ready) {
  const int lane = ls_lane(), r = lane & 15, q = lane >> 4;
  ls_f32x4 s[2][NC];
  const int ka = r * kRowB + 16 * (q ^ r);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) s[t][nc] = ls_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const ls_u32x4 kf = *reinterpret_cast<const ls_u32x4*>(sk + 16 * kRowB * t + (ka ^ (64 * ks)));
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) s[t][nc] = LsElem<DT>::mfma(kf, st.qf[nc][ks], s[t][nc]);
    }
  }
  constexpr bool MADE = CAP || ALIBI;  // scores in base-2 units already
  ls_u32x4 hi[NC], lo[NC], seen[NC];
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    float x[8];
    float top = -INFINITY;
    const float d0 = ALIBI ? st.pos[nc] - (float)(key0 + 4 * q) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 16 * (e >> 2) + (e & 3);  // + key0 + 4 q
      x[e] = s[e >> 2][nc][e & 3];
      if (CAP) {
        // cap tanh(x / cap) = cap - 2 cap / (1 + exp(2 x / cap))
        const float w = __builtin_amdgcn_exp2f(x[e] * a.cap_b);
        x[e] = fmaf(-2.f * a.cap_a, __builtin_amdgcn_rcpf(1.f + w), a.cap_a);
      } else if (MADE) {
        x[e] *= a.scale2;
      }
      if (ALIBI) x[e] = fmaf(-st.slope2[nc], fabsf(d0 - (float)k), x[e]);
      if (!FULL) {
        const int key = key0 + 4 * q + k;
        const bool see = key >= st.lo[nc] && key < st.hi[nc];
        x[e] = see ? x[e] : -INFINITY;
        if (e & 1) seen[nc][e >> 1] |= see ? 0xffff0000u : 0u;
        else seen[nc][e >> 1] = see ? 0xffffu : 0u;
      }
      top = fmaxf(top, x[e]);
    }
    top = ca_max4(top);
    if (!MADE) top *= a.scale2;  // (scale2 is positive)
    if (__any(top > st.m[nc] + kLazy)) {
      const float m = fmaxf(st.m[nc], top);
      const float ref = m == -INFINITY ? 0.f : m;
      const float f = __builtin_amdgcn_exp2f(st.m[nc] - ref);
      st.m[nc] = m;
      st.l[nc] *= f;
#pragma unroll
      for (int db = 0; db < 8; ++db) st.o[db][nc] *= f;
    }
    const float ref = (st.m[nc] == -INFINITY ? 0.f : st.m[nc]) - CaBias<DT>::value;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p0 = __builtin_amdgcn_exp2f(MADE ? x[2 * e] - ref : fmaf(x[2 * e], a.scale2, -ref));
      const float p1 = __builtin_amdgcn_exp2f(MADE ? x[2 * e + 1] - ref : fmaf(x[2 * e + 1], a.scale2, -ref));
      sum += p0 + p1;
      const uint16_t h0 = LsElem<DT>::from_f(p0), h1 = LsElem<DT>::from_f(p1);
      hi[nc][e] = ls_pack2(h0, h1);
      lo[nc][e] = ls_pack2(LsElem<DT>::from_f(p0 - LsElem<DT>::to_f(h0)),
                           LsElem<DT>::from_f(p1 - LsElem<DT>::to_f(h1)));
    }
    st.l[nc] += sum;
  }
  v_ready();
  // Lane (r, q) of the transposing read gives its group of 16 the rows 4 q + (r >> 2), 8 bytes each,
  // and gets dim r of the rows 4 q .. 4 q + 3.
  const int row = 4 * q + (r >> 2);
  const int va = row * kRowB + 32 * (row & 7) + 8 * (r & 3);
  auto values = [&](int db) {
    const uint8_t* p = sv + (va ^ (32 * db));
    const CaS4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CaLdsS4)(p));
    const CaS4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CaLdsS4)(p + 16 * kRowB));
    const uint2 w0 = __builtin_bit_cast(uint2, v0), w1 = __builtin_bit_cast(uint2, v1);
    return ls_u32x4{w0.x, w0.y, w1.x, w1.y};
  };
  if (!FULL) {
    // Where a key is hidden from some column, its weight there is 0 and its values must not count:
    // 0 times an infinity or NaN would.  Such values are rare: they leave the product, and the
    // channels of the columns that see one become NaN.
    constexpr uint32_t kExp = DT == LS_BF16 ? 0x7f80u : 0x7c00u, kOne = DT == LS_BF16 ? 0x3f80u : 0x3c00u;
    auto odd = [&](uint32_t w) {
      return ((w & kExp) == kExp ? 0xffffu : 0u) | ((w >> 16 & kExp) == kExp ? 0xffff0000u : 0u);
    };
    uint32_t any = 0;
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      const ls_u32x4 v = values(db);
#pragma unroll
      for (int e = 0; e < 4; ++e) any |= odd(v[e]);
    }
    if (__any(any != 0)) {
      const uint32_t one = kOne | kOne << 16;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        ls_u32x4 v = values(db), is;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t mask = odd(v[e]);
          v[e] &= ~mask;
          is[e] = mask & one;
        }
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          ls_u32x4 see;
#pragma unroll
          for (int e = 0; e < 4; ++e) see[e] = seen[nc][e] & one;
          const ls_f32x4 hits = LsElem<DT>::mfma(is, see, ls_f32x4{0.f, 0.f, 0.f, 0.f});
          st.o[db][nc] = LsElem<DT>::mfma(v, hi[nc], st.o[db][nc]);
          st.o[db][nc] = LsElem<DT>::mfma(v, lo[nc], st.o[db][nc]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hits[e] > 0.f) st.o[db][nc][e] = __builtin_nanf("");
        }
      }
      return;
    }
  }
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    const ls_u32x4 v = values(db);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      st.o[db][nc] = LsElem<DT>::mfma(v, hi[nc], st.o[db][nc]);
      st.o[db][nc] = LsElem<DT>::mfma(v, lo[nc], st.o[db][nc]);
    }
  }
}

// The tile of `unit` among the batch's tiles of R tokens: its sequence, or -1 past the last; `unit`
// becomes the tile's number in it.
__device__ __forceinline__ int ca_find(const CaArgs& a, int& unit, int& n0, int& n1) {
  const int lane = ls_lane();
  for (int s0 = 0; s0 < a.batch; s0 += 64) {
    const int i = min(s0 + lane, a.batch - 1);
    const int lo = a.cu_q[i], hi = a.cu_q[i + 1];
    const int mine = s0 + lane < a.batch && hi > lo && lo >= 0 ? (hi - lo + a.tokens - 1) / a.tokens : 0;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(upto, d, 64);
      if (lane >= d) upto += y;
    }
    const uint64_t past = __ballot(unit < upto);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      unit -= __builtin_amdgcn_readlane(upto - mine, at);
      n0 = __builtin_amdgcn_readlane(lo, at);
      n1 = __builtin_amdgcn_readlane(hi, at);
      return s0 + at;
    }
    unit -= __builtin_amdgcn_readlane(upto, 63);
  }
  return -1;
}

// A workgroup's piece of work: tokens [t0, t1) of group g against keys of one source.
struct CaWork {
  int g, t0, t1, slice, slices, slot;  // slot: of the slice among the row's
  int seq, n0, n1, len;                // of the own keys; seq < 0: the prefix
  int n_keys, first;                   // the source's, and its first key's position
  const uint16_t* k;
  const uint16_t* v;
  int64_t rs;
};

// False where there is nothing to do or write.
__device__ __forceinline__ bool ca_work(const CaArgs& a, CaWork& w) {
  int item = blockIdx.x;
  const int units = a.prefix_slices * a.G, n_prefix = a.prefix_tiles * units;
  if (item < n_prefix) {
    // Workgroups go to the eight compute dies in turn: the row tiles of a slice stay on one, whose
    // cache then serves all but the first.
    const int block = item / (8 * a.prefix_tiles), in = item % (8 * a.prefix_tiles);
    const int some = min(8, units - 8 * block);
    const int u = 8 * block + in % some;
    w.g = u % a.G;
    w.slice = w.slot = u / a.G;
    w.slices = a.prefix_slices;
    w.t0 = in / some * a.tokens;
    w.t1 = (int)min(min((int64_t)w.t0 + a.tokens, a.total_q), (int64_t)a.cu_q[a.batch]);
    w.seq = -1;
    w.n_keys = a.p_len;
    w.first = 0;
    w.k = a.kp + (int64_t)w.g * kDim;
    w.v = a.vp + (int64_t)w.g * kDim;
    w.rs = a.p_rs;
    return w.t0 < w.t1;
  }
  item -= n_prefix;
  w.slice = item % a.own_slices;
  w.slices = a.own_slices;
  w.slot = a.prefix_slices + w.slice;
  item /= a.own_slices;
  w.g = item % a.G;
  int tile = item / a.G;
  w.seq = ca_find(a, tile, w.n0, w.n1);
  if (w.seq < 0) return false;
  w.t0 = w.n0 + tile * a.tokens;
  w.t1 = (int)min(min((int64_t)w.t0 + a.tokens, a.total_q), (int64_t)w.n1);
  w.len = w.n_keys = max(0, min(a.lens[w.seq], a.capacity));
  w.first = a.p_len;
  w.k = a.kc + (int64_t)w.seq * a.c_bs + (int64_t)w.g * kDim;
  w.v = a.vc + (int64_t)w.seq * a.c_bs + (int64_t)w.g * kDim;
  w.rs = a.c_rs;
  return w.t0 < w.t1;
}

// What column c (token c / gs, head c % gs) sees.
template <int NC, bool ALIBI>
__device__ __forceinline__ void ca_columns(const CaArgs& a, const CaWork& w, int c0, CaState<NC>& st) {
  const int lane = ls_lane(), r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    const int c = c0 + 16 * nc + r, tk = c / a.gs, h = c - tk * a.gs;
    const bool valid = tk < a.tokens && w.t0 + tk < w.t1;
    const int t = valid ? w.t0 + tk : w.t0;
    const uint16_t* qp = a.q + (int64_t)t * a.q_rs + ((int64_t)w.g * a.gs + h) * kDim + 8 * q;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) st.qf[nc][ks] = ls_load16(qp + 32 * ks);
    st.lo[nc] = 0;
    st.hi[nc] = w.n_keys;
    st.m[nc] = -INFINITY;
    st.l[nc] = 0.f;
    if (ALIBI || a.causal || a.left >= 0 || a.right >= 0) {
      int n0 = w.n0, n1 = w.n1, len = w.len, b = w.seq;
      if (b < 0) {
        b = ls_find_segment(a.cu_q, a.batch, t);
        n0 = a.cu_q[b];
        n1 = a.cu_q[b + 1];
        len = max(0, min(a.lens[b], a.capacity));
      }
      const int p = a.p_len + len - (n1 - n0) + (t - n0) - w.first;
      if (ALIBI) {
        st.pos[nc] = (float)p;
        st.slope2[nc] = a.slopes[b * a.slopes_bs + w.g * a.gs + h] * kLog2e;
      }
      if (a.causal) st.hi[nc] = min(st.hi[nc], p + 1);
      if (a.left >= 0) st.lo[nc] = max(0, p - a.left);
      if (a.right >= 0) st.hi[nc] = min(st.hi[nc], p + a.right + 1);
      if (st.hi[nc] <= st.lo[nc]) st.hi[nc] = st.lo[nc] = 0;
    }
    if (!valid) st.lo[nc] = -1;
#pragma unroll
    for (int db = 0; db < 8; ++db) st.o[db][nc] = ls_f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// The keys that some column sees, [klo, khi), and those that all do, [flo, fhi).  Columns beyond the
// tile's (lo = -1) see everything and count for neither.
template <int NC>
__device__ __forceinline__ void ca_range(CaState<NC>& st, int& klo, int& khi, int& flo, int& fhi) {
  klo = fhi = 0x7fffffff;
  khi = flo = 0;
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    const bool valid = st.lo[nc] >= 0, some = valid && st.hi[nc] > st.lo[nc];
    klo = some ? min(klo, st.lo[nc]) : klo;
    khi = some ? max(khi, st.hi[nc]) : khi;
    flo = valid ? max(flo, st.lo[nc]) : flo;
    fhi = valid ? min(fhi, st.hi[nc]) : fhi;
    if (!valid) st.lo[nc] = 0, st.hi[nc] = 0x7fffffff;
  }
  klo = ca_min64(klo);
  khi = ca_max64(khi);
  flo = ca_max64(flo);
  fhi = ca_min64(fhi);
}

// 32 rows from `row0` of one tensor into LDS: row i at 256 i, its 16-byte chunk C at place C ^ x(i),
// x(i) = i & 15 for K (a lane reads chunk 4 ks + q of row r) and 2 (i & 7) for V (the transposing
// read takes 32 bytes of each of 16 rows).  Rows past the last are the last one again.
template <bool IS_V>
__device__ __forceinline__ void ca_fetch(const uint16_t* base, int64_t rs, int row0, int n_keys, uint32_t lds) {
  const int lane = ls_lane(), i4 = lane >> 4;
  const uint32_t rb = 2 * (uint32_t)rs;
  const uint16_t* p = base + (int64_t)row0 * rs;
  const bool whole = row0 + kSub <= n_keys;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = 4 * j + i4;
    const uint32_t chunk = (uint32_t)(lane & 15) ^ (uint32_t)(IS_V ? 2 * (i & 7) : i & 15);
    if (whole)
      ls_dma16(p + 4 * j * rs, (uint32_t)i4 * rb + 16 * chunk, lds + 1024 * j);
    else
      ls_dma16(p, (uint32_t)min(i, n_keys - 1 - row0) * rb + 16 * chunk, lds + 1024 * j);
  }
}

// The final values or the slice's part of column c.
__device__ __forceinline__ void ca_store4(const CaArgs& a, int64_t row, int slot, int d, ls_f32x4 v) {
  *reinterpret_cast<ls_f32x4*>(a.part + (row * (a.prefix_slices + a.own_slices) + slot) * kDim + d) = v;
}

template <int DT>
__device__ __forceinline__ void ca_out4(uint16_t* p, ls_f32x4 v, float inv) {
  uint2 w;
  w.x = ls_pack2(LsElem<DT>::from_f(v[0] * inv), LsElem<DT>::from_f(v[1] * inv));
  w.y = ls_pack2(LsElem<DT>::from_f(v[2] * inv), LsElem<DT>::from_f(v[3] * inv));
  *reinterpret_cast<uint2*>(p) = w;
}

// Few columns (16 NC): the waves share a step's keys, 32 each, and hold every column.  So each key's
// bytes are read from LDS once, by one wave, in a ring of its own with no barrier; the waves' sums
// are joined through LDS at the end.
template <int DT, int NC, bool CAP, bool ALIBI>
__global__ __launch_bounds__(256) void ls_cache_attn_keys_kernel(const CaArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kWaves][2][2 * kSubB];
  __shared__ float s_ml[kWaves][2][16 * NC];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  CaWork w;
  if (!ca_work(a, w)) return;
  CaState<NC> st;
  ca_columns<NC, ALIBI>(a, w, 0, st);
  int klo, khi, flo, fhi;
  ca_range<NC>(st, klo, khi, flo, fhi);
  // The slice's steps of 128 keys.
  int it = 0, end = 0;
  if (khi > klo) {
    const int u0 = klo / kUnit, n = (khi + kUnit - 1) / kUnit - u0;
    it = u0 + (int)((int64_t)n * w.slice / w.slices);
    end = u0 + (int)((int64_t)n * (w.slice + 1) / w.slices);
    if (end * kUnit - kUnit + wave * kSub >= khi) --end;  // the last step's keys may not reach this wave
  }
  uint8_t* mine = ring[wave][0];
  const uint32_t mine_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)mine;
  auto fetch = [&](int step) {
    const int row0 = step * kUnit + wave * kSub;
    const uint32_t at = mine_at + (step & 1) * 2 * kSubB;
    ca_fetch<false>(w.k, w.rs, row0, w.n_keys, at);
    ca_fetch<true>(w.v, w.rs, row0, w.n_keys, at + kSubB);
  };
  if (it < end) fetch(it);
  for (; it < end; ++it) {
    const bool more = it + 1 < end;
    const uint8_t* sk = mine + (it & 1) * 2 * kSubB;
    if (more) {
      CA_WAIT_LDS();  // the other half has been read
      fetch(it + 1);
      CA_WAIT_VM(24);
    } else {
      CA_WAIT_VM(8);
    }
    auto v_ready = [&]() {
      if (more) CA_WAIT_VM(16);
      else CA_WAIT_VM(0);
    };
    const int key0 = it * kUnit + wave * kSub;
    if (key0 >= flo && key0 + kSub <= fhi)
      ca_step<DT, NC, CAP, ALIBI, true>(sk, sk + kSubB, key0, st, a, v_ready);
    else
      ca_step<DT, NC, CAP, ALIBI, false>(sk, sk + kSubB, key0, st, a, v_ready);
  }
  CA_WAIT_LDS();
  // The waves' sums: column c's 128 values at 512 c, 16-byte chunk C at place C ^ (c & 15).
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    const int c = 16 * nc + r;
    const float l = ca_sum4(st.l[nc]);
    if (q == 0) {
      s_ml[wave][0][c] = st.m[nc];
      s_ml[wave][1][c] = l;
    }
#pragma unroll
    for (int db = 0; db < 8; ++db)
      *reinterpret_cast<ls_f32x4*>(mine + 512 * c + 16 * ((4 * db + q) ^ r)) = st.o[db][nc];
  }
  __syncthreads();
  const int H = a.G * a.gs, slots = a.prefix_slices + a.own_slices;
  for (int e = tid; e < 16 * NC * 32; e += 256) {
    const int c = e >> 5, ch = e & 31, tk = c / a.gs, h = c - tk * a.gs;
    if (tk >= a.tokens || w.t0 + tk >= w.t1) break;  // (later columns are beyond the tile's, too)
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) M = fmaxf(M, s_ml[i][0][c]);
    ls_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float m = s_ml[i][0][c], l = s_ml[i][1][c];
      if (l == 0.f) continue;  // nothing visible
      const float f = m == M ? 1.f : __builtin_amdgcn_exp2f(m - M);
      L += f * l;
      v += f * *reinterpret_cast<const ls_f32x4*>(ring[i][0] + 512 * c + 16 * (ch ^ (c & 15)));
    }
    const int64_t row = (int64_t)(w.t0 + tk) * H + w.g * a.gs + h;
    M -= CaBias<DT>::value;
    if (a.part) {
      if (L != 0.f) ca_store4(a, row, w.slot, 4 * ch, v);
      if (ch == 0) *reinterpret_cast<float2*>(a.ml + 2 * (row * slots + w.slot)) = make_float2(M, L);
    } else {
      ca_out4<DT>(a.out + row * kDim + 4 * ch, v, L == 0.f ? 0.f : 1.f / L);
      if (ch == 0 && a.lse)
        a.lse[(int64_t)(w.g * a.gs + h) * a.total_q + w.t0 + tk] = L == 0.f ? INFINITY : (M + log2f(L)) * kLn2;
    }
  }
}

// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over a row's slices; a wave per (row, head), two
// channels a lane, each lane the weights of up to four slices.
template <int DT>
__global__ __launch_bounds__(256) void ls_cache_attn_join_kernel(const CaArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int H = a.G * a.gs, slots = a.prefix_slices + a.own_slices;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.total_q * H || row / H >= a.cu_q[a.batch]) return;
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + row * slots;
  float m[4], l[4], M = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = 64 * i + lane;
    const float2 x = s < slots ? ml[s] : make_float2(-INFINITY, 0.f);
    m[i] = x.x;
    l[i] = x.y;
    M = fmaxf(M, m[i]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, ls_shfl_xor(M, o));
  float L = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // A slice's weight; one without a visible key has no sums.
    m[i] = l[i] == 0.f ? 0.f : m[i] == M ? 1.f : __builtin_amdgcn_exp2f(m[i] - M);
    L += l[i] == 0.f ? 0.f : m[i] * l[i];
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) L += ls_shfl_xor(L, o);
  const float2* p = reinterpret_cast<const float2*>(a.part) + row * slots * (kDim / 2) + lane;
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = min(64, slots - 64 * i);
    for (int s = 0; s < n; ++s) {
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m[i]), s));
      if (f == 0.f) continue;
      const float2 x = p[(64 * i + s) * (kDim / 2)];
      acc.x = fmaf(f, x.x, acc.x);
      acc.y = fmaf(f, x.y, acc.y);
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  reinterpret_cast<uint32_t*>(a.out)[row * (kDim / 2) + lane] =
      ls_pack2(LsElem<DT>::from_f(acc.x * inv), LsElem<DT>::from_f(acc.y * inv));
  if (lane == 0 && a.lse)
    a.lse[(row % H) * a.total_q + row / H] = L == 0.f ? INFINITY : (M + log2f(L)) * kLn2;
}

// How a call is cut.
struct CaPlan {
  int nc, tokens;
  int prefix_tiles, prefix_slices, own_tiles, own_slices;
  int64_t items;
  size_t part, total;
};

constexpr int kMaxSlots = 256;

CaPlan ca_plan(int64_t total_q, int batch, int H, int G, int64_t p_len, int64_t max_len, int n_splits) {
  CaPlan p;
  const int gs = H / G;
  const int64_t rows = batch > 0 ? (total_q + batch - 1) / batch : 0;  // of a sequence
  const int64_t cols = (p_len > 0 ? total_q : rows) * gs;
  p.nc = cols <= 16 ? 1 : cols <= 32 ? 2 : 4;
  p.tokens = std::max(1, 16 * p.nc / gs);
  p.own_tiles = (int)std::min<int64_t>(total_q, total_q / p.tokens + batch);
  p.prefix_tiles = p_len > 0 ? (int)((total_q + p.tokens - 1) / p.tokens) : 0;
  const int64_t own_steps = std::max<int64_t>(1, (max_len + kUnit - 1) / kUnit);
  const int64_t prefix_steps = (p_len + kUnit - 1) / kUnit;
  auto cut = [&](int64_t tiles, int64_t steps) {
    return (int)std::max<int64_t>(1, std::min<int64_t>({steps, 256 / std::max<int64_t>(1, tiles * G), kMaxSlots / 2}));
  };
  if (n_splits > 0) {
    p.prefix_slices = p_len > 0 ? std::min(n_splits, kMaxSlots / 2) : 0;
    p.own_slices = std::min(n_splits, kMaxSlots / 2);
  } else {
    p.prefix_slices = p_len > 0 ? cut(p.prefix_tiles, prefix_steps) : 0;
    p.own_slices = cut(p.own_tiles, own_steps);
  }
  const int slots = p.prefix_slices + p.own_slices;
  p.items = ((int64_t)p.prefix_tiles * p.prefix_slices + (int64_t)p.own_tiles * p.own_slices) * G;
  p.part = slots > 1 ? ls_align256(4 * (size_t)total_q * H * slots * kDim) : 0;
  p.total = slots > 1 ? p.part + 8 * (size_t)total_q * H * slots : 0;
  return p;
}

}  // namespace

extern "C" size_t ls_cache_attn_workspace_size(int64_t total_q, int32_t batch, int32_t num_heads,
                                               int32_t num_kv_heads, int64_t prefix_len, int64_t max_len,
                                               int32_t n_splits) {
  if (total_q <= 0 || batch <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads || prefix_len < 0) return 0;
  return ca_plan(total_q, batch, num_heads, num_kv_heads, prefix_len, max_len, n_splits).total;
}

extern "C" int ls_cache_attn(const void* q, int64_t q_row_stride, const int32_t* cu_seqlens_q,
                             int64_t total_q, const void* k_prefix, const void* v_prefix,
                             int64_t prefix_row_stride, int64_t prefix_len, const void* k_cache,
                             const void* v_cache, int64_t cache_batch_stride, int64_t cache_row_stride,
                             int64_t capacity, const int32_t* cache_seqlens, int32_t batch,
                             int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                             int64_t max_len, float softmax_scale, int32_t causal, float softcap,
                             const float* alibi_slopes, int64_t alibi_batch_stride, int32_t window_left,
                             int32_t window_right, int32_t n_splits, void* out, float* softmax_lse,
                             void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "ls_cache_attn";
  LS_REQUIRE(batch > 0 && total_q >= 0 && num_kv_heads > 0 && num_heads > 0 &&
                 num_heads % num_kv_heads == 0 && prefix_len >= 0 && capacity >= 0 && max_len >= 0,
             LS_ERR_INVALID, "%s: bad sizes", who);
  const int gs = num_heads / num_kv_heads;
  LS_REQUIRE(head_dim == kDim && gs <= 16, LS_ERR_UNSUPPORTED,
             "%s: head_dim 128 and at most 16 query heads per KV head", who);
  LS_REQUIRE(dtype == LS_BF16 || dtype == LS_F16, LS_ERR_UNSUPPORTED, "%s: bf16 or fp16", who);
  LS_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY && softcap >= 0.f && softcap < INFINITY,
             LS_ERR_INVALID, "%s: softmax_scale must be positive and softcap not negative", who);
  LS_REQUIRE(n_splits >= 0 && n_splits <= kMaxSlots / 2, LS_ERR_INVALID, "%s: 0 <= n_splits <= %d", who,
             kMaxSlots / 2);
  LS_REQUIRE(prefix_len + capacity < (1 << 30) && total_q < (1 << 30), LS_ERR_UNSUPPORTED,
             "%s: fewer than 2^30 keys a sequence and rows", who);
  LS_REQUIRE(q_row_stride % 8 == 0 && cache_row_stride % 8 == 0 && cache_batch_stride % 8 == 0 &&
                 prefix_row_stride % 8 == 0,
             LS_ERR_UNSUPPORTED, "%s: strides must be multiples of 8", who);
  LS_REQUIRE(cache_row_stride >= 0 && prefix_row_stride >= 0 && cache_row_stride < (1 << 24) &&
                 prefix_row_stride < (1 << 24),
             LS_ERR_UNSUPPORTED, "%s: key rows must be less than 2^24 elements apart", who);
  if (total_q == 0) return LS_OK;
  LS_REQUIRE(q && cu_seqlens_q && cache_seqlens && out && (capacity == 0 || (k_cache && v_cache)) &&
                 (prefix_len == 0 || (k_prefix && v_prefix)),
             LS_ERR_INVALID, "%s: null pointer", who);
  LS_REQUIRE(ls_aligned16(q) && ls_aligned16(k_cache) && ls_aligned16(v_cache) && ls_aligned16(k_prefix) &&
                 ls_aligned16(v_prefix) && ls_aligned16(out) && ls_aligned16(workspace),
             LS_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned", who);
  const CaPlan p = ca_plan(total_q, batch, num_heads, num_kv_heads, prefix_len, max_len, n_splits);
  LS_REQUIRE(workspace_bytes >= p.total && (p.total == 0 || workspace), LS_ERR_WORKSPACE,
             "%s: workspace %zu < %zu", who, workspace_bytes, p.total);
  LS_REQUIRE(p.items < (1 << 23) && total_q * num_heads < (1 << 25), LS_ERR_UNSUPPORTED,
             "%s: more workgroups than a launch holds", who);
  CaArgs a = {};
  a.q = (const uint16_t*)q;
  a.q_rs = q_row_stride;
  a.cu_q = cu_seqlens_q;
  a.total_q = total_q;
  a.kp = (const uint16_t*)k_prefix;
  a.vp = (const uint16_t*)v_prefix;
  a.p_rs = prefix_row_stride;
  a.p_len = (int)prefix_len;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.c_bs = cache_batch_stride;
  a.c_rs = cache_row_stride;
  a.capacity = (int)capacity;
  a.lens = cache_seqlens;
  a.batch = batch;
  a.G = num_kv_heads;
  a.gs = gs;
  a.scale2 = softmax_scale * kLog2e;
  a.cap_a = softcap * kLog2e;
  a.cap_b = softcap > 0.f ? 2.f * softmax_scale * kLog2e / softcap : 0.f;
  a.slopes = alibi_slopes;
  a.slopes_bs = alibi_batch_stride;
  a.causal = causal != 0;
  a.left = window_left < 0 ? -1 : std::min(window_left, 1 << 30);
  a.right = window_right < 0 ? -1 : std::min(window_right, (1 << 30) - 1);
  a.tokens = p.tokens;
  a.prefix_tiles = p.prefix_tiles;
  a.prefix_slices = p.prefix_slices;
  a.own_tiles = p.own_tiles;
  a.own_slices = p.own_slices;
  a.part = p.total ? (float*)workspace : nullptr;
  a.ml = p.total ? (float*)((uint8_t*)workspace + p.part) : nullptr;
  a.out = (uint16_t*)out;
  a.lse = softmax_lse;
  hipStream_t s = (hipStream_t)stream;
  auto by_type = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto by_score = [&](auto nc) {
      constexpr int NC = decltype(nc)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)p.items), dim3(256), 0, s, a);
      };
      if (softcap > 0.f)
        alibi_slopes ? go(ls_cache_attn_keys_kernel<DT, NC, true, true>)
                     : go(ls_cache_attn_keys_kernel<DT, NC, true, false>);
      else
        alibi_slopes ? go(ls_cache_attn_keys_kernel<DT, NC, false, true>)
                     : go(ls_cache_attn_keys_kernel<DT, NC, false, false>);
    };
    if (p.nc == 1) by_score(std::integral_constant<int, 1>());
    else if (p.nc == 2) by_score(std::integral_constant<int, 2>());
    else by_score(std::integral_constant<int, 4>());
    int rc = ls_check_launch("ls_cache_attn_keys_kernel");
    if (rc || !p.total) return rc;
    hipLaunchKernelGGL(ls_cache_attn_join_kernel<DT>, dim3((unsigned)((total_q * num_heads + 3) / 4)),
                       dim3(256), 0, s, a);
    return ls_check_launch("ls_cache_attn_join_kernel");
  };
  return dtype == LS_BF16 ? by_type(std::integral_constant<int, LS_BF16>())
                          : by_type(std::integral_constant<int, LS_F16>());
}
