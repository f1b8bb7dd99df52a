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
// What bounds it (4.9 TB/s is what a large copy reaches here, 1400 TFLOP/s a large bf16 product).  Few rows:
// the keys' bytes; sixteen sequences of 2K to 64K take 66 us (4.6 TB/s), eight of up to 16K with 8 KV heads
// 53 us (4.0), and one row with a window of 4096 16 us, which are two launches and one step's latency.  Many
// rows: the vector units and the matrix units of a wave and its neighbour, which overlap only in part: of a
// 1024-row chunk behind 32K tokens with capped scores (855 us, 654 TFLOP/s of plain products, 1000 with those
// of the remainders) the matrix units are busy 35% and the vector ones 52% of the time, of two prompts
// in fp16 with a bias (204 us) 44% and 69%.  Two groups of waves held half a step apart by barriers, so that
// one's products meet the other's exponentials, took 898 us; the next step's scores in between this one's
// weights and the last one's products, 1038 where the plain order took 1027.
//
// Extends ls_dense_attn_kvcache (options that infllmv2_attn_with_kvcache takes:
// third_party/infllmv2/paper1.patch:2511-2615).
#include <algorithm>
#include <type_traits>

#include "ls_common.h"

namespace {

constexpr int kDim = 128;
constexpr int kRowB = 2 * kDim;  // a key's bytes
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

// Keys form: the waves share a step's keys, 32 each, and hold all of the tile's 16 columns.
constexpr int kKeysSub = 32;
constexpr int kKeysStep = kWaves * kKeysSub;
constexpr int kSubB = kKeysSub * kRowB;
constexpr int kKeysCols = 16;
constexpr int kManyCols = 64;  // up to which tiles of 16 may take more columns
// Rows form: the waves share the tile's 256 columns, 32 each, and walk the same keys, 64 a step.
constexpr int kRowsCols = 32 * kWaves;
constexpr int kRowsStep = 64;
constexpr int kRowsB = kRowsStep * kRowB;
constexpr int kRing = 4;

constexpr int kLdsBytes = 2 * kWaves * kSubB;  // 128 KB: the keys form's, and a ring of 4 in the rows form
static_assert(kLdsBytes == kRing * 2 * kRowsB, "one allocation serves both forms");

// LDS by 32-bit offsets: a pointer of the general kind takes two registers.
typedef short CaS4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) CaS4 CaLdsS4;
typedef __attribute__((address_space(3))) const ls_u32x4 CaLdsU4;
typedef __attribute__((address_space(3))) ls_f32x4 CaLdsF4;

#define CA_WAIT_VM(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")
#define CA_WAIT_LDS() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")

// How one source's keys are cut: tiles of `tokens` query tokens, `cols` columns in the workspace.
struct CaCut {
  int tokens;
  int cols;
  int tiles;   // upper bound
  int slices;  // of a tile; 0: by its length (keys form)
  int items;   // workgroups
};

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
  // Base-2 scores are alpha z + beta: z = q.k, alpha = scale log2(e), beta = 0, or with a cap
  // z = -1 / (1 + 2^(cap_b q.k)), alpha = 2 cap log2(e), beta = alpha / 2, cap_b = 2 scale log2(e) / cap
  // (cap tanh(x / cap) = cap - 2 cap / (1 + exp(2 x / cap))); with slopes the score itself, less its bias.
  float alpha;
  float beta;
  float cap_b;  // 0: no cap.  z is off by 2^-23 or so, at most 2^-22, and the score by 2 cap times that
  const float* slopes;
  int64_t slopes_bs;
  int causal;
  int left;
  int right;
  CaCut pre;
  CaCut own;
  // Workspace (NULL: every row is one workgroup's): per item [cols][128] sums and [cols] (maximum, sum),
  // the prefix's items first; per (row, head) the first of its
  // sequence's items, a tile's slices times 256 plus the row's column, its tile and the sequence's tiles.
  float* part;
  float2* ml;
  int4* rows;
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
__device__ __forceinline__ int ca_min64(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = min(x, __shfl_xor(x, d, 64));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int ca_max64(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = max(x, __shfl_xor(x, d, 64));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int ca_upto64(int x) {
  const int lane = ls_lane();
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

// Softmax weights are held as a 16-bit head and its remainder, a product each (2^-17 of a weight in
// bf16; in fp16, whose range is small, 2^value times the weight, 2^-21 of it or 2^-35 of the largest),
// so that the output's rounding is the one that shows: one bf16 a weight would add as much error again.
template <int DT> struct CaBias { static constexpr float value = 0.f; };
template <> struct CaBias<LS_F16> { static constexpr float value = 10.f; };
// The maximum follows once it is this far behind (base-2 units): weights reach 2^(kLazy + value).
constexpr float kLazy = 5.f;

// Two floats as bf16, to nearest even.
__device__ __forceinline__ uint32_t ca_bf16x2(float a, float b) {
  typedef float F2 __attribute__((ext_vector_type(2)));
  typedef __bf16 B2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{a, b}), B2));
}

// Two weights' heads (x), cut off, and remainders (y).
template <int DT>
__device__ __forceinline__ uint2 ca_split(float p0, float p1) {
  if constexpr (DT == LS_BF16) {
    const uint32_t b0 = __float_as_uint(p0) & 0xffff0000u, b1 = __float_as_uint(p1) & 0xffff0000u;
    return make_uint2(__builtin_amdgcn_perm(b1, b0, 0x07060302u),
                      ca_bf16x2(p0 - __uint_as_float(b0), p1 - __uint_as_float(b1)));
  } else {
    // (each weight less its half of the pair in one instruction; the pair stands behind the weights)
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    float r0, r1;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(h), "v"(p0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(h), "v"(p1));
    return make_uint2(h, __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r0, r1)));
  }
}

// All ones in each half that holds an infinity or NaN: an exponent of ones plus its lowest bit carries
// into the sign.
template <int DT>
__device__ __forceinline__ uint32_t ca_odd(uint32_t w) {
  typedef short S2 __attribute__((ext_vector_type(2)));
  constexpr uint32_t kExp = DT == LS_BF16 ? 0x7f807f80u : 0x7c007c00u, kLow = DT == LS_BF16 ? 0x00800080u : 0x04000400u;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(S2, (w & kExp) + kLow) >> 15);
}

// What a wave's columns see, and what is carried over its keys.
template <int NC>
struct CaState {
  ls_u32x4 qf[NC][4];
  ls_f32x4 o[8][NC];
  ls_f32x4 l[NC];             // the sum of a column's weights, by a product with ones: four times the same
  float m[NC];
  float slope2[NC];
  int pos[NC];                // position among the source's keys, less the lane's first key of a step
  int lo[NC], hi[NC];         // visible keys, among the source's
};

// One step: 16 KB keys from key0, K rows at sk and V rows at sv (LDS, swizzled).  `k_read` is called
// once K has been read, `v_ready` before V is, `v_read` after.  FULL: every column sees all of them.
template <int DT, int NC, int KB, bool FULL, class KRead, class VReady, class VRead>
__device__ __forceinline__ void ca_step(uint32_t sk, uint32_t sv, int key0, CaState<NC>& st,
                                        const CaArgs& a, KRead k_read, VReady v_ready, VRead v_read) {
  const int lane = ls_lane(), r = lane & 15, q = lane >> 4;
  // K is read one block ahead of its products, V two: further ahead gained nothing (a 1024-row chunk
  // behind 32K tokens 850 us either way).
  ls_f32x4 s[KB][NC];
  const uint32_t ka = r * kRowB + 16 * (q ^ r);
  ls_u32x4 kf[2][4];
  auto keys = [&](int t, ls_u32x4(&f)[4]) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
      f[ks] = *(CaLdsU4*)(sk + 16 * kRowB * t + (ka ^ (64 * ks)));
  };
  // A wave that feeds the matrix unit goes first; the other one of its SIMD has vector work to do
  // (a 1024-row chunk behind 32K tokens 1076 -> 1025 us).
  __builtin_amdgcn_s_setprio(1);
  keys(0, kf[0]);
#pragma unroll
  for (int t = 0; t < KB; ++t) {
    if (t + 1 < KB) keys(t + 1, kf[(t + 1) & 1]);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) s[t][nc] = ls_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) s[t][nc] = LsElem<DT>::mfma(kf[t & 1][ks], st.qf[nc][ks], s[t][nc]);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
  k_read();
  float alpha = a.alpha, beta = a.beta;
  if (a.cap_b > 0.f) {
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int t = 0; t < KB; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[t][nc][i] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s[t][nc][i] * a.cap_b));
  }
  if (a.slopes) {
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      // In whole numbers: both may be past 2^24.  (key0 said to be scalar: else the loops' counter goes to a vector
      // register for it, and a 1024-row chunk behind 32K tokens, which has no slopes, takes 870 us, not 855.)
      const float d0 = (float)(st.pos[nc] - __builtin_amdgcn_readfirstlane(key0));
#pragma unroll
      for (int t = 0; t < KB; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[t][nc][i] = fmaf(-st.slope2[nc], fabsf(d0 - (float)(16 * t + i)), fmaf(s[t][nc][i], alpha, beta));
    }
    alpha = 1.f;
    beta = 0.f;
  }
  if (!FULL) {
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      const int l0 = st.lo[nc] - (key0 + 4 * q), h0 = st.hi[nc] - (key0 + 4 * q);
#pragma unroll
      for (int t = 0; t < KB; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * t + i < l0 || 16 * t + i >= h0) s[t][nc][i] = -INFINITY;
    }
  }
  ls_u32x4 hi[KB / 2][NC], lo[KB / 2][NC];
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    float top = s[0][nc][0];
#pragma unroll
    for (int t = 0; t < KB; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = ls_fmax_nan(top, s[t][nc][i]);
    top = fmaf(ca_max4(top), alpha, beta);
    if (__any(top > st.m[nc] + kLazy)) {
      const float m = fmaxf(st.m[nc], top);
      const float f = __builtin_amdgcn_exp2f(st.m[nc] - (m == -INFINITY ? 0.f : m));
      st.m[nc] = m;
      st.l[nc] *= f;
#pragma unroll
      for (int db = 0; db < 8; ++db) st.o[db][nc] *= f;
    }
    const float ref = beta + CaBias<DT>::value - (st.m[nc] == -INFINITY ? 0.f : st.m[nc]);
#pragma unroll
    for (int t = 0; t < KB; ++t) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][nc][i], alpha, ref));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint2 w = ca_split<DT>(p[2 * e], p[2 * e + 1]);
        hi[t / 2][nc][2 * (t & 1) + e] = w.x;
        lo[t / 2][nc][2 * (t & 1) + e] = w.y;
      }
    }
  }
  v_ready();
  __builtin_amdgcn_s_setprio(1);
  // Lane (r, q) of the transposing read gives its group of 16 the rows 4 q + (r >> 2), 8 bytes each,
  // and gets dim r of the rows 4 q .. 4 q + 3.
  const int row = 4 * q + (r >> 2);
  const uint32_t va = row * kRowB + 32 * (row & 7) + 8 * (r & 3);
  auto values = [&](int half, int db) {
    const uint32_t p = sv + 32 * kRowB * half + (va ^ (32 * db));
    const CaS4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CaLdsS4*)p);
    const CaS4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CaLdsS4*)(p + 16 * kRowB));
    const uint2 w0 = __builtin_bit_cast(uint2, v0), w1 = __builtin_bit_cast(uint2, v1);
    return ls_u32x4{w0.x, w0.y, w1.x, w1.y};
  };
  constexpr uint32_t kOne = DT == LS_BF16 ? 0x3f80u : 0x3c00u;
  auto total = [&]() {
    constexpr uint32_t kOnes = kOne | kOne << 16;
    const ls_u32x4 ones = {kOnes, kOnes, kOnes, kOnes};
#pragma unroll
    for (int half = 0; half < KB / 2; ++half)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        st.l[nc] = LsElem<DT>::mfma(ones, hi[half][nc], st.l[nc]);
        st.l[nc] = LsElem<DT>::mfma(ones, lo[half][nc], st.l[nc]);
      }
  };
  if (FULL) {
    constexpr int kBlocks = 4 * KB;  // (half, db)
    constexpr int kPairs = 3;
    ls_u32x4 vf[kPairs][2];
    auto pair = [&](int i, ls_u32x4(&f)[2]) {
      f[0] = values(i >> 3, i & 7);
      f[1] = values(i >> 3, (i & 7) + 1);
    };
#pragma unroll
    for (int i = 0; i + 1 < kPairs; ++i) pair(2 * i, vf[i]);
    total();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kBlocks; i += 2) {
      if (i + 2 * (kPairs - 1) < kBlocks) pair(i + 2 * (kPairs - 1), vf[(i / 2 + kPairs - 1) % kPairs]);
      const int half = i >> 3, db = i & 7;
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int nc = 0; nc < NC; ++nc)
            st.o[db + e][nc] = LsElem<DT>::mfma(vf[i / 2 % kPairs][e], part ? lo[half][nc] : hi[half][nc], st.o[db + e][nc]);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    // Where a key is hidden from some column, its weight there is 0 and its values must not count:
    // 0 times an infinity or NaN would.  Such values leave the product.
    uint32_t some = 0;
    total();
#pragma unroll
    for (int half = 0; half < KB / 2; ++half)
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        ls_u32x4 v = values(half, db);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t odd = ca_odd<DT>(v[e]);
          v[e] &= ~odd;
          some |= odd;
        }
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) st.o[db][nc] = LsElem<DT>::mfma(v, hi[half][nc], st.o[db][nc]);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) st.o[db][nc] = LsElem<DT>::mfma(v, lo[half][nc], st.o[db][nc]);
        __builtin_amdgcn_sched_barrier(0);
      }
    if (__any(some != 0)) {
      // The channels of the columns that see one become NaN.
#pragma unroll
      for (int half = 0; half < KB / 2; ++half) {
        ls_u32x4 see[NC];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          const int l0 = st.lo[nc] - (key0 + 4 * q), h0 = st.hi[nc] - (key0 + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = 32 * half + 16 * (e >> 1) + 2 * (e & 1);
            see[nc][e] = (k >= l0 && k < h0 ? kOne : 0u) | (k + 1 >= l0 && k + 1 < h0 ? kOne << 16 : 0u);
          }
        }
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          ls_u32x4 is = values(half, db);
#pragma unroll
          for (int e = 0; e < 4; ++e) is[e] = ca_odd<DT>(is[e]) & (kOne | kOne << 16);
#pragma unroll
          for (int nc = 0; nc < NC; ++nc) {
            const ls_f32x4 hits = LsElem<DT>::mfma(is, see[nc], ls_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hits[e] > 0.f) st.o[db][nc][e] = __builtin_nanf("");
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  __builtin_amdgcn_s_setprio(0);
  v_read();
}

// A workgroup's piece of work: tokens [t0, t1) of group g against a slice of one source's keys.
struct CaWork {
  int item;  // its place in the workspace
  int base;  // the first item of the sequence, its tiles and this one's place among them
  int tiles, tile;
  int g, t0, t1, slice, slices;
  int seq, n0, n1, len;  // of the own keys; seq < 0: the prefix
  int n_keys, first;     // the source's, and its first key's position
  const uint16_t* k;
  const uint16_t* v;
  int64_t rs;
};

// Items of `units` slices, each with the same `tiles` of rows, go to the eight compute dies in turn: the tiles of
// a slice stay on one, whose cache then serves all but the first.
__device__ __forceinline__ void ca_split_item(int item, int units, int tiles, int& unit, int& tile) {
  const int block = item / (8 * tiles), in = item % (8 * tiles), some = min(8, units - 8 * block);
  unit = 8 * block + in % some;
  tile = in / some;
}
__device__ __forceinline__ int ca_join_item(int unit, int tile, int units, int tiles) {
  const int block = unit / 8;
  return block * 8 * tiles + tile * min(8, units - 8 * block) + unit % 8;
}

// The item-th workgroup of the prefix.
__device__ __forceinline__ bool ca_prefix_work(const CaArgs& a, int item, CaWork& w) {
  int u, tile;
  ca_split_item(item, a.pre.slices * a.G, a.pre.tiles, u, tile);
  w.item = item;
  w.base = 0;
  w.g = u % a.G;
  w.slice = u / a.G;
  w.slices = a.pre.slices;
  w.t0 = tile * a.pre.tokens;
  w.t1 = (int)min(min((int64_t)w.t0 + a.pre.tokens, a.total_q), (int64_t)a.cu_q[a.batch]);
  w.seq = -1;
  w.n_keys = a.p_len;
  w.first = 0;
  w.k = a.kp + (int64_t)w.g * kDim;
  w.v = a.vp + (int64_t)w.g * kDim;
  w.rs = a.p_rs;
  return w.t0 < w.t1;
}

// The item-th workgroup of the own keys.  Keys form: a sequence's tiles are cut into slices of about
// the same length, as many as the workgroups allow: rows of a batch differ much in length.
__device__ __forceinline__ bool ca_own_work(const CaArgs& a, int item, CaWork& w) {
  const int lane = ls_lane();
  w.item = a.pre.items + item;
  int64_t length = 0;  // of a slice, in steps; 0: fixed numbers of slices
  auto tiles_of = [&](int s0, int& lo, int& hi, int& len) {
    const int i = min(s0 + lane, a.batch - 1);
    lo = a.cu_q[i];
    hi = a.cu_q[i + 1];
    len = max(0, min(a.lens[i], a.capacity));
    return s0 + lane < a.batch && hi > lo && lo >= 0 ? (hi - lo + a.own.tokens - 1) / a.own.tokens : 0;
  };
  auto steps_of = [&](int lo, int hi, int len) {
    const int from = a.left >= 0 ? min(len, max(0, len - (hi - lo) - a.left)) : 0;
    return (len - from + kKeysStep - 1) / kKeysStep;
  };
  if (a.own.slices == 0 && !a.part) {
    length = (int64_t)1 << 40;
  } else if (a.own.slices == 0) {
    int64_t work = 0;
    int tiles = 0;
    for (int s0 = 0; s0 < a.batch; s0 += 64) {
      int lo, hi, len;
      const int n = tiles_of(s0, lo, hi, len);
      tiles += __builtin_amdgcn_readlane(ca_upto64(n), 63);
      // (steps of 64 sequences and tiles of 2^20 tokens: fewer than 2^31)
      int64_t mine = (int64_t)n * steps_of(lo, hi, len);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) mine += __shfl_xor(mine, d, 64);
      work += mine;
    }
    const int spare = a.own.items - tiles * a.G;
    length = spare <= 0 ? (int64_t)1 << 40 : max((int64_t)1, (work * a.G + spare - 1) / spare);
  }
  for (int s0 = 0; s0 < a.batch; s0 += 64) {
    int lo, hi, len;
    const int n = tiles_of(s0, lo, hi, len);
    const int slices = length ? (int)max((int64_t)1, (steps_of(lo, hi, len) + length - 1) / length) : a.own.slices;
    const int mine = n * a.G * slices, upto = ca_upto64(mine);
    const uint64_t past = __ballot(item < upto);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      item -= __builtin_amdgcn_readlane(upto - mine, at);
      w.seq = s0 + at;
      w.n0 = __builtin_amdgcn_readlane(lo, at);
      w.n1 = __builtin_amdgcn_readlane(hi, at);
      w.len = w.n_keys = __builtin_amdgcn_readlane(len, at);
      w.slices = __builtin_amdgcn_readlane(slices, at);
      w.base = w.item - a.pre.items - item;
      w.tiles = __builtin_amdgcn_readlane(n, at);
      int u;
      ca_split_item(item, w.slices * a.G, w.tiles, u, w.tile);
      w.g = u % a.G;
      w.slice = u / a.G;
      // The last tiles, which see the most keys where causal, first.
      w.t0 = w.n0 + (w.tiles - 1 - w.tile) * a.own.tokens;
      w.t1 = (int)min(min((int64_t)w.t0 + a.own.tokens, a.total_q), (int64_t)w.n1);
      w.first = a.p_len;
      w.k = a.kc + (int64_t)w.seq * a.c_bs + (int64_t)w.g * kDim;
      w.v = a.vc + (int64_t)w.seq * a.c_bs + (int64_t)w.g * kDim;
      w.rs = a.c_rs;
      return w.t0 < w.t1;
    }
    item -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// The tile's columns c0 + 16 nc + r (token c / gs, head c % gs) and what they see.
template <int NC>
__device__ __forceinline__ void ca_columns(const CaArgs& a, const CaWork& w, int tokens, int c0, CaState<NC>& st) {
  const int lane = ls_lane(), r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    const int c = c0 + 16 * nc + r, tk = c / a.gs, h = c - tk * a.gs;
    const bool valid = tk < tokens && w.t0 + tk < w.t1;
    const int t = valid ? w.t0 + tk : w.t0;
    const uint16_t* qp = a.q + (int64_t)t * a.q_rs + ((int64_t)w.g * a.gs + h) * kDim + 8 * q;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) st.qf[nc][ks] = ls_load16(qp + 32 * ks);
    st.lo[nc] = 0;
    st.hi[nc] = w.n_keys;
    st.m[nc] = -INFINITY;
    st.l[nc] = ls_f32x4{0.f, 0.f, 0.f, 0.f};
    st.slope2[nc] = 0.f;
    st.pos[nc] = 0;
    if (a.slopes || a.causal || a.left >= 0 || a.right >= 0) {
      int n0 = w.n0, n1 = w.n1, len = w.len, b = w.seq;
      if (b < 0) {
        b = ls_find_segment(a.cu_q, a.batch, t);
        n0 = a.cu_q[b];
        n1 = a.cu_q[b + 1];
        len = max(0, min(a.lens[b], a.capacity));
      }
      const int p = a.p_len + len - (n1 - n0) + (t - n0) - w.first;
      st.pos[nc] = p - 4 * q;
      if (a.slopes) st.slope2[nc] = a.slopes[b * a.slopes_bs + w.g * a.gs + h] * kLog2e;
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

// The keys that some column of the wave sees, [klo, khi), and those that all do, [flo, fhi).  Columns
// beyond the tile's (lo = -1) see everything and count for neither.
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

// The slice's steps of `step` keys of the tile's [klo, khi).
__device__ __forceinline__ void ca_steps(const CaWork& w, int klo, int khi, int step, int& it, int& end) {
  it = end = 0;
  if (khi <= klo) return;
  const int u0 = klo / step, n = (khi + step - 1) / step - u0;
  it = u0 + (int)((int64_t)n * w.slice / w.slices);
  end = u0 + (int)((int64_t)n * (w.slice + 1) / w.slices);
}

// 4 N rows from `row0` of one tensor into LDS, whose place there is row i0 of a tile (a multiple of 4): row i
// at 256 i, its 16-byte chunk C at place C ^ x(i), x(i) = i & 15 for K (a lane reads chunk 4 ks + q of row
// r) and 2 (i & 7) for V (the transposing read takes 32 bytes of each of 16 rows).  Rows past the
// last are the last one again.
template <bool IS_V, int N>
__device__ __forceinline__ void ca_fetch(const uint16_t* base, int64_t rs, int row0, int n_keys, int i0, uint32_t lds) {
  int lane = ls_lane();
  asm volatile("" : "+v"(lane));  // offsets are formed here, not kept in registers over a loop
  const int i4 = lane >> 4;
  const uint32_t rb = 2 * (uint32_t)rs;
  auto chunk = [&](int j) {
    const int i = i0 + 4 * j + i4;
    return 16 * ((uint32_t)(lane & 15) ^ (uint32_t)(IS_V ? 2 * (i & 7) : i & 15));
  };
  if (row0 + 4 * N <= n_keys) {
    const uint16_t* p = base + (int64_t)row0 * rs;
#pragma unroll
    for (int j = 0; j < N; ++j) ls_dma16(p + 4 * j * rs, (uint32_t)i4 * rb + chunk(j), lds + 1024 * j);
  } else {
    const int first = min(row0, n_keys - 1);
    const uint16_t* p = base + (int64_t)first * rs;
#pragma unroll
    for (int j = 0; j < N; ++j)
      ls_dma16(p, (uint32_t)(min(row0 + 4 * j + i4, n_keys - 1) - first) * rb + chunk(j), lds + 1024 * j);
  }
}

template <int DT>
__device__ __forceinline__ void ca_out4(uint16_t* p, ls_f32x4 v, float inv) {
  uint2 w;
  w.x = ls_pack2(LsElem<DT>::from_f(v[0] * inv), LsElem<DT>::from_f(v[1] * inv));
  w.y = ls_pack2(LsElem<DT>::from_f(v[2] * inv), LsElem<DT>::from_f(v[3] * inv));
  *reinterpret_cast<uint2*>(p) = w;
}

__device__ __forceinline__ float ca_lse(float M, float L) {
  return L == 0.f ? INFINITY : (M + log2f(L)) * kLn2;
}

// Whether the workgroup's rows are its own alone; else the first of a tile's tells the join.
__device__ __forceinline__ bool ca_alone(const CaArgs& a, const CaWork& w) {
  return a.part == nullptr || (a.pre.items == 0 && w.slices == 1);
}

// Four channels (chunk ch of 32) of a column's sums: the final values, or the item's for the join.
template <int DT>
__device__ __forceinline__ void ca_store(const CaArgs& a, const CaWork& w, const CaCut& cut, bool alone, int c, int tk,
                                         int h, int ch, float M, float L, ls_f32x4 v) {
  const int64_t row = (int64_t)(w.t0 + tk) * (a.G * a.gs) + w.g * a.gs + h;
  if (alone) {
    ca_out4<DT>(a.out + row * kDim + 4 * ch, v, L == 0.f ? 0.f : 1.f / L);
    if (ch == 0 && a.lse) a.lse[(int64_t)(w.g * a.gs + h) * a.total_q + w.t0 + tk] = ca_lse(M, L);
  } else {
    const int64_t place = (w.seq < 0 ? (int64_t)w.item * cut.cols
                                     : (int64_t)a.pre.items * a.pre.cols + (int64_t)(w.item - a.pre.items) * cut.cols) + c;
    if (L != 0.f) *reinterpret_cast<ls_f32x4*>(a.part + place * kDim + 4 * ch) = v;
    if (ch == 0) a.ml[place] = make_float2(M, L);
  }
  if (ch == 0 && a.part && w.seq >= 0 && w.slice == 0)
    a.rows[row] = alone ? make_int4(0, 0, 0, 1) : make_int4(w.base, w.slices << 8 | c, w.tile, w.tiles);
}

// ---------------------------------------------------------------------------
// Keys form, few columns (16).  Each key's bytes are read from LDS once, by one wave, from a place of
// the wave's own, with no barrier: the next step's K is on its way from when this one's has been
// read, V likewise.  The waves' sums are joined through LDS at the end.  128 KB of a unit's keys are on
// their way at a time: 4.6 TB/s on sixteen ragged sequences.
// ---------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void ca_keys_form(const CaArgs& a, const CaWork& w, const CaCut& cut, uint32_t lds,
                                             float* s_m, float* s_l) {
  constexpr int NC = 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  CaState<NC> st;
  ca_columns<NC>(a, w, cut.tokens, 0, st);
  int klo, khi, flo, fhi, it, end;
  ca_range<NC>(st, klo, khi, flo, fhi);
  ca_steps(w, klo, khi, kKeysStep, it, end);
  const int sub = wave * kKeysSub;
  while (it < end && (end - 1) * kKeysStep + sub >= khi) --end;  // the last step may not reach this wave
  while (it < end && it * kKeysStep + sub + kKeysSub <= klo) ++it;
  const uint32_t mine = lds + 2 * wave * kSubB;
  auto fetch_k = [&](int i) { ca_fetch<false, 8>(w.k, w.rs, i * kKeysStep + sub, w.n_keys, 0, mine); };
  auto fetch_v = [&](int i) { ca_fetch<true, 8>(w.v, w.rs, i * kKeysStep + sub, w.n_keys, 0, mine + kSubB); };
  if (it < end) {
    fetch_k(it);
    fetch_v(it);
  }
  auto full = [&](int i) { return i * kKeysStep + sub >= flo && i * kKeysStep + sub + kKeysSub <= fhi; };
  auto step = [&](auto is_full) {
    const bool more = it + 1 < end;
    CA_WAIT_VM(8);  // V behind K
    ca_step<DT, NC, 2, decltype(is_full)::value>(
        mine, mine + kSubB, it * kKeysStep + sub, st, a,
        [&]() {
          CA_WAIT_LDS();
          if (more) fetch_k(it + 1);
        },
        [&]() {
          if (more) CA_WAIT_VM(8);
          else CA_WAIT_VM(0);
        },
        [&]() {
          CA_WAIT_LDS();
          if (more) fetch_v(it + 1);
        });
  };
  while (it < end) {  // (loops of their own: the sums stay in one set of registers)
    for (; it < end && !full(it); ++it) step(std::false_type());
    for (; it < end && full(it); ++it) step(std::true_type());
  }
  // The waves' sums: column c's 128 values at 512 c, 16-byte chunk C at place C ^ (c & 15).
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    const int c = 16 * nc + r;
    const float l = st.l[nc][0];
    if (q == 0) {
      s_m[wave * kKeysCols + c] = st.m[nc];
      s_l[wave * kKeysCols + c] = l;
    }
#pragma unroll
    for (int db = 0; db < 8; ++db)
      *(CaLdsF4*)(mine + 512 * c + 16 * ((4 * db + q) ^ r)) = st.o[db][nc];
  }
  __syncthreads();
  const int c = tid >> 5, ch = tid & 31, tk = c / a.gs, h = c - tk * a.gs;
  if (tk >= cut.tokens || w.t0 + tk >= w.t1) return;
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) M = fmaxf(M, s_m[i * kKeysCols + c]);
  ls_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const float m = s_m[i * kKeysCols + c], l = s_l[i * kKeysCols + c];
    if (l == 0.f) continue;  // nothing visible
    const float f = m == M ? 1.f : __builtin_amdgcn_exp2f(m - M);
    L += f * l;
    v += f * *(CaLdsF4*)(lds + 2 * i * kSubB + 512 * c + 16 * (ch ^ (c & 15)));
  }
  ca_store<DT>(a, w, cut, ca_alone(a, w), c, tk, h, ch, M - CaBias<DT>::value, L, v);
}

// ---------------------------------------------------------------------------
// Rows form, many columns: 32 a wave, so that what is read from LDS (two bytes for every 32 multiplications
// of a key's element) keeps up with the matrix units.  A ring of four steps of 64 keys; each wave fetches 8
// rows of a step's K and V.  A barrier every two steps tells that the next two have come and the two
// before have been read (every step: 1078 us for the chunk at the time, every two 1027).  The sums, scores and
// weights of a wave take its registers; nothing may go to scratch memory, whose loads wait for the
// keys on their way (with it: 2550).
// ---------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void ca_rows_form(const CaArgs& a, const CaWork& w, const CaCut& cut, uint32_t lds,
                                             int* s_range) {
  constexpr int NC = 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  CaState<NC> st;
  ca_columns<NC>(a, w, cut.tokens, 16 * NC * wave, st);
  int klo, khi, flo, fhi, it, end;
  ca_range<NC>(st, klo, khi, flo, fhi);
  if (lane == 0) {
    s_range[wave] = klo;
    s_range[kWaves + wave] = khi;
  }
  __syncthreads();
  int lo_all = s_range[0], hi_all = s_range[kWaves];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) {
    lo_all = min(lo_all, s_range[i]);
    hi_all = max(hi_all, s_range[kWaves + i]);
  }
  lo_all = __builtin_amdgcn_readfirstlane(lo_all);
  hi_all = __builtin_amdgcn_readfirstlane(hi_all);
  ca_steps(w, lo_all, hi_all, kRowsStep, it, end);
  auto fetch = [&](int i) {
    const uint32_t to = lds + (uint32_t)(i & (kRing - 1)) * 2 * kRowsB + 2048 * wave;
    ca_fetch<false, 2>(w.k, w.rs, i * kRowsStep + 8 * wave, w.n_keys, 8 * wave, to);
    ca_fetch<true, 2>(w.v, w.rs, i * kRowsStep + 8 * wave, w.n_keys, 8 * wave, to + kRowsB);
  };
  auto fetch_pair = [&](int i) {
    if (i < end) fetch(i);
    if (i + 1 < end) fetch(i + 1);
  };
  const int begin = it;
  fetch_pair(it);
  auto next = [&]() {
    if ((it - begin) & 1) return;
    CA_WAIT_VM(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    fetch_pair(it + 2);
  };
  // (a wave without columns only fetches)
  auto full = [&](int i) { return khi > klo && i * kRowsStep >= flo && i * kRowsStep + kRowsStep <= fhi; };
  auto step = [&](auto is_full) {
    const uint32_t sk = lds + (uint32_t)(it & (kRing - 1)) * 2 * kRowsB;
    ca_step<DT, NC, 4, decltype(is_full)::value>(sk, sk + kRowsB, it * kRowsStep, st, a, []() {}, []() {},
                                                 []() { CA_WAIT_LDS(); });
  };
  while (it < end) {  // (loops of their own: the sums stay in one set of registers)
    for (; it < end && !full(it); ++it) {
      next();
      if (it * kRowsStep < khi && it * kRowsStep + kRowsStep > klo) step(std::false_type());
    }
    for (; it < end && full(it); ++it) {
      next();
      step(std::true_type());
    }
  }
  const bool alone = ca_alone(a, w);
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    const int c = 16 * (NC * wave + nc) + r, tk = c / a.gs, h = c - tk * a.gs;
    if (tk >= cut.tokens || w.t0 + tk >= w.t1) continue;
#pragma unroll
    for (int db = 0; db < 8; ++db)
      ca_store<DT>(a, w, cut, alone, c, tk, h, 4 * db + q, st.m[nc] - CaBias<DT>::value, st.l[nc][0], st.o[db][nc]);
  }
}

// Forms: 0: no such items, 1: keys, 2: rows.
template <int DT, int FORM>
__device__ __forceinline__ void ca_form(const CaArgs& a, const CaWork& w, const CaCut& cut, uint32_t lds, float* small) {
  if constexpr (FORM == 1) ca_keys_form<DT>(a, w, cut, lds, small, small + kKeysCols * kWaves);
  if constexpr (FORM == 2) ca_rows_form<DT>(a, w, cut, lds, reinterpret_cast<int*>(small));
}

template <int DT, int PRE, int OWN>
__global__ __launch_bounds__(kThreads) void ls_cache_attn_kernel(const CaArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kLdsBytes];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring;
  __shared__ float small[2 * kKeysCols * kWaves];
  const int item = blockIdx.x;
  const bool prefix = PRE != 0 && item < a.pre.items;
  CaWork w;
  if (!(prefix ? ca_prefix_work(a, item, w) : ca_own_work(a, item - a.pre.items, w))) return;
  if constexpr (PRE == OWN || PRE == 0)
    ca_form<DT, OWN>(a, w, prefix ? a.pre : a.own, lds, small);
  else if (prefix)
    ca_form<DT, PRE>(a, w, a.pre, lds, small);
  else
    ca_form<DT, OWN>(a, w, a.own, lds, small);
}

// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over a row's slices, the prefix's and its own.  SHARE
// half waves per (row, head), each every SHARE-th slice, four channels a lane: 8 where a row has many slices, so
// that 32 of them are on their way at once, 1 where it has few.
template <int DT, int SHARE>
__global__ __launch_bounds__(256) void ls_cache_attn_join_kernel(const CaArgs a) {
  const int tid = threadIdx.x;
  const int H = a.G * a.gs;
  const int64_t row = SHARE == 8 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 8 + (tid >> 5);
  if (row >= a.total_q * H) return;
  const int t = (int)(row / H), head = (int)(row % H), g = head / a.gs, h = head % a.gs;
  if (t < a.cu_q[0] || t >= a.cu_q[a.batch]) return;
  const int4 own = a.rows[row];
  if (own.y <= 0) return;               // written already
  const int before = a.pre.items ? a.pre.slices : 0;
  // (in bounds whatever cu_seqlens_q holds)
  const int own_slices = min(own.y >> 8, a.own.items), own_col = min(own.y & 255, a.own.cols - 1);
  const int slots = before + own_slices, tiles = max(1, own.w);
  auto place = [&](int s) -> int64_t {
    if (s < before)
      return (int64_t)ca_join_item(s * a.G + g, t / a.pre.tokens, a.pre.slices * a.G, a.pre.tiles) * a.pre.cols +
             t % a.pre.tokens * a.gs + h;
    const int at = own.x + ca_join_item((s - before) * a.G + g, own.z, own_slices * a.G, tiles);
    return (int64_t)a.pre.items * a.pre.cols + (int64_t)min(max(at, 0), a.own.items - 1) * a.own.cols + own_col;
  };
  // The maximum of all, a slice a thread.
  const int ch = tid & 31, at = SHARE == 8 ? tid >> 5 : 0;
  float M = -INFINITY;
  for (int s = SHARE == 8 ? tid : ch; s < slots; s += 32 * SHARE) M = fmaxf(M, a.ml[place(s)].x);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, ls_shfl_xor(M, o));
  __shared__ float s_m[8], s_l[8];
  __shared__ ls_f32x4 s_o[8][32];
  if (SHARE == 8) {
    if (ch == 0) s_m[at] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) M = fmaxf(M, s_m[i]);
  }
  ls_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int s0 = at; s0 < slots; s0 += 4 * SHARE) {
    ls_f32x4 v[4];
    float2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t p = place(min(s0 + SHARE * i, slots - 1));
      x[i] = a.ml[p];
      v[i] = *reinterpret_cast<const ls_f32x4*>(a.part + p * kDim + 4 * ch);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s0 + SHARE * i >= slots || x[i].y == 0.f) continue;  // (one without a visible key has no sums)
      const float f = x[i].x == M ? 1.f : __builtin_amdgcn_exp2f(x[i].x - M);
      L += f * x[i].y;
      acc += f * v[i];
    }
  }
  if (SHARE == 8) {
    s_o[at][ch] = acc;
    if (ch == 0) s_l[at] = L;
    __syncthreads();
    if (tid >= 32) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      acc += s_o[i][ch];
      L += s_l[i];
    }
  }
  ca_out4<DT>(a.out + row * kDim + 4 * ch, acc, L == 0.f ? 0.f : 1.f / L);
  if (ch == 0 && a.lse) a.lse[(int64_t)head * a.total_q + t] = ca_lse(M, L);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int kUnits = 256;  // compute units
constexpr int kMaxSplits = 128;
// Above the largest cap the score's error would be more than the output's rounding in fp16; a form that is exact there
// (the series of tanh near 0) in the same loop took 6% of the chunk's time from every other cap.
constexpr float kMinCap = 1e-20f, kMaxCap = 512.f;

struct CaPlan {
  CaCut pre, own;
  size_t part, ml, total;  // total 0: no join
};

CaPlan ca_plan(int64_t total_q, int batch, int H, int G, int64_t p_len, int64_t max_len, int left, int n_splits) {
  // A workgroup has a unit to itself.  What one takes, in us: a step of 256 keys of 16 columns, or of 64
  // keys of 256; and what stands in front of and behind its steps.
  constexpr double kKeysUs = 1.6, kRowsUs = 3.0, kItemUs = 8.0;
  CaPlan p = {};
  const int gs = H / G;
  const int64_t rows = (total_q + batch - 1) / batch;  // of a sequence
  auto shape = [&](CaCut& c, int64_t cols) {
    c.cols = cols <= kKeysCols ? kKeysCols : kRowsCols;
    c.tokens = std::max(1, c.cols / gs);
    return c.cols == kKeysCols ? kKeysStep : kRowsStep;
  };
  auto count = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
  // The own keys' tiles, G groups of them, and the most steps that one has to take.
  struct Own {
    int step;
    double us;
    int64_t tiles, steps;
  };
  auto cut_own = [&](int64_t cols) {
    Own o;
    o.step = shape(p.own, cols);
    o.us = p.own.cols == kKeysCols ? kKeysUs : kRowsUs;
    p.own.tiles = (int)std::min<int64_t>(total_q, (total_q + (int64_t)batch * (p.own.tokens - 1)) / p.own.tokens);
    o.tiles = (int64_t)p.own.tiles * G;
    const int64_t seen = left >= 0 ? std::min<int64_t>(max_len, (int64_t)left + p.own.tokens) : max_len;
    o.steps = std::max<int64_t>(1, count(seen, o.step));
    return o;
  };
  auto balanced = [&](const Own& o) {
    return std::min<int64_t>(o.tiles * o.steps, std::max<int64_t>(kUnits, o.tiles + kUnits / 2));
  };
  Own own = cut_own(rows * gs);
  if (rows * gs > kKeysCols && rows * gs <= kManyCols) {
    // Two to four tiles of 16 columns, or one of 256 that is mostly empty.  With all units at it a step of the
    // first takes what its keys take to arrive: 3.5 us where a die's cache serves a slice's other tiles, else
    // 5.4; the second needs no more of them, but fewer units have work and its prologue and join take 20 us.
    // 8 and 24 sequences of 32K, 32 heads to 2, in us, the first against the second: 2 rows 49 / 88 and 202 /
    // 263, 3 rows 52 / 98 and 288 / 238, 4 rows 81 / 99 and 375 / 236; one sequence 21 / 33.
    const Own many = own;
    own = cut_own(kKeysCols);
    const double c = balanced(own) * G >= 8 * own.tiles ? 3.5 : 5.4;
    if ((double)(own.tiles * own.steps) / kUnits * c + kItemUs > (double)(many.tiles * many.steps) / kUnits * kRowsUs + 20.0)
      own = cut_own(rows * gs);
  }
  const double own_us = own.us;
  const int64_t tiles = own.tiles, steps = own.steps;
  if (p_len > 0) {
    const int step = shape(p.pre, total_q * gs);
    p.pre.tiles = (int)count(total_q, p.pre.tokens);
    const int64_t pre_tiles = (int64_t)p.pre.tiles * G, pre_steps = count(p_len, step);
    // Some units take the own keys' items one after the other while the rest take a slice of the prefix each.
    const double pre_us = pre_tiles * pre_steps * (p.pre.cols == kKeysCols ? kKeysUs : kRowsUs);
    const double each = (tiles * (steps * own_us + kItemUs) + pre_us) / kUnits + kItemUs;
    const int64_t slices = n_splits > 0 ? n_splits : std::max<int64_t>(1, (int64_t)(2 * steps * own_us / each));
    p.own.slices = (int)std::min<int64_t>({slices, std::max<int64_t>(steps, n_splits), kMaxSplits});
    const double busy = tiles * (steps * own_us + p.own.slices * kItemUs) / each;
    // (the same number of units on each of the eight dies, to which items go in turn)
    const int64_t spare = std::max<int64_t>(1, kUnits - 8 * ((int64_t)(busy / 8) + 1));
    p.pre.slices = (int)std::max<int64_t>(
        1, std::min<int64_t>({n_splits > 0 ? n_splits : spare / pre_tiles, pre_steps, kMaxSplits}));
    p.pre.items = p.pre.tiles * p.pre.slices * G;
    p.own.items = (int)std::min<int64_t>(tiles * p.own.slices, 0x7fffffff);
  } else if (n_splits > 0) {
    p.own.slices = n_splits;
    p.own.items = (int)std::min<int64_t>(tiles * n_splits, 0x7fffffff);
  } else if (p.own.cols == kKeysCols) {
    p.own.slices = 0;
    p.own.items = (int)balanced(own);
  } else {
    // Rounds of a workgroup a unit: the number of slices that makes them shortest (more than one
    // are also written, and joined).
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && s <= steps; ++s) {
      const double us = count(tiles * s, kUnits) * (kRowsUs * count(steps, s) + kItemUs) + (s > 1 ? 2 * kItemUs : 0.0);
      if (us < least) least = us, best = s;
    }
    p.own.slices = best;
    p.own.items = (int)std::min<int64_t>(tiles * best, 0x7fffffff);
  }
  if (p.pre.items > 0 || p.own.items > tiles) {
    const size_t places = (size_t)p.pre.items * p.pre.cols + (size_t)p.own.items * p.own.cols;
    p.part = ls_align256(4 * places * kDim);
    p.ml = ls_align256(8 * places);
    p.total = p.part + p.ml + 16 * (size_t)total_q * H;
  }
  return p;
}

template <int DT, int PRE, int OWN>
void ca_launch(const CaArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((ls_cache_attn_kernel<DT, PRE, OWN>), dim3((unsigned)(a.pre.items + a.own.items)),
                     dim3(kThreads), 0, s, a);
}

template <int DT>
void ca_by_form(const CaArgs& a, hipStream_t s) {
  const bool keys = a.own.cols == kKeysCols;
  if (a.pre.items == 0) return keys ? ca_launch<DT, 0, 1>(a, s) : ca_launch<DT, 0, 2>(a, s);
  if (a.pre.cols == kKeysCols) return ca_launch<DT, 1, 1>(a, s);  // (then the own ones, too)
  keys ? ca_launch<DT, 2, 1>(a, s) : ca_launch<DT, 2, 2>(a, s);
}

}  // namespace

extern "C" size_t ls_cache_attn_workspace_size(int64_t total_q, int32_t batch, int32_t num_heads,
                                               int32_t num_kv_heads, int64_t prefix_len, int64_t max_len,
                                               int32_t window_left, int32_t n_splits) {
  if (total_q <= 0 || batch <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads || prefix_len < 0) return 0;
  return ca_plan(total_q, batch, num_heads, num_kv_heads, prefix_len, max_len, window_left, n_splits).total;
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
  LS_REQUIRE(softcap == 0.f || (softcap >= kMinCap && softcap <= kMaxCap), LS_ERR_UNSUPPORTED,
             "%s: softcap must be 0 or from %g to %g", who, kMinCap, kMaxCap);
  LS_REQUIRE(n_splits >= 0 && n_splits <= kMaxSplits, LS_ERR_INVALID, "%s: 0 <= n_splits <= %d", who,
             kMaxSplits);
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
  const CaPlan p = ca_plan(total_q, batch, num_heads, num_kv_heads, prefix_len, max_len, window_left, n_splits);
  LS_REQUIRE(workspace_bytes >= p.total && (p.total == 0 || workspace), LS_ERR_WORKSPACE,
             "%s: workspace %zu < %zu", who, workspace_bytes, p.total);
  LS_REQUIRE((int64_t)p.pre.items + p.own.items < (1 << 22) && total_q * num_heads < (1 << 23),
             LS_ERR_UNSUPPORTED, "%s: more workgroups than a launch holds", who);
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
  a.alpha = softcap > 0.f ? 2.f * softcap * kLog2e : softmax_scale * kLog2e;
  a.beta = softcap > 0.f ? softcap * kLog2e : 0.f;
  // (a factor past float32's range either way gives what its end does: +-cap for any product but 0, or 0 for all)
  a.cap_b = softcap > 0.f ? (float)std::min(std::max(2.0 * softmax_scale * kLog2e / softcap, 0x1p-126), 0x1.fffffep127)
                          : 0.f;
  a.slopes = alibi_slopes;
  a.slopes_bs = alibi_batch_stride;
  a.causal = causal != 0;
  a.left = window_left < 0 ? -1 : std::min(window_left, 1 << 30);
  a.right = window_right < 0 ? -1 : std::min(window_right, (1 << 30) - 1);
  a.pre = p.pre;
  a.own = p.own;
  if (p.total) {
    a.part = (float*)workspace;
    a.ml = (float2*)((uint8_t*)workspace + p.part);
    a.rows = (int4*)((uint8_t*)workspace + p.part + p.ml);
  }
  a.out = (uint16_t*)out;
  a.lse = softmax_lse;
  hipStream_t s = (hipStream_t)stream;
  dtype == LS_BF16 ? ca_by_form<LS_BF16>(a, s)
                   : ca_by_form<LS_F16>(a, s);
  int rc = ls_check_launch("ls_cache_attn_kernel");
  if (rc || !p.total) return rc;
  const int64_t all = total_q * num_heads;
  const bool few = p.own.slices > 0 && p.pre.slices + p.own.slices <= 8;
  auto join = [&](auto one, auto eight) {
    hipLaunchKernelGGL(few ? one : eight, dim3((unsigned)(few ? (all + 7) / 8 : all)), dim3(256), 0, s, a);
  };
  if (dtype == LS_BF16)
    join(ls_cache_attn_join_kernel<LS_BF16, 1>, ls_cache_attn_join_kernel<LS_BF16, 8>);
  else
    join(ls_cache_attn_join_kernel<LS_F16, 1>, ls_cache_attn_join_kernel<LS_F16, 8>);
  return ls_check_launch("ls_cache_attn_join_kernel");
}
