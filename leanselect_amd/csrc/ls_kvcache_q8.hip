// Decode over a KV cache held in 8 bits: quantising append and attention.
//
// Cache layout (the caller's tensors), a page being 64 tokens of one KV head:
//   k8 [batch][pages][G][64 tokens][128]  e4m3
//   v8 [batch][pages][G][128][64 tokens]  e4m3, a channel's 64 tokens together,
//                                          token 16 t + 4 q + i at place 16 q + 4 t + i
//   k_scale, v_scale [batch][pages][G]    uint8 codes, code c standing for 2^(c - 127)
// An element stands for its e4m3 value times its page's power of two.  The code of a
// page is the least c >= 1 with max |x| <= 448 2^(c - 127) over the finite rows it has
// held since its first token, so nothing saturates; a power of two costs no precision
// (e4m3 is a float) and changing it leaves a stored row exact unless it becomes subnormal.
// Infinities and NaN are stored as NaN (e4m3 has no infinity) and do not count for the code.
//
// The orders are those in which the attention's matrix instructions read a page, so a
// wave takes it from memory to registers in 16-byte loads without LDS:
// S^T = K Q^T (rows are keys) gives lane (r, q) = (lane & 15, lane >> 4) the scores of head
// r and tokens 16 t + 4 q + i, and P^T is the right operand of O^T = V^T P^T as it stands
// when lane (r, q)'s 16 bytes of a channel's values are the tokens 16 t + 4 q + i.
//
// Extends ls_kvcache_append, ls_sparse_attn_kvcache and ls_dense_attn_kvcache (the
// reference's cache is 16-bit: leanselect/models/minicpm.py:1188-1490).
#include <algorithm>
#include <type_traits>

#include "ls_common.h"

namespace {

constexpr int kPage = 64;
constexpr int kDim = 128;
constexpr int kPageBytes = kPage * kDim;

typedef float Q8F2 __attribute__((ext_vector_type(2)));

// Largest finite magnitude of eight 16-bit values as 16 bits (their order is that of the
// values); an infinity or NaN counts as zero.
template <int DT>
__device__ __forceinline__ uint32_t q8_abs_max(ls_u32x4 x, uint32_t top) {
  constexpr uint32_t kInf = DT == LS_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = x[e] & 0x7fffu, hi = (x[e] >> 16) & 0x7fffu;
    top = max(top, lo < kInf ? lo : 0u);
    top = max(top, hi < kInf ? hi : 0u);
  }
  return top;
}

// The least code c >= 1 with m <= 448 2^(c - 127): 448 = 1.75 2^8.
template <int DT>
__device__ __forceinline__ uint32_t q8_code(uint32_t top16) {
  const uint32_t bits = __float_as_uint(LsElem<DT>::to_f((uint16_t)top16));
  const int c = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(c, 1);
}

// 2^(e - 127) for e in [1, 254].
__device__ __forceinline__ float q8_pow(int e) { return __uint_as_float((uint32_t)e << 23); }

// Four floats as four e4m3 bytes, to nearest even (overflow and non-finite: NaN).
__device__ __forceinline__ uint32_t q8_pack(float a, float b, float c, float d) {
  uint32_t v = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, (int)v, true);
}

// Four stored bytes under a smaller power: times f, rounded to e4m3 again.
__device__ __forceinline__ uint32_t q8_rescale(uint32_t v, float f) {
  const Q8F2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false);
  const Q8F2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
  return q8_pack(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

// The sequence that gets the `unit`-th of the batch's pages with new rows, in order, its length
// and its new rows [n0, n1); `unit` becomes the page's number among the sequence's.  -1 past the
// last page.  A wave scans 64 sequences at a time, and what it found stays in its lanes.
__device__ __forceinline__ int q8_find(int& unit, int batch, const int32_t* __restrict__ lens,
                                       const int32_t* __restrict__ cu_new, int& len, int& n0, int& n1) {
  const int lane = ls_lane();
  for (int s0 = 0; s0 < batch; s0 += 64) {
    const int i = min(s0 + lane, batch - 1);
    const int l = lens[i], lo = cu_new[i], hi = cu_new[i + 1];
    const bool some = s0 + lane < batch && hi > lo && l >= 0 && lo >= 0;
    const int mine = some ? (int)(((int64_t)l + (hi - lo) + kPage - 1) / kPage) - l / kPage : 0;
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
      len = __builtin_amdgcn_readlane(l, at);
      n0 = __builtin_amdgcn_readlane(lo, at);
      n1 = __builtin_amdgcn_readlane(hi, at);
      return s0 + at;
    }
    unit -= __builtin_amdgcn_readlane(upto, 63);
  }
  return -1;
}

// ---------------------------------------------------------------------------
// Append: a workgroup per (page that gets new rows, KV head).  It finds the largest
// magnitude of the page's new rows, takes the page's code (at least the old one where the
// page holds older rows), brings older rows under a raised code, and writes the new rows.
// A page of a sequence belongs to one workgroup, so nothing is shared between them.
// K: thread (r, c) takes 8 channels of the rows r, r + 16, r + 32, r + 48.
// V: thread (quad, octet) takes 8 channels of the four tokens that share a 4-byte word.
//
// Compressed keys: window w is the mean of the 32 stored keys from token 16 w, so it is two
// of the 16-row halves of pages.  The halves of the page are summed from the bytes in LDS,
// with the last half of the page before and the first of the page after.  A window across
// two pages belongs to the first one if the call writes to it: the second one's rows are
// then all new, and their code and bytes are formed here once more from the new keys (a
// page's older rows may be changing under another workgroup's hands, its new ones not).
// Otherwise the first page is at rest and is read as it is.  So the windows need no second
// launch: 3 to 5 us a call, against reading a prompt's keys twice.
//
// Bound by memory for prompts (32768 tokens of two heads: 12.7 us without windows, 50 MB at 4.0
// TB/s, a copy of the same rows 12.1; 15.3 with them), by a launch and the chain of lengths,
// rows, code and stores for a step (16 sequences, a token each: 5.1 us, 5.9 where windows end;
// with conditional loads, each waited for before the next, 6.2 and 7.0).
// ---------------------------------------------------------------------------
// Eight 16-bit values as eight e4m3 bytes under a scale.
template <int DT>
__device__ __forceinline__ uint2 q8_pack8(ls_u32x4 x, float inv) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = LsElem<DT>::to_f((uint16_t)(x[e] & 0xffffu)) * inv;
    f[2 * e + 1] = LsElem<DT>::to_f((uint16_t)(x[e] >> 16)) * inv;
  }
  return make_uint2(q8_pack(f[0], f[1], f[2], f[3]), q8_pack(f[4], f[5], f[6], f[7]));
}

// (One argument: a launch with twenty costs the host 0.6 us more.)
struct Q8AppendArgs {
  uint8_t* k8;
  uint8_t* v8;
  int64_t cbs;
  uint8_t* ks;
  uint8_t* vs;
  int64_t sbs;
  int64_t pages;
  const int32_t* cache_seqlens;
  const uint16_t* kn;
  const uint16_t* vn;
  int64_t nrs;
  const int32_t* cu_new;
  int64_t total_new;
  int batch;
  int G;
  uint16_t* kcc;
  int64_t kbs;
  int64_t krs;
  int64_t kc_rows;
};

template <int DT>
__global__ __launch_bounds__(256) void ls_q8_append_kernel(const Q8AppendArgs args) {
  uint8_t* __restrict__ k8 = args.k8;
  uint8_t* __restrict__ v8 = args.v8;
  const int64_t cbs = args.cbs;
  uint8_t* __restrict__ ks = args.ks;
  uint8_t* __restrict__ vs = args.vs;
  const int64_t sbs = args.sbs;
  const int64_t pages = args.pages;
  const int32_t* __restrict__ cache_seqlens = args.cache_seqlens;
  const uint16_t* __restrict__ kn = args.kn;
  const uint16_t* __restrict__ vn = args.vn;
  const int64_t nrs = args.nrs;
  const int32_t* __restrict__ cu_new = args.cu_new;
  const int64_t total_new = args.total_new;
  const int batch = args.batch;
  const int G = args.G;
  uint16_t* __restrict__ kcc = args.kcc;
  const int64_t kbs = args.kbs;
  const int64_t krs = args.krs;
  const int64_t kc_rows = args.kc_rows;
  __shared__ uint32_t s_top[3][4];
  // Keys by half of a page: the last one before, the page's four, the first one after.
  constexpr int kPitch = kDim + 4;
  __shared__ uint32_t s_k[96 * kPitch / 4];
  __shared__ ls_f32x4 s_half[6][kDim / 4];
  constexpr int kVPitch = kPage + 4;
  __shared__ uint32_t s_v[kDim * kVPitch / 4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int g = blockIdx.y;
  // Workgroups go to the eight compute dies in turn: of each 128 pages a die takes 16 in a row, so
  // that the next page's keys are in its cache (32768 tokens 17.0 -> 15.5 us; a die's whole share
  // in a row 15.9, and 131072 tokens 49.2 against 44.8).
  int unit = blockIdx.x, len_b, n0_b, n1_b;
  if (unit < (int)(gridDim.x & ~127u)) unit = (unit & ~127) | (unit & 7) << 4 | (unit >> 3 & 15);
  const int b = q8_find(unit, batch, cache_seqlens, cu_new, len_b, n0_b, n1_b);
  if (b < 0) return;
  const int64_t len = len_b, n0 = n0_b, n1 = min((int64_t)n1_b, total_new);
  const int64_t page = len / kPage + unit;
  const int64_t base = page * kPage, end = len + (n1 - n0);
  if (page >= pages || base >= end || len >= end) return;  // (the later two: offsets past total_new)
  const int r0 = (int)max<int64_t>(0, len - base);  // the page's new rows: r0 <= row < r1
  const int r1 = (int)min<int64_t>(kPage, end - base);
  const int64_t at = (int64_t)b * cbs + (page * G + g) * kPageBytes;
  const int64_t sat = (int64_t)b * sbs + page * G + g;
  const int64_t first = (n0 + base - len) * nrs + (int64_t)g * kDim;  // the page's row 0, if it were new

  // The window of halves i and i + 1 (0: the page before's last and the page's first).
  const int after = page + 1 < pages ? (int)max<int64_t>(0, min<int64_t>(kPage, end - base - kPage)) : 0;
  auto complete = [&](int i) {
    if (!kcc) return false;
    if (i == 4) return after >= 16;
    return r0 <= 16 * i + 15 && 16 * i + 15 < r1 && (i > 0 || (unit == 0 && page > 0));
  };
  const bool windows = complete(0) || complete(1) || complete(2) || complete(3) || complete(4);

  const int krow = tid >> 4, kc = 8 * (tid & 15);  // rows krow + 16 j
  auto knew = [&](int j) { return krow + 16 * j >= r0 && krow + 16 * j < r1; };
  const int quad = tid >> 4, oct = tid & 15;  // quad = 4 q + t
  const int tok = 16 * (quad & 3) + 4 * (quad >> 2);
  ls_u32x4 kx[4], vx[4], nx[4];
  uint2 ko[4];
  uint32_t ktop = 0, vtop = 0, ntop = 0;
  // Every load is made on one path, in front of the first wait: where a row is not new, a new
  // one takes its place (it changes no maximum and is not written).
  auto held = [&](int row) { return (int64_t)min(max(row, r0), r1 - 1) * nrs; };
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kx[j] = ls_load16(kn + first + held(krow + 16 * j) + kc);
    vx[j] = ls_load16(vn + first + held(tok + j) + 8 * oct);
  }
  uint8_t* kp = k8 + at + krow * kDim + kc;
  if (r0 > 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) ko[j] = *reinterpret_cast<const uint2*>(kp + 16 * kDim * j);
  }
  // Bytes of a V word that are new, and those that are older; the words as they are, where
  // some of a word is new.  (Wholly older words are read later, if the page's code rises.)
  uint32_t is_new = 0, is_old = 0, vo[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (tok + j >= r0 && tok + j < r1) is_new |= 0xffu << (8 * j);
    if (tok + j < r0) is_old |= 0xffu << (8 * j);
  }
  uint8_t* vp = v8 + at + (8 * oct) * kPage + 4 * quad;
  if (is_new != 0 && is_new != 0xffffffffu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vo[e] = *reinterpret_cast<const uint32_t*>(vp + e * kPage);
  }
  uint32_t kold = ks[sat], vold = vs[sat];
  if (r0 == 0) kold = vold = 1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ktop = q8_abs_max<DT>(kx[j], ktop);
    vtop = q8_abs_max<DT>(vx[j], vtop);
  }
  // The next page's keys after this page's have come: by then its own workgroup has read them.
  // They are not looked at before this page is written (131072 tokens 44.8 -> 42.7 us).
  if (complete(4)) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      nx[j] = ls_load16(kn + first + (kPage + min(krow + 16 * j, after - 1)) * nrs + kc);
  }
  ktop = ls_wave_max_u32(ktop);
  vtop = ls_wave_max_u32(vtop);
  if (lane == 0) {
    s_top[0][w] = ktop;
    s_top[1][w] = vtop;
  }
  __syncthreads();
  auto all_waves = [&](int i) { return max(max(s_top[i][0], s_top[i][1]), max(s_top[i][2], s_top[i][3])); };
  const uint32_t kcode = max(q8_code<DT>(all_waves(0)), kold);
  const uint32_t vcode = max(q8_code<DT>(all_waves(1)), vold);
  if (tid == 0) {
    ks[sat] = (uint8_t)kcode;
    vs[sat] = (uint8_t)vcode;
  }
  const float kinv = q8_pow(254 - (int)kcode), vinv = q8_pow(254 - (int)vcode);
  const float kdown = q8_pow(max(127 + (int)kold - (int)kcode, 0));
  const float vdown = q8_pow(max(127 + (int)vold - (int)vcode, 0));

  auto keep = [&](int row, uint2 v) {  // a row's bytes into LDS
    uint32_t* p = s_k + (row * kPitch + kc) / 4;
    p[0] = v.x;
    p[1] = v.y;
  };
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (krow + 16 * j >= r1) continue;
    uint2 v;
    if (knew(j)) {
      v = q8_pack8<DT>(kx[j], kinv);
    } else {
      v = ko[j];
      if (kcode > kold) v = make_uint2(q8_rescale(v.x, kdown), q8_rescale(v.y, kdown));
    }
    if (knew(j) || kcode > kold) *reinterpret_cast<uint2*>(kp + 16 * kDim * j) = v;
    if (windows) keep(16 + krow + 16 * j, v);
  }

  const bool lower = vcode > vold && is_old != 0;
  const bool whole = r0 == 0 && r1 == kPage;
  if (is_new != 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = LsElem<DT>::to_f((uint16_t)(vx[j][e >> 1] >> (16 * (e & 1)))) * vinv;
      uint32_t v = q8_pack(f[0], f[1], f[2], f[3]);
      if (is_new != 0xffffffffu) {
        const uint32_t l = lower ? q8_rescale(vo[e], vdown) : vo[e];
        v = (v & is_new) | (l & is_old) | (vo[e] & ~(is_new | is_old));
      }
      if (whole)
        s_v[(8 * oct + e) * (kVPitch / 4) + quad] = v;
      else
        *reinterpret_cast<uint32_t*>(vp + e * kPage) = v;
    }
  }
  if (lower && is_new == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vo[e] = *reinterpret_cast<const uint32_t*>(vp + e * kPage);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<uint32_t*>(vp + e * kPage) = (q8_rescale(vo[e], vdown) & is_old) | (vo[e] & ~is_old);
  }
  if (complete(4)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) ntop = q8_abs_max<DT>(nx[j], ntop);
    ntop = ls_wave_max_u32(ntop);
    if (lane == 0) s_top[2][w] = ntop;
  }
  if (whole || complete(4)) __syncthreads();
  if (whole) {  // through LDS, so that a wave writes whole lines
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = 256 * i + tid, c = u >> 2;
      const uint32_t* p = s_v + c * (kVPitch / 4) + 4 * (u & 3);
      *reinterpret_cast<ls_u32x4*>(v8 + at + 16 * u) = ls_u32x4{p[0], p[1], p[2], p[3]};
    }
  }

  if (!windows) return;
  const uint32_t ncode = q8_code<DT>(all_waves(2));
  uint32_t pcode = 1;
  if (complete(0)) {
    pcode = ks[sat - G];
    keep(krow, *reinterpret_cast<const uint2*>(kp - (int64_t)G * kPageBytes + 48 * kDim));
  }
  if (complete(4)) keep(80 + krow, q8_pack8<DT>(nx[0], q8_pow(254 - (int)ncode)));
  __syncthreads();
  // Halves in float32 in token order, four channels a thread (a half that no window needs
  // may be anything).
  if (tid < 6 * 32) {
    const int half = tid >> 5, c = tid & 31;
    const uint32_t* p = s_k + half * 16 * (kPitch / 4) + c;
    ls_f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t x = p[r * (kPitch / 4)];
      const Q8F2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false);
      const Q8F2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
      a += ls_f32x4{lo[0], lo[1], hi[0], hi[1]};
    }
    s_half[half][c] = a * q8_pow((int)(half == 0 ? pcode : half == 5 ? ncode : kcode));
  }
  __syncthreads();
  const int i = tid >> 5, c = tid & 31;
  const int64_t win = 4 * page - 1 + i;
  if (i < 5 && complete(i) && win < kc_rows) {
    const ls_f32x4 a = (s_half[i][c] + s_half[i + 1][c]) * (1.f / 32.f);
    *reinterpret_cast<uint2*>(kcc + (int64_t)b * kbs + win * krs + (int64_t)g * kDim + 4 * c) =
        make_uint2(ls_pack2(LsElem<DT>::from_f(a[0]), LsElem<DT>::from_f(a[1])),
                   ls_pack2(LsElem<DT>::from_f(a[2]), LsElem<DT>::from_f(a[3])));
  }
}

// ---------------------------------------------------------------------------
// Attention of decode rows.  Workgroup (slice s, row t, KV head g): NW waves, each a
// share of the row's pages with a running maximum and sum, joined through LDS; with
// several slices, partial results go to the workspace and a second kernel joins them.
// Row i of sequence b sees keys j < len_b, or j <= len_b - len_q(b) + i (causal).
// K's bytes become the query's type (exact) for S^T = K Q^T, V's become fp16 (exact) for
// O^T = V^T P^T with 2^15 P <= 2^15 as an fp16 head and an fp16 remainder, a product of each: 22
// bits of a weight, 2^-40 of the largest where the head or the remainder is subnormal.  (The
// head alone holds 11: its error, 2^-11 of a weight, passes a bf16 output's own rounding where
// values nearly cancel.  Unscaled, weights below 2^-25 of the largest would vanish, and a row of
// 100000 of them with it.)
// A page's powers of two go into the scores' scale and into the sum of O.
//
// A wave takes ppw plan slots, or (DENSE) pages, or more of a row that is longer than the
// caller said; a row's later slices, past its last page, only say that they hold nothing.
// The next page's K and V are loaded as soon as this page's have been used, into the same
// registers.
//
// What bounds it: a compute unit's reads from memory.  Operands read in their own order (lanes
// 16 apart on neighbouring bytes) reach 50 GB/s a unit however many waves read; 1 KB a load in
// the lanes' order (kStage), brought into the operands' order through LDS, 63 GB/s with eight
// waves (131071 keys, one slice, the weights' heads alone: 671 us, 538 us; with their remainders,
// which are in a lone row's chain, 618), but with four waves, alone on their SIMDs, the way
// through LDS is in the page's chain (two slices of 256 pages: 50 us, 54 us).  So rows of one
// slice, which need their unit's rate, take eight waves and kStage; slices take neither.
// 131071 keys in 128 slices: 19.0 us with the join (67 MB, 3.5 TB/s; a launch, the chain of
// lengths, page and sum, and the join are 9 us of it); 16 rows of 64 pages in eight slices:
// 14.2 us (34 MB, 2.4 TB/s); 72 rows of 4000 keys, one slice: 36 us (150 MB, 4.1 TB/s).
// ---------------------------------------------------------------------------
#define LS_Q8_MAX_SPLITS 256
constexpr int kSplitWaves = 4, kWholeWaves = 8;  // of a workgroup: one of several slices, or the row
#define LS_Q8_PITCH 132             // floats per head of a wave's O in LDS
#define LS_Q8_ID_REGS 4             // plan ids held in registers: topk <= 256

// Workspace: O float [G][total_q][n_splits][gs][128], then (m, l) float2 [G][total_q][gs][n_splits].
struct Q8Part {
  float* o;
  float2* ml;
};

// The decode row: its sequence, and the keys j < limit it sees (<= 0: none).
struct Q8Row {
  int b;
  int64_t limit;
};

// Row t of the batch, b = -1 behind the last sequence.  A batch of at most 64 is read by the
// lanes at once.
__device__ __forceinline__ Q8Row q8_row(const int32_t* __restrict__ cu_q,
                                        const int32_t* __restrict__ lens, int batch, int64_t t,
                                        int64_t capacity, int causal) {
  Q8Row r;
  int b, c0, c1, len;
  if (batch <= 64) {
    const int i = min(ls_lane(), batch - 1);
    const int lo = cu_q[i], hi = cu_q[i + 1], n = lens[i];
    b = __popcll(__ballot(ls_lane() < batch && t >= hi));  // sequences that end at or before t
    if (b >= batch) return Q8Row{-1, 0};
    c0 = __builtin_amdgcn_readlane(lo, b);
    c1 = __builtin_amdgcn_readlane(hi, b);
    len = __builtin_amdgcn_readlane(n, b);
  } else {
    if (t >= cu_q[batch]) return Q8Row{-1, 0};
    b = ls_find_segment(cu_q, batch, t);
    c0 = cu_q[b];
    c1 = cu_q[b + 1];
    len = lens[b];
  }
  r.b = b;
  const int64_t held = min((int64_t)len, capacity);
  r.limit = causal ? held - (c1 - c0) + (t - c0) + 1 : held;
  return r;
}

// Pages a wave takes of a dense row, at least ppw and enough for n_splits slices of NW waves,
// and the slices that the row's pages then fill.
struct Q8Share {
  int pages, share, slices;
};
template <int NW>
__device__ __forceinline__ Q8Share q8_share(int64_t limit, int ppw, int n_splits) {
  Q8Share x;
  x.pages = limit <= 0 ? 0 : (int)((limit + kPage - 1) / kPage);
  x.share = max(ppw, (x.pages + NW * n_splits - 1) / (NW * n_splits));
  x.slices = (x.pages + NW * x.share - 1) / (NW * x.share);
  return x;
}

// Orders a wave's accesses to LDS among its lanes (its instructions reach LDS in order: no wait).
__device__ __forceinline__ void q8_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Eight e4m3 bytes as eight values of the query's type.
template <int DT>
__device__ __forceinline__ ls_u32x4 q8_expand(uint32_t lo, uint32_t hi) {
  ls_u32x4 o;
  if constexpr (DT == LS_BF16) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  } else {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
  }
  return o;
}

// Arguments of the attention and of the join.
struct Q8AttnArgs {
  const uint16_t* q;
  int64_t qrs;
  const int32_t* cu_q;
  int batch;
  int64_t total_q;
  const uint8_t* k8;
  const uint8_t* v8;
  int64_t cbs;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t sbs;
  int64_t pages;
  const int32_t* cache_seqlens;
  int gs;
  const int32_t* topk_idx;
  int topk;
  int ppw;
  int n_splits;
  float scale_log2;
  int causal;
  Q8Part part;
  uint16_t* out;
  float* lse;
};

template <int DT, bool DENSE, int NW>
__global__ __launch_bounds__(64 * NW) void ls_q8_attn_kernel(const Q8AttnArgs args) {
  const uint16_t* __restrict__ q = args.q;
  const int64_t qrs = args.qrs;
  const int32_t* __restrict__ cu_q = args.cu_q;
  const int batch = args.batch;
  const int64_t total_q = args.total_q;
  const uint8_t* __restrict__ k8 = args.k8;
  const uint8_t* __restrict__ v8 = args.v8;
  const int64_t cbs = args.cbs;
  const uint8_t* __restrict__ ks = args.ks;
  const uint8_t* __restrict__ vs = args.vs;
  const int64_t sbs = args.sbs;
  const int64_t pages = args.pages;
  const int32_t* __restrict__ cache_seqlens = args.cache_seqlens;
  const int gs = args.gs;
  const int32_t* __restrict__ topk_idx = args.topk_idx;
  const int topk = args.topk;
  const int ppw = args.ppw;
  const int n_splits = args.n_splits;
  const float scale_log2 = args.scale_log2;
  const int causal = args.causal;
  const Q8Part part = args.part;
  uint16_t* __restrict__ out = args.out;
  float* __restrict__ lse = args.lse;
  // Each wave's O at its end; before, where kStage, a page's K and V in turn.
  __shared__ __attribute__((aligned(16))) float s_o[NW][16 * LS_Q8_PITCH];
  __shared__ float s_ml[NW][2][16];
  constexpr bool kStage = NW == kWholeWaves;
  static_assert(kPageBytes <= (int)sizeof(s_o[0]), "a page fits where a wave's O lies");
  const int64_t t = blockIdx.x / (unsigned)n_splits;
  const int s = (int)(blockIdx.x - (unsigned)t * (unsigned)n_splits);
  const int g = blockIdx.y, G = gridDim.y;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, qg = lane >> 4;
  // The row's plan ids, 64 per register.  (A vector: an array indexed in the lambda below
  // would be kept in LDS.)
  typedef int IdRegs __attribute__((ext_vector_type(LS_Q8_ID_REGS)));
  IdRegs idr = -1;
  if constexpr (!DENSE) {
    const int32_t* idrow = topk_idx + ((int64_t)g * total_q + t) * topk;
#pragma unroll
    for (int k = 0; k < LS_Q8_ID_REGS; ++k)
      if (64 * k + lane < topk) idr[k] = idrow[64 * k + lane];
  }
  // Queries: step k4 of the product takes channels 32 qg + 8 k4 + [0, 8), as K's loads do.
  ls_u32x4 qf[4];
  const uint16_t* qrow = q + t * qrs + ((int64_t)g * gs + r) * kDim + 32 * qg;
#pragma unroll
  for (int k4 = 0; k4 < 4; ++k4)
    qf[k4] = r < gs ? ls_load16(qrow + 8 * k4) : ls_u32x4{0u, 0u, 0u, 0u};
  const Q8Row row = q8_row(cu_q, cache_seqlens, batch, t, pages * kPage, causal);
  if (row.b < 0) return;
  const int64_t limit = row.limit;
  Q8Share cut = {topk, ppw, n_splits};
  if constexpr (DENSE) {
    cut = q8_share<NW>(limit, ppw, n_splits);
    if (s > 0 && s >= cut.slices) {  // nothing left for this slice
      if (tid < gs) part.ml[(((int64_t)g * total_q + t) * gs + tid) * n_splits + s] = make_float2(-INFINITY, 0.f);
      return;
    }
  }
  const uint8_t* kseq = k8 + (int64_t)row.b * cbs + (int64_t)g * kPageBytes;
  const uint8_t* vseq = v8 + (int64_t)row.b * cbs + (int64_t)g * kPageBytes;
  const uint8_t* kss = ks + (int64_t)row.b * sbs + g;
  const uint8_t* vss = vs + (int64_t)row.b * sbs + g;

  int slot = (NW * s + w) * cut.share;  // the wave's next plan slot (DENSE: page) and its end
  const int slot1 = min(cut.pages, slot + cut.share);
  // The page of the next valid slot (-1 at the end of the share).
  auto next_page = [&]() -> int {
    int found = -1;
    while (found < 0 && slot < slot1) {
      const int at = slot++;
      if constexpr (DENSE) {
        found = at;
      } else {
        const int held = at < 128 ? (at < 64 ? idr[0] : idr[1]) : (at < 192 ? idr[2] : idr[3]);
        const int id = __builtin_amdgcn_readlane(held, at & 63);
        if (id < 0 || (int64_t)kPage * id >= limit) continue;  // limit <= pages * 64
        bool dup = false;  // a repeated id counts once, as a bitmask of pages would have it
#pragma unroll
        for (int k = 0; k < LS_Q8_ID_REGS; ++k)
          dup |= __ballot(64 * k + lane < at && idr[k] == id) != 0ull;
        if (!dup) found = id;
      }
    }
    return found;
  };

  float m_run = -INFINITY, l_run = 0.f;
  ls_f32x4 o[8];
#pragma unroll
  for (int db = 0; db < 8; ++db) o[db] = ls_f32x4{0.f, 0.f, 0.f, 0.f};
  ls_u32x4 kl[8], vl[8];
  uint32_t kcode, vcode;
  auto load_k = [&](int page) {
    const uint8_t* kp = kseq + (int64_t)page * G * kPageBytes;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      kl[j] = ls_load16(kp + (kStage ? 1024 * j + 16 * lane
                                     : (16 * (j >> 1) + r) * kDim + 32 * qg + 16 * (j & 1)));
    kcode = kss[(int64_t)page * G];
  };
  auto load_v = [&](int page) {
    const uint8_t* vp = vseq + (int64_t)page * G * kPageBytes;
#pragma unroll
    for (int j = 0; j < 8; ++j) vl[j] = ls_load16(vp + 1024 * j + (kStage ? 16 * lane : r * kPage + 16 * qg));
    vcode = vss[(int64_t)page * G];
  };
  // Piece p of 16 bytes of 128-byte line n lies at 8 n + (p ^ (n & 7)): both the writes (a line
  // for eight lanes) and the reads (a piece of eight lines) then touch every bank once.
  ls_u32x4* stage = reinterpret_cast<ls_u32x4*>(s_o[w]);
  const int put_at = (lane & 56) | ((lane ^ (lane >> 3)) & 7);
  auto put = [&](const ls_u32x4 (&x)[8]) {
    q8_wave_sync();
#pragma unroll
    for (int j = 0; j < 8; ++j) stage[64 * j + put_at] = x[j];
    q8_wave_sync();
  };
  // K: key r of 16, channels 32 qg + 16 h + [0, 16).  V: channel r of 16, the qg-th 16 bytes.
  int k_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) k_at[h] = 8 * r + ((2 * qg + h) ^ (r & 7));
  const int v_at = 8 * (r >> 1) + ((4 * (r & 1) + qg) ^ (r >> 1));
  // One page whose K and V are in registers (or on their way), with the loads of the page
  // after it.  The last page is its own copy of this code, so that the loads are on every
  // path of the loop (a conditional load would be waited for where the paths meet).
  auto attend = [&](int page, int after, auto more) {
    constexpr bool kMore = decltype(more)::value;
    const int64_t left = limit - (int64_t)kPage * page;
    const int nvis = left < kPage ? (int)left : kPage;
    const float kscale = scale_log2 * q8_pow(kcode);
    float sv[16], pm = -INFINITY;
    if constexpr (kStage) {
      put(kl);
      if constexpr (kMore) load_k(after);
    }
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      ls_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ls_u32x4 kk;
        if constexpr (kStage)
          kk = stage[128 * kb + k_at[h]];
        else
          kk = kl[2 * kb + h];
        acc = LsElem<DT>::mfma(q8_expand<DT>(kk[0], kk[1]), qf[2 * h], acc);
        acc = LsElem<DT>::mfma(q8_expand<DT>(kk[2], kk[3]), qf[2 * h + 1], acc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[4 * kb + i] = acc[i] * kscale;
    }
    if constexpr (!kStage && kMore) load_k(after);
    const bool part_page = nvis < kPage;  // keys past the end have no weight, and may be anything
    if (part_page) {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * kb + 4 * qg + i >= nvis) sv[4 * kb + i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) pm = fmaxf(pm, sv[i]);
    pm = fmaxf(pm, ls_shfl_xor(pm, 16));
    pm = fmaxf(pm, ls_shfl_xor(pm, 32));
    const float m_new = fmaxf(m_run, pm);
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    float sum = 0.f;  // of the page alone first: small weights would be lost beside a large sum
    ls_u32x4 ph[2], pl[2];  // heads and remainders of the weights
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(sv[8 * c + 2 * e] - m_new);
        const float p1 = __builtin_amdgcn_exp2f(sv[8 * c + 2 * e + 1] - m_new);
        sum += p0 + p1;
        const float u0 = p0 * 0x1p15f, u1 = p1 * 0x1p15f;
        const uint16_t h0 = ls_f32_to_f16(u0), h1 = ls_f32_to_f16(u1);
        ph[c][e] = ls_pack2(h0, h1);
        pl[c][e] = ls_pack2(ls_f32_to_f16(u0 - ls_f16_to_f32(h0)), ls_f32_to_f16(u1 - ls_f16_to_f32(h1)));
      }
    l_run = l_run * alpha + sum;
    auto weigh = [&](ls_u32x4 (&vf)[8], uint32_t code) {
      if (part_page) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const int n = min(4, max(0, nvis - 16 * kb - 4 * qg));
          const uint32_t keep = n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
#pragma unroll
          for (int db = 0; db < 8; ++db) vf[db][kb] &= keep;
        }
      }
      const float vscale = q8_pow(code) * 0x1p-15f;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const ls_u32x4 v0 = q8_expand<LS_F16>(vf[db][0], vf[db][1]);
        const ls_u32x4 v1 = q8_expand<LS_F16>(vf[db][2], vf[db][3]);
        ls_f32x4 pv = {0.f, 0.f, 0.f, 0.f};
        pv = LsElem<LS_F16>::mfma(v0, ph[0], pv);
        pv = LsElem<LS_F16>::mfma(v1, ph[1], pv);
        pv = LsElem<LS_F16>::mfma(v0, pl[0], pv);
        pv = LsElem<LS_F16>::mfma(v1, pl[1], pv);
        o[db] = o[db] * alpha + pv * vscale;
      }
    };
    if constexpr (kStage) {
      put(vl);
      const uint32_t code = vcode;
      if constexpr (kMore) load_v(after);
      ls_u32x4 vf[8];
#pragma unroll
      for (int db = 0; db < 8; ++db) vf[db] = stage[64 * db + v_at];
      weigh(vf, code);
    } else {
      weigh(vl, vcode);
      if constexpr (kMore) load_v(after);
    }
  };
  int page = next_page();
  if (page >= 0) {
    load_k(page);
    load_v(page);
    for (;;) {
      const int after = next_page();
      if (after < 0) break;
      attend(page, after, std::true_type());
      page = after;
    }
    attend(page, -1, std::false_type());
  }
  l_run += ls_shfl_xor(l_run, 16);
  l_run += ls_shfl_xor(l_run, 32);
  q8_wave_sync();
#pragma unroll
  for (int db = 0; db < 8; ++db)  // o[db][i]: head r, channel 16 db + 4 qg + i
    *reinterpret_cast<ls_f32x4*>(&s_o[w][r * LS_Q8_PITCH + 16 * db + 4 * qg]) = o[db];
  if (qg == 0) {
    s_ml[w][0][r] = m_run;
    s_ml[w][1][r] = l_run;
  }
  __syncthreads();
  // Join the waves, a few channels of a head a thread.  A wave without a page has sum 0 and
  // is left out; one whose sum is NaN is not.
  constexpr int kCh = 16 * kDim / (64 * NW);  // channels a thread: 8 or 4
  const int h = tid / (kDim / kCh), d = kCh * (tid % (kDim / kCh));
  if (h >= gs) return;
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) M = fmaxf(M, s_ml[i][0][h]);
  ls_f32x4 a[kCh / 4];
#pragma unroll
  for (int e = 0; e < kCh / 4; ++e) a[e] = ls_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const float l = s_ml[i][1][h];
    const float wt = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(s_ml[i][0][h] - M);
#pragma unroll
    for (int e = 0; e < kCh / 4; ++e)
      a[e] += wt * *reinterpret_cast<const ls_f32x4*>(&s_o[i][h * LS_Q8_PITCH + d + 4 * e]);
    L += wt * l;
  }
  const int64_t tg = (int64_t)g * total_q + t;
  if (n_splits == 1) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint16_t* po = out + ((t * G + g) * (int64_t)gs + h) * kDim + d;
#pragma unroll
    for (int e = 0; e < kCh / 4; ++e)
      *reinterpret_cast<uint2*>(po + 4 * e) =
          make_uint2(ls_pack2(LsElem<DT>::from_f(a[e][0] * inv), LsElem<DT>::from_f(a[e][1] * inv)),
                     ls_pack2(LsElem<DT>::from_f(a[e][2] * inv), LsElem<DT>::from_f(a[e][3] * inv)));
    if (lse && d == 0)
      lse[((int64_t)g * gs + h) * total_q + t] =
          L == 0.f ? INFINITY : (M + __log2f(L)) * 0.69314718055994531f;
  } else {
    float* po = part.o + ((tg * n_splits + s) * gs + h) * kDim + d;
#pragma unroll
    for (int e = 0; e < kCh / 4; ++e) *reinterpret_cast<ls_f32x4*>(po + 4 * e) = a[e];
    if (d == 0) part.ml[(tg * gs + h) * n_splits + s] = make_float2(M, L);
  }
}

// out[t][g*gs + h] = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s; a row that sees no key gives
// zeros and lse = +inf.  A workgroup per (row, KV head, query head): each wave forms the maximum
// and sum of all slices (at most four a lane), then thread (p, c) sums four channels of every
// P-th slice, and the P parts are added in LDS in order.  The first 8 P slices' values are
// loaded with the maxima (a slice of sum 0 may hold anything and is left out); with P = 8 there
// are no more.  Bound by its launch
// and the reads of its chain: 3.5 us for 16 slices of a row; P = 8 up to 64 slices, 16 above (131071
// keys in 128 slices, with the attention: 19.0 us, and 19.5 with P = 8).
template <int DT, int P>
__global__ __launch_bounds__(32 * P) void ls_q8_join_kernel(const Q8AttnArgs args) {
  const Q8Part part = args.part;
  const int64_t total_q = args.total_q;
  const int gs = args.gs, n = args.n_splits;
  constexpr int kAhead = 8;
  constexpr int kMost = P == 8 ? 64 : LS_Q8_MAX_SPLITS;  // slices
  __shared__ float s_w[kMost];
  __shared__ ls_f32x4 s_a[P][32];
  const int64_t t = blockIdx.x;
  const int g = blockIdx.y, h = blockIdx.z, G = gridDim.y;
  const int tid = threadIdx.x, lane = tid & 63;
  const int c = tid & 31, p = tid >> 5;
  const int64_t tg = (int64_t)g * total_q + t;
  const float2* __restrict__ ml = part.ml + (tg * gs + h) * n;
  const float* __restrict__ po = part.o + (tg * n * gs + h) * kDim + 4 * c;
  float ms[kMost / 64], sum[kMost / 64], M = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMost / 64; ++k) {
    const int i = 64 * k + lane;
    const float2 x = i < n ? ml[i] : make_float2(-INFINITY, 0.f);
    ms[k] = x.x;
    sum[k] = x.y;
  }
  ls_f32x4 ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    ahead[k] = *reinterpret_cast<const ls_f32x4*>(po + (int64_t)min(p + P * k, n - 1) * gs * kDim);
  if (t >= args.cu_q[args.batch]) return;  // a row behind the last sequence
#pragma unroll
  for (int k = 0; k < kMost / 64; ++k) M = fmaxf(M, ms[k]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, ls_shfl_xor(M, o));
  float L = 0.f;
#pragma unroll
  for (int k = 0; k < kMost / 64; ++k) {
    ms[k] = sum[k] == 0.f ? 0.f : __builtin_amdgcn_exp2f(ms[k] - M);
    L += ms[k] * sum[k];
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) L += ls_shfl_xor(L, o);
  if (tid < 64) {
#pragma unroll
    for (int k = 0; k < kMost / 64; ++k)
      if (64 * k + lane < n) s_w[64 * k + lane] = ms[k];
  }
  __syncthreads();
  ls_f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const float wt = p + P * k < n ? s_w[p + P * k] : 0.f;
    if (wt != 0.f) a += wt * ahead[k];
  }
  if constexpr (P * kAhead < kMost) {
    const int s0 = p + P * kAhead;
    static_assert(2 * P * kAhead == kMost, "one more round");
    if (s0 < n) {
      ls_f32x4 x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        x[k] = *reinterpret_cast<const ls_f32x4*>(po + (int64_t)min(s0 + P * k, n - 1) * gs * kDim);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float wt = s0 + P * k < n ? s_w[s0 + P * k] : 0.f;
        if (wt != 0.f) a += wt * x[k];
      }
    }
  }
  s_a[p][c] = a;
  __syncthreads();
  if (tid < 32) {
    a = s_a[0][c];
#pragma unroll
    for (int i = 1; i < P; ++i) a += s_a[i][c];
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint2 x;
    x.x = ls_pack2(LsElem<DT>::from_f(a[0] * inv), LsElem<DT>::from_f(a[1] * inv));
    x.y = ls_pack2(LsElem<DT>::from_f(a[2] * inv), LsElem<DT>::from_f(a[3] * inv));
    *reinterpret_cast<uint2*>(args.out + ((t * G + g) * (int64_t)gs + h) * kDim + 4 * c) = x;
    if (args.lse && tid == 0)
      args.lse[((int64_t)g * gs + h) * total_q + t] =
          L == 0.f ? INFINITY : (M + __log2f(L)) * 0.69314718055994531f;
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {
constexpr int64_t kMaxThreads = 0xffffffffLL;  // of a launch along a dimension
}  // namespace

extern "C" int ls_kvcache_append_q8(void* k8, void* v8, int64_t cache_batch_stride,
                                    uint8_t* k_scale, uint8_t* v_scale,
                                    int64_t scale_batch_stride, int64_t pages,
                                    const int32_t* cache_seqlens, const void* k_new,
                                    const void* v_new, int64_t new_row_stride,
                                    const int32_t* cu_seqlens_new, int64_t total_new,
                                    int32_t batch, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t dtype, void* kc_cache, int64_t kc_batch_stride,
                                    int64_t kc_row_stride, int64_t kc_rows, void* stream) {
  const char* who = "ls_kvcache_append_q8";
  LS_REQUIRE(batch >= 0 && total_new >= 0 && num_kv_heads > 0 && pages >= 0 && kc_rows >= 0,
             LS_ERR_INVALID, "%s: bad sizes", who);
  LS_REQUIRE(head_dim == kDim, LS_ERR_UNSUPPORTED, "%s: head_dim must be 128", who);
  LS_REQUIRE(dtype == LS_BF16 || dtype == LS_F16, LS_ERR_UNSUPPORTED,
             "%s: new keys and values are bf16 or fp16", who);
  LS_REQUIRE(num_kv_heads <= 65535, LS_ERR_INVALID, "%s: too many heads", who);
  LS_REQUIRE(new_row_stride % 8 == 0 && cache_batch_stride % 16 == 0, LS_ERR_UNSUPPORTED,
             "%s: rows must be 16-byte aligned", who);
  if (total_new == 0 || batch == 0) return LS_OK;
  LS_REQUIRE(k8 && v8 && k_scale && v_scale && k_new && v_new && cache_seqlens && cu_seqlens_new,
             LS_ERR_INVALID, "%s: null pointer", who);
  LS_REQUIRE(ls_aligned16(k8) && ls_aligned16(v8) && ls_aligned16(k_new) && ls_aligned16(v_new),
             LS_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned", who);
  // A sequence's n > 0 new tokens touch at most (n + 126) / 64 <= n pages.
  const int64_t nb = std::min<int64_t>(batch, total_new);
  const int64_t units = std::min(total_new, (total_new + 126 * nb) / 64);
  LS_REQUIRE(units * 256 <= kMaxThreads, LS_ERR_UNSUPPORTED, "%s: too many new tokens", who);
  LS_REQUIRE(!kc_cache || (ls_aligned16(kc_cache) && kc_row_stride % 8 == 0 && kc_batch_stride % 8 == 0),
             LS_ERR_UNSUPPORTED, "%s: compressed cache must be 16-byte aligned", who);
  const Q8AppendArgs args = {
      (uint8_t*)k8,        (uint8_t*)v8,     cache_batch_stride, k_scale,   v_scale,
      scale_batch_stride,  pages,            cache_seqlens,      (const uint16_t*)k_new,
      (const uint16_t*)v_new, new_row_stride, cu_seqlens_new,    total_new, batch,
      num_kv_heads,        (uint16_t*)kc_cache, kc_batch_stride, kc_row_stride, kc_rows};
  auto append = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)units, num_kv_heads), dim3(256), 0,
                       (hipStream_t)stream, args);
    return ls_check_launch("ls_q8_append_kernel");
  };
  return dtype == LS_BF16 ? append(ls_q8_append_kernel<LS_BF16>)
                          : append(ls_q8_append_kernel<LS_F16>);
}

extern "C" size_t ls_attn_kvcache_q8_workspace_size(int64_t total_q, int32_t num_heads,
                                                    int32_t n_splits) {
  if (n_splits <= 1 || total_q <= 0 || num_heads <= 0) return 0;
  return 4 * (size_t)total_q * num_heads * n_splits * (kDim + 2);
}

extern "C" int ls_attn_kvcache_q8(const void* q, int64_t q_row_stride, const int32_t* cu_seqlens_q,
                                  int64_t total_q, const void* k8, const void* v8,
                                  int64_t cache_batch_stride, const uint8_t* k_scale,
                                  const uint8_t* v_scale, int64_t scale_batch_stride,
                                  int64_t pages, const int32_t* cache_seqlens, int32_t batch,
                                  int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                  int32_t dtype, const int32_t* topk_idx, int32_t n_pages,
                                  float softmax_scale, int32_t causal, int32_t n_splits, void* out,
                                  float* softmax_lse, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const char* who = "ls_attn_kvcache_q8";
  LS_REQUIRE(batch > 0 && total_q >= 0 && num_kv_heads > 0 && num_heads > 0 &&
                 num_heads % num_kv_heads == 0 && pages >= 0,
             LS_ERR_INVALID, "%s: bad sizes", who);
  const int gs = num_heads / num_kv_heads;
  LS_REQUIRE(head_dim == kDim && gs <= 16, LS_ERR_UNSUPPORTED,
             "%s: head_dim 128 and at most 16 query heads per KV head", who);
  LS_REQUIRE(dtype == LS_BF16 || dtype == LS_F16, LS_ERR_UNSUPPORTED,
             "%s: queries are bf16 or fp16", who);
  const bool dense = topk_idx == nullptr;
  LS_REQUIRE(n_pages >= 1 && n_splits >= 1 && n_splits <= LS_Q8_MAX_SPLITS, LS_ERR_INVALID,
             "%s: need n_pages >= 1 and 1 <= n_splits <= %d", who, LS_Q8_MAX_SPLITS);
  LS_REQUIRE(dense || n_pages <= 64 * LS_Q8_ID_REGS, LS_ERR_UNSUPPORTED,
             "%s: at most %d plan ids per row (got %d)", who, 64 * LS_Q8_ID_REGS, n_pages);
  LS_REQUIRE(total_q <= kMaxThreads / (512LL * n_splits) && num_kv_heads <= 65535, LS_ERR_UNSUPPORTED,
             "%s: too many rows or KV heads", who);
  LS_REQUIRE(pages <= 0x1000000, LS_ERR_UNSUPPORTED, "%s: at most 2^24 pages a sequence", who);
  LS_REQUIRE(q_row_stride % 8 == 0 && cache_batch_stride % 16 == 0, LS_ERR_UNSUPPORTED,
             "%s: rows must be 16-byte aligned", who);
  if (total_q == 0) return LS_OK;
  LS_REQUIRE(q && k8 && v8 && k_scale && v_scale && cu_seqlens_q && cache_seqlens && out,
             LS_ERR_INVALID, "%s: null pointer", who);
  LS_REQUIRE(ls_aligned16(q) && ls_aligned16(k8) && ls_aligned16(v8) && ls_aligned16(out) &&
                 ls_aligned16(workspace),
             LS_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned", who);
  // ppw plan slots or pages a wave; with every wave's share rounded up, fewer slices may do.
  const int waves = n_splits == 1 ? kWholeWaves : kSplitWaves;
  const int ppw = (int)((n_pages + (int64_t)waves * n_splits - 1) / (waves * n_splits));
  const int splits = (int)((n_pages + (int64_t)waves * ppw - 1) / (waves * ppw));
  const size_t need = ls_attn_kvcache_q8_workspace_size(total_q, num_heads, splits);
  LS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), LS_ERR_WORKSPACE,
             "%s: workspace %zu < %zu", who, workspace ? workspace_bytes : (size_t)0, need);
  hipStream_t s = (hipStream_t)stream;
  const float scale_log2 = softmax_scale * 1.4426950408889634f;
  Q8Part part;
  part.o = (float*)workspace;
  part.ml = (float2*)(part.o + (splits > 1 ? (size_t)total_q * num_heads * splits * kDim : 0));
  const Q8AttnArgs args = {
      (const uint16_t*)q, q_row_stride, cu_seqlens_q, batch, total_q, (const uint8_t*)k8,
      (const uint8_t*)v8, cache_batch_stride, k_scale, v_scale, scale_batch_stride, pages,
      cache_seqlens, gs, topk_idx, n_pages, ppw, splits, scale_log2, causal, part,
      (uint16_t*)out, softmax_lse};
  auto attend = [&](auto dt, auto dn, auto nw) {
    constexpr int NW = decltype(nw)::value;
    hipLaunchKernelGGL((ls_q8_attn_kernel<decltype(dt)::value, decltype(dn)::value, NW>),
                       dim3((unsigned)(total_q * splits), num_kv_heads), dim3(64 * NW), 0, s, args);
    return ls_check_launch("ls_q8_attn_kernel");
  };
  auto by_waves = [&](auto dt, auto dn) {
    return n_splits == 1 ? attend(dt, dn, std::integral_constant<int, kWholeWaves>())
                         : attend(dt, dn, std::integral_constant<int, kSplitWaves>());
  };
  auto by_plan = [&](auto dt) {
    return dense ? by_waves(dt, std::true_type()) : by_waves(dt, std::false_type());
  };
  const int rc = dtype == LS_BF16 ? by_plan(std::integral_constant<int, LS_BF16>())
                                  : by_plan(std::integral_constant<int, LS_F16>());
  if (rc || splits == 1) return rc;
  auto join = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)total_q, num_kv_heads, gs), dim3(threads), 0, s, args);
    return ls_check_launch("ls_q8_join_kernel");
  };
  if (splits > 64)
    return dtype == LS_BF16 ? join(ls_q8_join_kernel<LS_BF16, 16>, 512)
                            : join(ls_q8_join_kernel<LS_F16, 16>, 512);
  return dtype == LS_BF16 ? join(ls_q8_join_kernel<LS_BF16, 8>, 256)
                          : join(ls_q8_join_kernel<LS_F16, 8>, 256);
}
