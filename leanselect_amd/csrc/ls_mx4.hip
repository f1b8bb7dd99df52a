// Products of a few rows with 4-bit weights (E2M1 values, an E8M0 scale per 32 inputs).
//
//   out[m][n] = sum_k x[m][k] * e2m1(codes[n][k]) * 2^(scales[n][k / 32] - 127)
//
// Layout (laid out once): tiles of 16 outputs by 128 inputs, zero-padded,
//   codes  [ceil(N/16)][ceil(K/128)][64 lanes][16 bytes]   lane 16 q + r: output r of the
//          tile, inputs 32 q .. 32 q + 31, the even input in a byte's low half
//   scales [ceil(N/16)][ceil(K/512)][64 lanes][4 bytes]    the same lanes, byte i: the i-th of
//          four tiles; codes c in [8, 252], 2^(c - 127)
// A lane's 16 bytes are one scale group, and the four 8-input pieces of it are its left
// operands of four 16x16x32 matrix instructions (the instruction's 32 inputs then are piece s
// of each of the four groups; the rows of x are read in the same order).  So a wave takes a
// tile from memory with one 16-byte load a lane, and each pair of weights becomes two exact
// 16-bit values, scale included, in one conversion.
//
// No counterpart in the reference, whose projections are 16-bit (leanselect/models/
// minicpm.py:2176-2222, 1098-1135, 3987-4090).
#include <algorithm>
#include <type_traits>

#include "ls_common.h"

namespace {

// Four bytes (inputs 8 s .. 8 s + 7) as eight values times the scale.
template <int DT>
__device__ __forceinline__ ls_u32x4 mx4_expand(uint32_t v, float scale) {
  ls_u32x4 o;
  if constexpr (DT == LS_BF16) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, scale, 0));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, scale, 1));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, scale, 2));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, scale, 3));
  } else {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, scale, 0));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, scale, 1));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, scale, 2));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, scale, 3));
  }
  return o;
}

// Outputs col .. col + 3 of a row, as far as there are so many.
template <int DT>
__device__ __forceinline__ void mx4_store(ls_f32x4 y, uint16_t* row, int64_t col, int64_t n_out) {
  uint16_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = LsElem<DT>::from_f(y[i]);
  uint16_t* o = row + col;
  if (col + 4 <= n_out && ((uintptr_t)o & 7) == 0) {
    *reinterpret_cast<uint2*>(o) = make_uint2(ls_pack2(h[0], h[1]), ls_pack2(h[2], h[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < n_out) o[i] = h[i];
  }
}

__device__ __forceinline__ ls_f32x4 mx4_silu_mul(ls_f32x4 gate, ls_f32x4 up) {
#pragma unroll
  for (int i = 0; i < 4; ++i) gate[i] = gate[i] / (1.f + __expf(-gate[i])) * up[i];
  return gate;
}

// Four registers a lane, [piece][quarter of the wave] -> [quarter][piece]: what lane (r, q) holds
// as piece p goes to lane (r, p) as piece q.
__device__ __forceinline__ void mx4_transpose(ls_u32x4 (&x)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // Halves of the wave, pieces two apart; then odd and even quarters, pieces one apart.
    const auto a = __builtin_amdgcn_permlane32_swap(x[0][e], x[2][e], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(x[1][e], x[3][e], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    x[0][e] = c[0];
    x[1][e] = c[1];
    x[2][e] = d[0];
    x[3][e] = d[1];
  }
}

// Arguments of both products (one: a launch with many costs the host more).
struct Mx4Args {
  const uint16_t* x;
  int64_t xrs;
  int64_t m;
  int64_t K;
  const uint8_t* codes;
  const uint32_t* scales;
  int64_t kc;
  int64_t kc4;
  int64_t tiles;
  int64_t per_half;
  int64_t n_out;
  uint16_t* out;
  int64_t ors;
  float* part;
};

// Workgroup (RT tiles of 16 outputs, block of 16 MT rows of x): NW waves share the inputs, four
// tiles (512 inputs) at a time, and are summed through LDS in order, so a row's bits depend
// on neither MT nor RT.  PAIR: half of the tiles are `pair` tiles later, the up projections of
// the same outputs, and silu(gate) * up is written (float32 up to the one rounding).
//
// x is read as it lies, a load's lanes (r, p) taking 16 bytes each of 64 contiguous ones of row
// r: the operands' own order (64 bytes apart) would touch a cache line per lane, which bounded
// the kernel at 1.8 TB/s of weights at 16 rows.  Four registers' exchange between the
// quarters of the wave brings the pieces where the weights' order wants them.
// A wave's next weights are loaded into the registers of each tile that it has used.
//
// Bound by the weights' bytes where there are many tiles (73448 x 4096, 16 rows: 38.9 us in eager
// passes, 160 MB at 4.1 TB/s; one row 33.2, 35.5 with conditional loads of x), by a launch and one chain of load, product, LDS and
// store where there are few (4608 x 4096, one row: 5.9 us, 10 MB).
template <int DT, int MT, int RT, bool PAIR, int NW>
__global__ __launch_bounds__(64 * NW) void ls_mx4_kernel(const Mx4Args args) {
  const uint16_t* __restrict__ x = args.x;
  const int64_t xrs = args.xrs;
  const int64_t m = args.m;
  const int64_t K = args.K;
  const uint8_t* __restrict__ codes = args.codes;
  const uint32_t* __restrict__ scales = args.scales;
  const int64_t kc = args.kc;
  const int64_t kc4 = args.kc4;
  const int64_t tiles = args.tiles;
  const int64_t n_out = args.n_out;
  uint16_t* __restrict__ out = args.out;
  const int64_t ors = args.ors;
  constexpr int OT = PAIR ? RT / 2 : RT;  // tiles of outputs
  __shared__ __attribute__((aligned(16))) ls_f32x4 s_acc[NW][RT * MT][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  // Tile a of the workgroup; past the last one, the last again (not written).
  int64_t tile[RT];
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    const int64_t t = min((int64_t)blockIdx.x * OT + a % OT, tiles - 1);
    tile[a] = t + (a / OT) * tiles;
  }
  ls_f32x4 acc[RT][MT];
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int c = 0; c < MT; ++c) acc[a][c] = ls_f32x4{0.f, 0.f, 0.f, 0.f};

  ls_u32x4 wt[RT][4];
  uint32_t sc[RT];
  auto load_w = [&](int64_t j, int i) {
    const int64_t chunk = min(4 * j + i, kc - 1);  // past the last one: x is zero there
#pragma unroll
    for (int a = 0; a < RT; ++a) wt[a][i] = ls_load16(codes + ((tile[a] * kc + chunk) * 64 + lane) * 16);
  };
  auto load_s = [&](int64_t j) {
#pragma unroll
    for (int a = 0; a < RT; ++a) sc[a] = scales[(tile[a] * kc4 + j) * 64 + lane];
  };
  const uint16_t* xrow[MT];
#pragma unroll
  for (int c = 0; c < MT; ++c) xrow[c] = x + min(m0 + 16 * c + r, m - 1) * xrs;
  // Rows past the last are the last again (not written); inputs past the last are zero, as only
  // a wave's last group may have (`last`).  No load is conditional: it would be waited for
  // where the paths meet.
  ls_u32x4 xr[MT][4];
  auto load_x = [&](int64_t j, int i, auto last) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int64_t k = 512 * j + 128 * i + 32 * p + 8 * q;
#pragma unroll
      for (int c = 0; c < MT; ++c) {
        xr[c][p] = ls_load16(xrow[c] + (decltype(last)::value ? min(k, K - 8) : k));
        if (decltype(last)::value && k >= K) xr[c][p] = ls_u32x4{0u, 0u, 0u, 0u};
      }
    }
  };
  // 512 inputs whose weights are in registers (or on their way), with the loads of the wave's
  // next ones.
  auto group = [&](int64_t j, auto more) {
    constexpr bool kMore = decltype(more)::value;
    uint32_t s4[RT];
#pragma unroll
    for (int a = 0; a < RT; ++a) s4[a] = sc[a];
    if constexpr (kMore) load_s(j + NW);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ls_u32x4 xf[MT][4];
#pragma unroll
      for (int c = 0; c < MT; ++c) {
#pragma unroll
        for (int p = 0; p < 4; ++p) xf[c][p] = xr[c][p];
        mx4_transpose(xf[c]);
      }
      if (i < 3)
        load_x(j, i + 1, std::bool_constant<!kMore>());
      else if constexpr (kMore)
        load_x(j + NW, 0, std::true_type());
#pragma unroll
      for (int a = 0; a < RT; ++a) {
        const float f = __uint_as_float(((s4[a] >> (8 * i)) & 0xffu) << 23);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const ls_u32x4 wf = mx4_expand<DT>(wt[a][i][s], f);
#pragma unroll
          for (int c = 0; c < MT; ++c) acc[a][c] = LsElem<DT>::mfma(wf, xf[c][s], acc[a][c]);
        }
      }
      if constexpr (kMore) load_w(j + NW, i);
    }
  };
  int64_t j = w;
  if (j < kc4) {
    load_s(j);
    load_w(j, 0);
    load_x(j, 0, std::true_type());
#pragma unroll
    for (int i = 1; i < 4; ++i) load_w(j, i);
    for (; j + NW < kc4; j += NW) group(j, std::true_type());
    group(j, std::false_type());
  }
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int c = 0; c < MT; ++c) s_acc[w][a * MT + c][lane] = acc[a][c];
  __syncthreads();
  // acc[a][c][i]: output 16 tile + 4 q + i of row m0 + 16 c + r.  A wave a (tile, 16 rows).
  for (int u = w; u < OT * MT; u += NW) {
    const int a = u / MT, c = u - a * MT;
    ls_f32x4 y = s_acc[0][u][lane];
#pragma unroll
    for (int i = 1; i < NW; ++i) y += s_acc[i][u][lane];
    if constexpr (PAIR) {
      ls_f32x4 up = s_acc[0][u + OT * MT][lane];
#pragma unroll
      for (int i = 1; i < NW; ++i) up += s_acc[i][u + OT * MT][lane];
      y = mx4_silu_mul(y, up);
    }
    const int64_t t = (int64_t)blockIdx.x * OT + a, row = m0 + 16 * c + r;
    if (t < tiles && row < m) mx4_store<DT>(y, out + row * ors, 16 * t + 4 * q, n_out);
  }
}

// More rows: what x costs a compute unit then bounds the product (16 rows of x are 4 KB for
// every 1 KB of a tile), so eight tiles of outputs share it through LDS.  Workgroup (eight
// tiles, or four and their up projections; block of 16 MT rows; slice z of the inputs): eight
// waves, wave (n, h) two tiles over the h-th half of the slice.  256 inputs of each half are
// staged at a time, in two buffers: the four waves of a half load x as it lies (wave n the n-th
// 64 bytes of each 256, four neighbouring lanes a row: 73448 x 4096, 64 rows 77 us; with a
// row's four lanes 16 apart 84), and an operand is read back across the pieces, 256 contiguous
// bytes for 16 lanes.  The halves are summed through LDS; with several slices float32 parts go
// to the workspace, [slice][row][16 tiles], and a second kernel adds them in order.
//
// 16384 outputs of gate and up, 4096 inputs: one row 14.4 us, 71 MB at 4.9 TB/s; 33 rows 21.4, the
// reads of x from LDS and the matrix instructions adding some 3 us each.
template <int DT, int MT, bool PAIR>
__global__ __launch_bounds__(512) void ls_mx4_rows_kernel(const Mx4Args args) {
  const uint16_t* __restrict__ x = args.x;
  const int64_t xrs = args.xrs;
  const int64_t m = args.m;
  const int64_t K = args.K;
  const uint8_t* __restrict__ codes = args.codes;
  const uint32_t* __restrict__ scales = args.scales;
  const int64_t kc = args.kc;
  const int64_t kc4 = args.kc4;
  const int64_t tiles = args.tiles;
  const int64_t per_half = args.per_half;
  const int64_t n_out = args.n_out;
  uint16_t* __restrict__ out = args.out;
  const int64_t ors = args.ors;
  float* __restrict__ part = args.part;
  constexpr int OT = PAIR ? 4 : 8;  // tiles of outputs of the workgroup
  // [buffer][half][128 inputs][16 rows][32 inputs][16 p + r]: 16 bytes, piece p of row r
  __shared__ __attribute__((aligned(16))) ls_u32x4 s_x[2][2][2][MT][4][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = w & 3, h = w >> 2;
  const int r = lane & 15, q = lane >> 4;
  const int xr = lane >> 2, xp = lane & 3;  // row and piece of x that the lane stages
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  int64_t ot[2], tile[2];  // tile of outputs, tile of the weight (past the last: the last again)
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    ot[a] = (int64_t)blockIdx.x * OT + (PAIR ? wn : 2 * wn + a);
    tile[a] = min(ot[a], tiles - 1) + (PAIR ? a * tiles : 0);
  }
  const int64_t g0 = (2 * (int64_t)blockIdx.z + h) * per_half;  // groups of 512 inputs
  const int64_t g1 = min(kc4, g0 + per_half);
  ls_f32x4 acc[2][MT];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < MT; ++c) acc[a][c] = ls_f32x4{0.f, 0.f, 0.f, 0.f};

  // Past the half's end weights are those of the last tile under scale 1 (under another tile's
  // scale a value might not be finite in fp16), and x is zero.
  ls_u32x4 wt[2][4];
  uint32_t sc[2];
  auto load_w = [&](int64_t g, int i) {
    const int64_t chunk = min(4 * g + i, kc - 1);
#pragma unroll
    for (int a = 0; a < 2; ++a) wt[a][i] = ls_load16(codes + ((tile[a] * kc + chunk) * 64 + lane) * 16);
  };
  auto load_s = [&](int64_t g) {
#pragma unroll
    for (int a = 0; a < 2; ++a) sc[a] = scales[(tile[a] * kc4 + min(g, kc4 - 1)) * 64 + lane];
  };
  ls_u32x4 xs[2 * MT];
  auto load_x = [&](int64_t g, int st) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t k = 512 * g + 256 * st + 128 * i + 32 * wn + 8 * xp;
#pragma unroll
      for (int c = 0; c < MT; ++c) {
        const int64_t row = m0 + 16 * c + xr;
        xs[i * MT + c] = row < m && k < K && g < g1 ? ls_load16(x + row * xrs + k)
                                                    : ls_u32x4{0u, 0u, 0u, 0u};
      }
    }
  };
  auto store_x = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < MT; ++c) s_x[buf][h][i][c][wn][16 * xp + xr] = xs[i * MT + c];
  };
  load_s(g0);
  load_x(g0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) load_w(g0, i);
  store_x(0);
  for (int64_t j = 0; j < per_half; ++j) {
    const int64_t g = g0 + j;
    const uint32_t s4[2] = {g < g1 ? sc[0] : 0x7f7f7f7fu, g < g1 ? sc[1] : 0x7f7f7f7fu};
    load_s(g + 1);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      __syncthreads();  // buffer st is whole, and nobody reads the other any more
      load_x(g + st, st ^ 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float f[2];
#pragma unroll
        for (int a = 0; a < 2; ++a)
          f[a] = __uint_as_float(((s4[a] >> (16 * st + 8 * i)) & 0xffu) << 23);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          ls_u32x4 xf[MT];
#pragma unroll
          for (int c = 0; c < MT; ++c) xf[c] = s_x[st][h][i][c][q][16 * s + r];
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const ls_u32x4 wf = mx4_expand<DT>(wt[a][2 * st + i][s], f[a]);
#pragma unroll
            for (int c = 0; c < MT; ++c) acc[a][c] = LsElem<DT>::mfma(wf, xf[c], acc[a][c]);
          }
        }
        load_w(g + 1, 2 * st + i);
      }
      store_x(st ^ 1);
    }
  }
  __syncthreads();
  ls_f32x4(*s_acc)[2][MT][64] = reinterpret_cast<ls_f32x4(*)[2][MT][64]>(&s_x[0][0][0][0][0][0]);
  if (h == 1) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int c = 0; c < MT; ++c) s_acc[wn][a][c][lane] = acc[a][c];
  }
  __syncthreads();
  if (h == 1) return;
  // acc[a][c][i]: output 16 tile + 4 q + i of row m0 + 16 c + r.
#pragma unroll
  for (int c = 0; c < MT; ++c) {
    const int64_t row = m0 + 16 * c + r;
    if (row >= m) continue;
#pragma unroll
    for (int a = 0; a < 2; ++a) acc[a][c] += s_acc[wn][a][c][lane];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      if (ot[a] >= tiles) continue;
      if (gridDim.z > 1) {
        const int64_t cols = 16 * tiles * (PAIR ? 2 : 1);
        *reinterpret_cast<ls_f32x4*>(part + ((int64_t)blockIdx.z * m + row) * cols + 16 * tile[a] + 4 * q) =
            acc[a][c];
      } else if (!PAIR) {
        mx4_store<DT>(acc[a][c], out + row * ors, 16 * ot[a] + 4 * q, n_out);
      } else if (a == 0) {
        mx4_store<DT>(mx4_silu_mul(acc[0][c], acc[1][c]), out + row * ors, 16 * ot[a] + 4 * q, n_out);
      }
    }
  }
}

// The slices' parts, added in order: a thread per four outputs of a row.  Bound by its launch (4096
// outputs, 7 rows, 8 slices: 3.0 us for 1 MB).
template <int DT, bool PAIR>
__global__ __launch_bounds__(256) void ls_mx4_join_kernel(const float* __restrict__ part,
                                                          int64_t slices, int64_t m, int64_t tiles,
                                                          int64_t n_out, uint16_t* __restrict__ out,
                                                          int64_t ors) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / (4 * tiles), col = 4 * (at - row * 4 * tiles);
  if (row >= m) return;
  const int64_t cols = 16 * tiles * (PAIR ? 2 : 1);
  ls_f32x4 y[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll 8
  for (int64_t z = 0; z < slices; ++z)
#pragma unroll
    for (int a = 0; a < (PAIR ? 2 : 1); ++a)
      y[a] += *reinterpret_cast<const ls_f32x4*>(part + (z * m + row) * cols + a * 16 * tiles + col);
  mx4_store<DT>(PAIR ? mx4_silu_mul(y[0], y[1]) : y[0], out + row * ors, col, n_out);
}

// ---------------------------------------------------------------------------
// Laying out: a wave per tile of 16 outputs by 128 inputs, a lane per scale group.
// The scale code is the least c >= 8 with max |w| <= 6 2^(c - 127) (127 for a group of
// zeros), at most 252, as 6 2^125 is the last product that bf16 holds: only magnitudes above
// it saturate.  Values go to the nearest E2M1 one, ties to the even code.  ALIGNED: rows in
// pieces of 16 bytes (all of a piece's eight inputs exist or none), else single elements.
// Bound by memory (32768 x 4096 bf16: 86 us, 340 MB at 4.0 TB/s; single elements 319).
// ---------------------------------------------------------------------------
template <int DT, bool ALIGNED>
__global__ __launch_bounds__(256) void ls_mx4_quantize_kernel(
    const typename LsElem<DT>::T* __restrict__ w, int64_t wrs, int64_t N, int64_t K, int64_t kc,
    int64_t kc4, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t nt = blockIdx.x / kc4, group = blockIdx.x - nt * kc4;  // a wave a chunk of the group
  const int64_t chunk = 4 * group + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t row = 16 * nt + (lane & 15), k0 = 128 * chunk + 32 * (lane >> 4);
  float v[32];
  float top = 0.f;
  if constexpr (ALIGNED) {
    constexpr int kBytes = sizeof(typename LsElem<DT>::T), kEach = 16 / kBytes;  // inputs a load
    const auto* wr = w + min(row, N - 1) * wrs;
    ls_u32x4 x[32 / kEach];
#pragma unroll
    for (int p = 0; p < 32 / kEach; ++p) x[p] = ls_load16(wr + min(k0 + kEach * p, K - kEach));
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const uint32_t u = x[e / kEach][e % kEach * kBytes / 4];
      if constexpr (kBytes == 4)
        v[e] = __uint_as_float(u);
      else
        v[e] = LsElem<DT>::to_f((uint16_t)(e & 1 ? u >> 16 : u & 0xffffu));
      if (row >= N || k0 + e >= K) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      v[e] = row < N && k0 + e < K ? LsElem<DT>::to_f(w[row * wrs + k0 + e]) : 0.f;
  }
#pragma unroll
  for (int e = 0; e < 32; ++e) top = fmaxf(top, fabsf(v[e]));
  const uint32_t bits = __float_as_uint(top);
  // 6 = 1.5 2^2.
  int c = (int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0);
  c = top == 0.f ? 127 : min(max(c, 8), 252);
  scales[((nt * kc4 + (chunk >> 2)) * 64 + lane) * 4 + (chunk & 3)] = (uint8_t)c;
  if (chunk >= kc) return;
  const float inv = __uint_as_float((uint32_t)(254 - c) << 23);
  ls_u32x4 o = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    const float a = fabsf(v[e]) * inv;
    const uint32_t m = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) +
                       (a >= 3.5f) + (a > 5.f);
    const uint32_t s = __float_as_uint(v[e]) >> 31;
    o[e >> 3] |= (m | (s << 3)) << (4 * (e & 7));
  }
  *reinterpret_cast<ls_u32x4*>(codes + ((nt * kc + chunk) * 64 + lane) * 16) = o;
}

// The weight's values in 16 bits (exact in bf16; rounded to fp16), rows of K.  Bound by what it
// writes (32768 x 4096: 70 us, 340 MB at 4.9 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void ls_mx4_dequantize_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t N, int64_t K,
    int64_t kc, int64_t kc4, uint16_t* __restrict__ out, int64_t ors) {
  const int64_t nt = blockIdx.y, chunk = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t row = 16 * nt + (lane & 15);
  if (chunk >= kc) return;
  const ls_u32x4 v = ls_load16(codes + ((nt * kc + chunk) * 64 + lane) * 16);
  const uint32_t c = scales[((nt * kc4 + (chunk >> 2)) * 64 + lane) * 4 + (chunk & 3)];
  const float f = __uint_as_float(c << 23);
  ls_u32x4 o[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) o[s] = mx4_expand<DT>(v[s], f);
  mx4_transpose(o);  // piece q of the four groups: four lanes write 64 bytes together
  if (row >= N) return;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int64_t k = 128 * chunk + 32 * s + 8 * (lane >> 4);
    if (k < K) *reinterpret_cast<ls_u32x4*>(out + row * ors + k) = o[s];
  }
}

constexpr int64_t kMaxThreads = 0xffffffffLL;  // of a launch along a dimension

bool mx4_sizes(int64_t n, int64_t k) {
  return n >= 1 && k >= 8 && k % 8 == 0 && n <= 0x7fffffffLL && k <= 0x7fffffffLL;
}

}  // namespace

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {
// How a product is cut.
struct Mx4Cut {
  bool shared;       // ls_mx4_rows_kernel, else ls_mx4_kernel
  int mt;            // 16-row blocks of x a workgroup
  int nw, rt;        // ls_mx4_kernel: waves and tiles of the weight a workgroup
  int64_t slices;    // ls_mx4_rows_kernel: of the inputs
  int64_t per_half;  // and groups of 512 inputs for each half of a slice
  int64_t tiles;     // of outputs (16 each)
  int64_t kc, kc4;   // tiles and groups of four tiles along the inputs
  int64_t blocks;    // of rows
};

// Measured with weights from memory (us; a large copy reaches 4.9 to 5.1 TB/s), outputs x inputs, rows:
//   waves and tiles a workgroup (8/1, 8/2, 4/4), one row: 4096 x 4096 5.2, 6.1, 9.0; 4608 x 4096
//   6.9, 6.2, 9.1; 16384 x 4096 12.6, 11.5, 12.7; 73448 x 4096 47, 36.5, 33.3 (floor 31).  So
//   eight waves up to 1024 tiles of the weight, one tile up to 256 (all workgroups in one round).
//   ls_mx4_kernel, ls_mx4_rows_kernel (with slices: a second launch, 4 us more of the host), above
//   16 rows: 4096 x 2048, 17 rows 5.3, 8.4, 64 rows 9.8, 12.3; 4096 x 4096, 17 rows 8.0, 10.3, 32
//   rows 10.5, 11.1, 33 rows 13.2, 12.4, 64 rows 17.7, 14.6; 2048 x 8192, 17 rows 12.5, 9.9, 32 rows
//   17.2, 10.4; [gate; up] 32768 x 4096, 33 rows 33.9, 23.7 (floor 13.9).  The first takes as long
//   as its rounds of 256 workgroups and the inputs each walks: up to 4096 inputs in one round or
//   2048 in two.  Without slices the second is as cheap to launch: 32768 x 1024, 33 rows 15.3,
//   10.4; 8192 x 1024, 17 rows (one round) 4.8, 6.4.
//   Up to 16 rows: [gate; up] 32768 x 4096, one row 18.6, 17.4, 16 rows 20.1, 17.6; 4608 x 4096,
//   16 rows 8.0, 9.7; 73448 x 4096, one row 33.3, 41.1: the second where its workgroups just fill
//   the chip's 256 units without slices.  And where inputs are long and tiles few, by rows:
//   1024 x 16384, one row 11.7, 8.6; 1024 x 12288, one row 9.2, 8.5, 8 rows 10.6, 9.1, 16 rows 14.0,
//   9.1; 1024 x 8192, one row 6.3, 6.9, 8 rows 7.3, 7.2, 16 rows 9.6, 7.4.  (These are times on the
//   GPU.  The rule's border lies above some sizes that the second form does faster, 1024 x 8192 at
//   16 rows among them: its second launch costs a call that is not captured 4 us more.)
Mx4Cut mx4_cut(int64_t rows, int64_t K, int64_t N, bool silu) {
  Mx4Cut c;
  const int64_t tiles = (N + 15) / 16;  // of the weight
  c.kc = (K + 127) / 128;
  c.kc4 = (c.kc + 3) / 4;
  c.tiles = silu ? tiles / 2 : tiles;
  c.mt = rows > 64 ? 4 : (int)((rows + 15) / 16);
  c.blocks = (rows + 16 * c.mt - 1) / (16 * c.mt);
  c.nw = tiles <= 1024 ? 8 : 4;
  c.rt = c.nw == 4 ? 4 : silu || tiles > 256 ? 2 : 1;
  const int64_t per_wg = silu ? 4 : 8;
  const int64_t wgs = (c.tiles + per_wg - 1) / per_wg * c.blocks;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(c.kc4 / 2, 256 / wgs));
  c.per_half = (c.kc4 + 2 * want - 1) / (2 * want);
  c.slices = (c.kc4 + 2 * c.per_half - 1) / (2 * c.per_half);
  const int64_t rounds = ((tiles + c.rt - 1) / c.rt * ((rows + 31) / 32) + 255) / 256;
  c.shared = rows > 16 ? K * rounds > 4096 || (c.slices == 1 && rounds > 1)
                       : (c.slices == 1 && wgs > 128 && wgs <= 256) ||
                             (tiles <= 256 && c.kc4 * (rows + 16) >= 544);
  if (!c.shared && c.mt > 2) {  // few tiles and many rows: blocks of 32, their registers bound the waves
    c.mt = 2;
    c.blocks = (rows + 31) / 32;
  }
  return c;
}
}  // namespace

extern "C" size_t ls_linear_mx4_workspace_size(int64_t rows, int64_t in_features,
                                               int64_t out_features, int32_t silu_mul) {
  if (rows <= 0 || !mx4_sizes(out_features, in_features)) return 0;
  const Mx4Cut c = mx4_cut(rows, in_features, out_features, silu_mul != 0);
  if (!c.shared || c.slices == 1) return 0;
  return 4 * (size_t)c.slices * rows * c.tiles * 16 * (silu_mul ? 2 : 1);
}

extern "C" int ls_linear_mx4(const void* x, int64_t x_row_stride, int64_t rows,
                             int64_t in_features, const void* codes, const void* scales,
                             int64_t out_features, int32_t silu_mul, int32_t dtype, void* out,
                             int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                             void* stream) {
  const char* who = "ls_linear_mx4";
  LS_REQUIRE(rows >= 0 && mx4_sizes(out_features, in_features), LS_ERR_INVALID,
             "%s: need rows >= 0, out_features >= 1 and in_features a multiple of 8", who);
  LS_REQUIRE(!silu_mul || out_features % 32 == 0, LS_ERR_UNSUPPORTED,
             "%s: the gated form needs out_features a multiple of 32", who);
  LS_REQUIRE(dtype == LS_BF16 || dtype == LS_F16, LS_ERR_UNSUPPORTED, "%s: x is bf16 or fp16", who);
  LS_REQUIRE(x_row_stride % 8 == 0, LS_ERR_UNSUPPORTED, "%s: rows of x must be 16-byte aligned",
             who);
  if (rows == 0) return LS_OK;
  LS_REQUIRE(x && codes && scales && out, LS_ERR_INVALID, "%s: null pointer", who);
  LS_REQUIRE(ls_aligned16(x) && ls_aligned16(codes) && ((uintptr_t)scales & 3) == 0 &&
                 ls_aligned16(workspace),
             LS_ERR_UNSUPPORTED, "%s: x, codes and workspace must be 16-byte aligned", who);
  const Mx4Cut cut = mx4_cut(rows, in_features, out_features, silu_mul != 0);
  const size_t need = ls_linear_mx4_workspace_size(rows, in_features, out_features, silu_mul);
  LS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), LS_ERR_WORKSPACE,
             "%s: workspace %zu < %zu", who, workspace ? workspace_bytes : (size_t)0, need);
  LS_REQUIRE(cut.blocks <= 65535, LS_ERR_UNSUPPORTED, "%s: too many rows", who);
  // (A large weight has 64 threads for each of its tiles.)
  LS_REQUIRE((out_features + 15) / 16 * 64 <= kMaxThreads - 512, LS_ERR_UNSUPPORTED,
             "%s: too many outputs", who);
  const int64_t n_out = silu_mul ? out_features / 2 : out_features;
  hipStream_t stm = (hipStream_t)stream;
  const Mx4Args args = {(const uint16_t*)x, x_row_stride, rows, in_features, (const uint8_t*)codes,
                        (const uint32_t*)scales, cut.kc, cut.kc4, cut.tiles, cut.per_half, n_out,
                        (uint16_t*)out, out_row_stride, (float*)workspace};
  using std::integral_constant;
  auto few = [&](auto dt, auto mtc, auto pr, auto rt, auto nw) {
    constexpr int RT = decltype(rt)::value, NW = decltype(nw)::value;
    constexpr bool PAIR = decltype(pr)::value;
    constexpr int OT = PAIR ? RT / 2 : RT;
    hipLaunchKernelGGL((ls_mx4_kernel<decltype(dt)::value, decltype(mtc)::value, RT, PAIR, NW>),
                       dim3((unsigned)((cut.tiles + OT - 1) / OT), (unsigned)cut.blocks),
                       dim3(64 * NW), 0, stm, args);
    return ls_check_launch("ls_mx4_kernel");
  };
  auto by_waves = [&](auto dt, auto mtc, auto pr) {
    constexpr int P = decltype(pr)::value ? 2 : 1;
    // (Over 16 rows of more than 1024 tiles take the shared form: two rounds at least, one slice.)
    if constexpr (decltype(mtc)::value == 1)
      if (cut.nw == 4)
        return few(dt, mtc, pr, integral_constant<int, 4>(), integral_constant<int, 4>());
    if (cut.rt == 2) return few(dt, mtc, pr, integral_constant<int, 2>(), integral_constant<int, 8>());
    return few(dt, mtc, pr, integral_constant<int, P>(), integral_constant<int, 8>());
  };
  auto shared = [&](auto dt, auto mtc, auto pr) {
    constexpr int DT = decltype(dt)::value;
    constexpr bool PAIR = decltype(pr)::value;
    constexpr int OT = PAIR ? 4 : 8;
    hipLaunchKernelGGL((ls_mx4_rows_kernel<DT, decltype(mtc)::value, PAIR>),
                       dim3((unsigned)((cut.tiles + OT - 1) / OT), (unsigned)cut.blocks,
                            (unsigned)cut.slices),
                       dim3(512), 0, stm, args);
    const int rc = ls_check_launch("ls_mx4_rows_kernel");
    if (rc || cut.slices == 1) return rc;
    hipLaunchKernelGGL((ls_mx4_join_kernel<DT, PAIR>),
                       dim3((unsigned)((rows * cut.tiles * 4 + 255) / 256)), dim3(256), 0, stm,
                       (const float*)workspace, cut.slices, rows, cut.tiles, n_out, (uint16_t*)out,
                       out_row_stride);
    return ls_check_launch("ls_mx4_join_kernel");
  };
  auto by_form = [&](auto dt, auto mtc, auto pr) {
    if constexpr (decltype(mtc)::value <= 2)
      if (!cut.shared) return by_waves(dt, mtc, pr);
    return shared(dt, mtc, pr);
  };
  auto by_pair = [&](auto dt, auto mtc) {
    return silu_mul ? by_form(dt, mtc, std::true_type()) : by_form(dt, mtc, std::false_type());
  };
  auto by_rows = [&](auto dt) {
    if (cut.mt == 1) return by_pair(dt, integral_constant<int, 1>());
    if (cut.mt == 2) return by_pair(dt, integral_constant<int, 2>());
    if (cut.mt == 3) return by_pair(dt, integral_constant<int, 3>());
    return by_pair(dt, integral_constant<int, 4>());
  };
  return dtype == LS_BF16 ? by_rows(integral_constant<int, LS_BF16>())
                          : by_rows(integral_constant<int, LS_F16>());
}

extern "C" int ls_quantize_mx4(const void* weight, int64_t weight_row_stride, int64_t out_features,
                               int64_t in_features, int32_t dtype, void* codes, void* scales,
                               void* stream) {
  const char* who = "ls_quantize_mx4";
  LS_REQUIRE(mx4_sizes(out_features, in_features), LS_ERR_INVALID,
             "%s: need out_features >= 1 and in_features a multiple of 8", who);
  LS_REQUIRE(dtype == LS_F32 || dtype == LS_BF16 || dtype == LS_F16, LS_ERR_INVALID,
             "%s: unknown dtype", who);
  LS_REQUIRE(weight && codes && scales, LS_ERR_INVALID, "%s: null pointer", who);
  LS_REQUIRE(ls_aligned16(codes), LS_ERR_UNSUPPORTED, "%s: codes must be 16-byte aligned", who);
  const int64_t tiles = (out_features + 15) / 16, kc = (in_features + 127) / 128, kc4 = (kc + 3) / 4;
  LS_REQUIRE(tiles * kc4 * 256 <= kMaxThreads, LS_ERR_UNSUPPORTED, "%s: weight too large", who);
  auto run = [&](auto dt, auto aligned) {
    constexpr int DT = decltype(dt)::value;
    hipLaunchKernelGGL((ls_mx4_quantize_kernel<DT, decltype(aligned)::value>),
                       dim3((unsigned)(tiles * kc4)), dim3(256), 0, (hipStream_t)stream,
                       (const typename LsElem<DT>::T*)weight, weight_row_stride, out_features,
                       in_features, kc, kc4, (uint8_t*)codes, (uint8_t*)scales);
    return ls_check_launch("ls_mx4_quantize_kernel");
  };
  auto launch = [&](auto dt) {
    return ls_aligned16(weight) && weight_row_stride % 8 == 0 ? run(dt, std::true_type())
                                                              : run(dt, std::false_type());
  };
  if (dtype == LS_F32) return launch(std::integral_constant<int, LS_F32>());
  return dtype == LS_BF16 ? launch(std::integral_constant<int, LS_BF16>())
                          : launch(std::integral_constant<int, LS_F16>());
}

extern "C" int ls_dequantize_mx4(const void* codes, const void* scales, int64_t out_features,
                                 int64_t in_features, int32_t dtype, void* out,
                                 int64_t out_row_stride, void* stream) {
  const char* who = "ls_dequantize_mx4";
  LS_REQUIRE(mx4_sizes(out_features, in_features), LS_ERR_INVALID,
             "%s: need out_features >= 1 and in_features a multiple of 8", who);
  LS_REQUIRE(dtype == LS_BF16 || dtype == LS_F16, LS_ERR_UNSUPPORTED, "%s: bf16 or fp16", who);
  LS_REQUIRE(codes && scales && out, LS_ERR_INVALID, "%s: null pointer", who);
  LS_REQUIRE(ls_aligned16(codes) && ls_aligned16(out) && out_row_stride % 8 == 0,
             LS_ERR_UNSUPPORTED, "%s: codes and output rows must be 16-byte aligned", who);
  const int64_t tiles = (out_features + 15) / 16, kc = (in_features + 127) / 128, kc4 = (kc + 3) / 4;
  // Tiles in the grid's second dimension, 65535 at a time.
  for (int64_t t0 = 0; t0 < tiles; t0 += 65535) {
    const int64_t n = std::min<int64_t>(65535, tiles - t0);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)((kc + 3) / 4), (unsigned)n), dim3(256), 0,
                         (hipStream_t)stream, (const uint8_t*)codes + t0 * kc * 1024,
                         (const uint8_t*)scales + t0 * kc4 * 256, out_features - 16 * t0,
                         in_features, kc, kc4, (uint16_t*)out + 16 * t0 * out_row_stride,
                         out_row_stride);
      return ls_check_launch("ls_mx4_dequantize_kernel");
    };
    const int rc = dtype == LS_BF16 ? launch(ls_mx4_dequantize_kernel<LS_BF16>)
                                    : launch(ls_mx4_dequantize_kernel<LS_F16>);
    if (rc) return rc;
  }
  return LS_OK;
}
