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

// Workgroup (tile of outputs, block of 16 MT rows of x): NW waves share the inputs, four tiles
// (512 inputs) at a time, and are summed through LDS in order.  PAIR: the tile and the one
// `pair` tiles later are the gate and up projections of the same outputs, and
// silu(gate) * up is written (float32 up to the one rounding).
template <int DT, int MT, bool PAIR, int NW>
__global__ __launch_bounds__(64 * NW) void ls_mx4_kernel(
    const uint16_t* __restrict__ x, int64_t xrs, int64_t m, int64_t K,
    const uint8_t* __restrict__ codes, const uint32_t* __restrict__ scales, int64_t kc, int64_t kc4,
    int64_t pair, int64_t n_out, uint16_t* __restrict__ out, int64_t ors) {
  constexpr int RT = PAIR ? 2 : 1;
  __shared__ __attribute__((aligned(16))) ls_f32x4 s_acc[NW][RT * MT][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int64_t nt = blockIdx.x, m0 = (int64_t)blockIdx.y * (16 * MT);
  ls_f32x4 acc[RT][MT];
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int c = 0; c < MT; ++c) acc[a][c] = ls_f32x4{0.f, 0.f, 0.f, 0.f};

  for (int64_t j = w; j < kc4; j += NW) {
    const int n = (int)min<int64_t>(4, kc - 4 * j);
    ls_u32x4 wt[RT][4];
    uint32_t sc[RT];
#pragma unroll
    for (int a = 0; a < RT; ++a) {
      const int64_t tile = nt + a * pair;
      sc[a] = scales[(tile * kc4 + j) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        wt[a][i] = i < n ? ls_load16(codes + ((tile * kc + 4 * j + i) * 64 + lane) * 16)
                         : ls_u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ls_u32x4 xf[MT][4];
      const int64_t k0 = 512 * j + 128 * i + 32 * q;
#pragma unroll
      for (int c = 0; c < MT; ++c) {
        const int64_t row = m0 + 16 * c + r;
#pragma unroll
        for (int s = 0; s < 4; ++s)
          xf[c][s] = row < m && k0 + 8 * s < K ? ls_load16(x + row * xrs + k0 + 8 * s)
                                               : ls_u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int a = 0; a < RT; ++a) {
        const float f = __uint_as_float(((sc[a] >> (8 * i)) & 0xffu) << 23);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const ls_u32x4 wf = mx4_expand<DT>(wt[a][i][s], f);
#pragma unroll
          for (int c = 0; c < MT; ++c) acc[a][c] = LsElem<DT>::mfma(wf, xf[c][s], acc[a][c]);
        }
      }
    }
  }
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int c = 0; c < MT; ++c) s_acc[w][a * MT + c][lane] = acc[a][c];
  __syncthreads();
  // acc[c][i]: output 16 nt + 4 q + i of row m0 + 16 c + r.
  for (int c = w; c < MT; c += NW) {
    ls_f32x4 y[RT];
#pragma unroll
    for (int a = 0; a < RT; ++a) {
      y[a] = s_acc[0][a * MT + c][lane];
#pragma unroll
      for (int i = 1; i < NW; ++i) y[a] += s_acc[i][a * MT + c][lane];
    }
    if constexpr (PAIR) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[0][i] = y[0][i] / (1.f + __expf(-y[0][i])) * y[1][i];
    }
    const int64_t row = m0 + 16 * c + r, col = 16 * nt + 4 * q;
    if (row >= m) continue;
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = LsElem<DT>::from_f(y[0][i]);
    uint16_t* o = out + row * ors + col;
    if (col + 4 <= n_out && ((uintptr_t)o & 7) == 0) {
      *reinterpret_cast<uint2*>(o) = make_uint2(ls_pack2(h[0], h[1]), ls_pack2(h[2], h[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col + i < n_out) o[i] = h[i];
    }
  }
}

// ---------------------------------------------------------------------------
// Laying out: a wave per tile of 16 outputs by 128 inputs, a lane per scale group.
// The scale code is the least c >= 8 with max |w| <= 6 2^(c - 127) (127 for a group of
// zeros), at most 252, as 6 2^125 is the last product that bf16 holds: only magnitudes above
// it saturate.  Values go to the nearest E2M1 one, ties to the even code.
// ---------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(64) void ls_mx4_quantize_kernel(
    const typename LsElem<DT>::T* __restrict__ w, int64_t wrs, int64_t N, int64_t K, int64_t kc,
    int64_t kc4, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t at = blockIdx.x;  // nt * 4 kc4 + chunk, chunks rounded up to whole scale words
  const int64_t nt = at / (4 * kc4), chunk = at - nt * 4 * kc4;
  const int lane = threadIdx.x;
  const int64_t row = 16 * nt + (lane & 15), k0 = 128 * chunk + 32 * (lane >> 4);
  float v[32];
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    v[e] = row < N && k0 + e < K ? LsElem<DT>::to_f(w[row * wrs + k0 + e]) : 0.f;
    top = fmaxf(top, fabsf(v[e]));
  }
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

// The weight's values in 16 bits (exact in bf16; rounded to fp16), rows of K.
template <int DT>
__global__ __launch_bounds__(256) void ls_mx4_dequantize_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t N, int64_t K,
    int64_t kc, int64_t kc4, uint16_t* __restrict__ out, int64_t ors) {
  const int64_t nt = blockIdx.y, chunk = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t row = 16 * nt + (lane & 15), k0 = 128 * chunk + 32 * (lane >> 4);
  if (chunk >= kc || row >= N) return;
  const ls_u32x4 v = ls_load16(codes + ((nt * kc + chunk) * 64 + lane) * 16);
  const uint32_t c = scales[((nt * kc4 + (chunk >> 2)) * 64 + lane) * 4 + (chunk & 3)];
  const float f = __uint_as_float(c << 23);
#pragma unroll
  for (int s = 0; s < 4; ++s)
    if (k0 + 8 * s < K)
      *reinterpret_cast<ls_u32x4*>(out + row * ors + k0 + 8 * s) = mx4_expand<DT>(v[s], f);
}

bool mx4_sizes(int64_t n, int64_t k) {
  return n >= 1 && k >= 8 && k % 8 == 0 && n <= 0x7fffffffLL && k <= 0x7fffffffLL;
}

}  // namespace

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
extern "C" int ls_linear_mx4(const void* x, int64_t x_row_stride, int64_t rows,
                             int64_t in_features, const void* codes, const void* scales,
                             int64_t out_features, int32_t silu_mul, int32_t dtype, void* out,
                             int64_t out_row_stride, void* stream) {
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
  LS_REQUIRE(ls_aligned16(x) && ls_aligned16(codes) && ((uintptr_t)scales & 3) == 0,
             LS_ERR_UNSUPPORTED, "%s: x and codes must be 16-byte aligned", who);
  const int64_t tiles = (out_features + 15) / 16, kc = (in_features + 127) / 128, kc4 = (kc + 3) / 4;
  const int64_t n_out = silu_mul ? out_features / 2 : out_features;
  const int64_t grid_x = silu_mul ? tiles / 2 : tiles;
  const int mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int64_t grid_y = (rows + 16 * mt - 1) / (16 * mt);
  LS_REQUIRE(grid_y <= 65535, LS_ERR_UNSUPPORTED, "%s: too many rows", who);
  auto launch = [&](auto dt, auto mtc, auto pr) {
    constexpr int NW = 4;
    hipLaunchKernelGGL((ls_mx4_kernel<decltype(dt)::value, decltype(mtc)::value,
                                      decltype(pr)::value, NW>),
                       dim3((unsigned)grid_x, (unsigned)grid_y), dim3(64 * NW), 0,
                       (hipStream_t)stream, (const uint16_t*)x, x_row_stride, rows, in_features,
                       (const uint8_t*)codes, (const uint32_t*)scales, kc, kc4, grid_x, n_out,
                       (uint16_t*)out, out_row_stride);
    return ls_check_launch("ls_mx4_kernel");
  };
  auto by_pair = [&](auto dt, auto mtc) {
    return silu_mul ? launch(dt, mtc, std::true_type()) : launch(dt, mtc, std::false_type());
  };
  auto by_rows = [&](auto dt) {
    if (mt == 1) return by_pair(dt, std::integral_constant<int, 1>());
    if (mt == 2) return by_pair(dt, std::integral_constant<int, 2>());
    return by_pair(dt, std::integral_constant<int, 4>());
  };
  return dtype == LS_BF16 ? by_rows(std::integral_constant<int, LS_BF16>())
                          : by_rows(std::integral_constant<int, LS_F16>());
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
  LS_REQUIRE(tiles * 4 * kc4 <= 0x7fffffffLL, LS_ERR_UNSUPPORTED, "%s: weight too large", who);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    hipLaunchKernelGGL(ls_mx4_quantize_kernel<DT>, dim3((unsigned)(tiles * 4 * kc4)), dim3(64), 0,
                       (hipStream_t)stream, (const typename LsElem<DT>::T*)weight,
                       weight_row_stride, out_features, in_features, kc, kc4, (uint8_t*)codes,
                       (uint8_t*)scales);
    return ls_check_launch("ls_mx4_quantize_kernel");
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
