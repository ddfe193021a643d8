// Grouped product of MXFP4 rows with MXFP4 expert weights on gfx950 (the format: mx.h):
//   y[r][n] = sum_k x[r][k] w_e[n][k] + b_e[n],   r in the rows of expert e,
// and, for the first of an expert's two layers, act(y) quantised again: y never reaches memory.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows of 128 codes by 16 rows of 128 codes and
// applies both operands' block scales itself, with f32 sums: lane l holds row l % 16, features
// 32 (l / 16) .. +31, i.e. one block, 16 bytes of codes and one scale byte.  The weights are the
// first operand (result rows = output features), so a lane ends up with 4 consecutive features
// of one token per fragment.  Which weight row a lane reads is free: fragment f of a group of 32
// features gives lane row m the feature 8 (m / 4) + 4 f + m % 4, so the two fragments of a group
// leave 8 CONSECUTIVE features of a token in a lane, and a block of 32 in four lanes: the output
// leaves in 16-byte packs, and the block maximum of the quantising epilogue takes two exchanges.
//
// Few rows are bound by the weights' bytes (17/32 of one per weight), many by the matrix cores;
// which of two kernels and three tile shapes runs: choose_kernel().
#include <algorithm>

#include "quant_gemm.h"

namespace fmoe {

__device__ __forceinline__ f32x4 mx_mfma(i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
  const i32x8 a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 b8 = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  // 4 = E2M1 in either operand; the scale bytes are the lowest ones of sa and sb
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, sa, 0, sb);
}

// gelu(x) = x Phi(x) with Phi(x) = 1 / (1 + 2^z), z = -log2(Phi(x) / Phi(-x)) = x P(x^2) for
// |x| <= 6 and x P(36) outside: P of degree 12 in x^2 / 18 - 1, a reweighted least-squares fit on
// Chebyshev nodes.  Within 2e-7 + 3e-7 |gelu| of gelu everywhere (the fit, evaluated in f32 with an
// exact exponential and quotient: 1.42e-7 + 1e-7 |gelu|; the two instructions for these are good to
// 1.2e-7 each), so that hardly more codes than the sums' own rounding makes land on the other side
// of a boundary (degree 9, three instructions less, was off by 7e-7), and, for |x| <= 6, within
// 5e-6 of its value (3.7e-6 likewise), so that blocks whose values all lie in the negative tail
// keep their digits as well.  26 issue slots where erff takes about
// 60, with branches, and loses the tail: with one wave on a SIMD nothing hides them (a 256 x 256
// tile of 4096 features: 27 us of matrix instructions, 26 us of erff).
__device__ __forceinline__ float mx_gelu(float x) {
  const float t = fminf(fmaf(x * x, 1.f / 18.f, -1.f), 1.f);
  float p = 0.00220932276f;
  p = fmaf(p, t, -0.00235819351f);
  p = fmaf(p, t, -0.00623256993f);
  p = fmaf(p, t, 0.0106137199f);
  p = fmaf(p, t, -0.00437692506f);
  p = fmaf(p, t, 0.0022452944f);
  p = fmaf(p, t, -0.00346183078f);
  p = fmaf(p, t, -0.00412944285f);
  p = fmaf(p, t, 0.0250278097f);
  p = fmaf(p, t, -0.0735082775f);
  p = fmaf(p, t, 0.223777682f);
  p = fmaf(p, t, -1.27482498f);
  p = fmaf(p, t, -3.8811202f);
  // (2^z overflows to infinity far down, its inverse is 0 there)
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * p));
}

// ------------------------------------------------------------------------- few rows
// Weights straight from memory into registers, since nothing would read them twice: a workgroup's
// 4 waves take 16 rows of an expert, 32 features, and a quarter of K each, whose sums meet in LDS.
// K is split because there are few tiles otherwise: 128 rows of 16 experts, 4096 -> 1024, are 512
// workgroups and take 10 us (36 MB; 7 at the rate of a large copy) where 128 x 64 tiles take 13.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void mx_stream_kernel(QuantGemmArgs a) {
  constexpr int kWaves = 4, kCols = 32;
  __shared__ int s_sum[2 * kWaves], s_out[4];
  __shared__ float part[(kWaves - 1) * 8 * kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowTiles<16, kOneHeight, kWaves> tiles;
  tiles.scan(a.seg_off, a.n_expert, s_sum);
  const int n_pad = mx_quantises(MODE) ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const int n_cols = (n_pad + kCols - 1) / kCols;
  if (tiles.rows_f == 0) return;
  const int col = blockIdx.x / tiles.rows_f, v = blockIdx.x - col * tiles.rows_f;
  if (col >= n_cols) return;
  const TileRows t = tiles.find(a.seg_off, v, false, s_out);

  const int m = lane & 15, g = lane >> 4, base = col * kCols;
  const int64_t code_row = mx_code_bytes(a.in_feat), scale_row = mx_scale_bytes(a.in_feat);
  // rows and features past the end repeat the last one; their results are not stored
  const uint8_t *wc[2], *ws[2];
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const int64_t n = (int64_t)t.e * a.out_feat + min(base + mx_feature(f, m), a.out_feat - 1);
    wc[f] = a.wc + n * code_row + g * 16;
    ws[f] = a.ws + n * scale_row;
  }
  const int64_t r = (int64_t)t.row0 + min(t.m0 + m, t.cnt - 1);
  const uint8_t *const xc = a.xc + r * code_row + g * 16, *const xs = a.xs + r * scale_row;
  const int steps = (a.in_feat + kMxStep - 1) / kMxStep, groups = (steps + 3) / 4;
  const int g1 = (wave + 1) * groups / kWaves;
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  for (int q = wave * groups / kWaves; q < g1; ++q) {
    const i32x4 xsv = *(const i32x4*)(xs + q * 16);
    i32x4 wsv[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) wsv[f] = *(const i32x4*)(ws[f] + q * 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (q * 4 + s >= steps) break;
      const int64_t off = (int64_t)(q * 4 + s) * 64;
      const i32x4 x = *(const i32x4*)(xc + off);
#pragma unroll
      for (int f = 0; f < 2; ++f)
        acc[f] = mx_mfma(*(const i32x4*)(wc[f] + off), (int)((uint32_t)wsv[f][s] >> (8 * g)), x,
                         (int)((uint32_t)xsv[s] >> (8 * g)), acc[f]);
    }
  }
  // the quarters meet in the first wave, always in the same order
  if (wave > 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[((wave - 1) * 8 + j) * kWave + lane] = acc[j >> 2][j & 3];
  }
  __syncthreads();
  if (wave > 0) return;
  float b[8], y[8];
  mx_load_bias(a, mx_bias_rows(a, t.e), base + 8 * g, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    y[j] = acc[j >> 2][j & 3];
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) y[j] += part[(w * 8 + j) * kWave + lane];
    y[j] += b[j];
  }
  const MxOutput<T, MODE> out(a, (int64_t)t.row0 + t.m0, min(16, t.cnt - t.m0));
  out.store(m, base + 8 * g, y);
}

template <typename T, int TN, int TM, int MODE>
__global__ __launch_bounds__(256, (QuantTile<false, TN, TM>::kGroups)) void mx_tile_kernel(
    QuantGemmArgs a) {
  quant_tiles<false, T, TN, TM, MODE>(a);
}

constexpr int kCus = 256;

// Which kernel: by the mean number of rows per expert, the features and the number of tiles this
// makes.  Measured with three sets of operands in turn (us; GELU and quantisation behind the
// products marked q), with even loads and, behind the slash, with half of all rows on one expert;
// two runs differ by up to 10 % below 100 us:
//   rows  experts  in -> out        stream     128x64   128x128  256x256
//    128   16    4096 -> 1024      11 / 13    12 / 12   14 / 14   27 / 27
//     64   16    1024 -> 4096      12 / 12    10 / 10   11 / 11   16 / 15
//    128    8    4096 -> 14336 q   68 / 85    54 / 51   60 / 62   91 / 90
//   4096   32    4096 -> 1024     114 / 118   18 / 26   18 / 25   29 / 29
//  15560  128    2048 -> 1408 q   338 / 280   78 / 75   62 / 78  102 / 130
//  30000   16    2048 -> 2048     727 / 725  110 / 109  80 / 79   74 / 74
//  32768    8    4096 -> 14336              1649 / 1661 1222 / 1231 917 / 959
//  16384    4    4096 -> 11008 q             696 / 706  510 / 526  495 / 515
//  32768    8    4096 -> 14336 q            1806 / 1825 1326 / 1384 1235 / 1272
// The mean stands for both: what it picks is within 5 % of the best under these uneven loads too.
// Few rows and few tiles: the kernel that splits K.  The largest tiles move the least through L2
// and win where K is long and there are rounds enough of them; smaller ones share a CU by two, so
// that one's beginning and end (with GELU, half its time) are the other's middle.
enum MxKernel { kStream, kTile128x64, kTile128x128, kTile256x256 };
static MxKernel choose_kernel(const QuantGemmArgs& a) {
  const double live = (double)std::min<int64_t>(a.n_expert, a.n_rows);
  const double mean = (double)a.n_rows / a.n_expert;
  // (an expert's last tile is half empty on average)
  auto tiles = [&](int tn, int tm) {
    return std::max((double)a.n_rows / tm + live / 2, live) * ceil_div(a.out_feat, tn);
  };
  if (mean <= 16 && tiles(128, 64) <= kCus / 2) return kStream;
  if (mean < 56) return kTile128x64;
  const bool quant = a.yc != nullptr;
  if (mean >= 192 && a.in_feat >= (quant ? 4096 : 2048) && tiles(256, 256) >= (quant ? 4000 : 600))
    return kTile256x256;
  return kTile128x128;
}

template <typename T, int MODE>
static int launch(const QuantGemmArgs& a, hipStream_t s) {
  const int n_pad = mx_quantises(MODE) ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
#define FMOE_TILE(TN, TM)                                                                        \
  do {                                                                                           \
    const int64_t rows = a.n_rows / TM + std::min<int64_t>(a.n_expert, a.n_rows);                \
    FMOE_REQUIRE(rows * ceil_div(n_pad, TN) <= INT32_MAX, FMOE_ERR_UNSUPPORTED,                  \
                 "mx_linear: too many tiles");                                                   \
    FMOE_SET_DYNAMIC_LDS_ONCE((mx_tile_kernel<T, TN, TM, MODE>), (QuantTile<false, TN, TM>::kLdsBytes)); \
    hipLaunchKernelGGL((mx_tile_kernel<T, TN, TM, MODE>), dim3(kCus * QuantTile<false, TN, TM>::kGroups),  \
                       dim3(256), (QuantTile<false, TN, TM>::kLdsBytes), s, a);                            \
  } while (0)
  switch (choose_kernel(a)) {
    case kStream: {
      const int64_t rows = a.n_rows / 16 + std::min<int64_t>(a.n_expert, a.n_rows);
      hipLaunchKernelGGL((mx_stream_kernel<T, MODE>), dim3((unsigned)(rows * ceil_div(n_pad, 32))),
                         dim3(256), 0, s, a);      // (few tiles, or this kernel is not chosen)
      break;
    }
    case kTile128x64: FMOE_TILE(128, 64); break;
    case kTile128x128: FMOE_TILE(128, 128); break;
    case kTile256x256: FMOE_TILE(256, 256); break;
  }
#undef FMOE_TILE
  FMOE_LAUNCH_CHECK("mx_linear");
  return FMOE_OK;
}

template <typename T> static int launch_y(const QuantGemmArgs& a, hipStream_t s) {
  constexpr int kN = Pack16<T>::kN;
  return a.out_feat % kN == 0 && (uintptr_t)a.y % 16 == 0 ? launch<T, kMxPacked>(a, s)
                                                          : launch<T, kMxAny>(a, s);
}

}  // namespace fmoe

extern "C" int fmoe_mx_linear_fwd(const void* x_codes, const void* x_scales, const void* w_codes,
                                  const void* w_scales, const void* bias, const int32_t* seg_off,
                                  int act, void* y, void* y_codes, void* y_scales, int64_t n_rows,
                                  int64_t in_feat, int64_t out_feat, int64_t n_expert, int dtype,
                                  void* stream) {
  using namespace fmoe;
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && n_expert >= 1 && n_expert < INT32_MAX &&
                   in_feat >= 1 && out_feat >= 1 && in_feat <= FMOE_MX_MAX_FEATURES &&
                   out_feat <= FMOE_MX_MAX_FEATURES,
               FMOE_ERR_INVALID, "mx_linear: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "mx_linear: unsupported dtype %d", dtype);
  FMOE_REQUIRE(act == FMOE_ACT_NONE || act == FMOE_ACT_GELU || act == FMOE_ACT_RELU,
               FMOE_ERR_INVALID, "mx_linear: unknown activation %d", act);
  FMOE_REQUIRE(act == FMOE_ACT_NONE || y == nullptr, FMOE_ERR_INVALID,
               "mx_linear: an activation only in front of y_codes");
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(x_codes && x_scales && w_codes && w_scales && seg_off, FMOE_ERR_INVALID,
               "mx_linear: null pointer");
  FMOE_REQUIRE((y != nullptr) != (y_codes != nullptr) && (y_codes != nullptr) == (y_scales != nullptr),
               FMOE_ERR_INVALID, "mx_linear: either y, or y_codes and y_scales");
  FMOE_REQUIRE(((uintptr_t)x_codes | (uintptr_t)x_scales | (uintptr_t)w_codes |
                (uintptr_t)w_scales | (uintptr_t)y_codes | (uintptr_t)y_scales) % 16 == 0,
               FMOE_ERR_INVALID, "mx_linear: codes and scales must be 16-byte aligned");
  const QuantGemmArgs a{(const uint8_t*)x_codes, (const uint8_t*)x_scales, (const uint8_t*)w_codes,
                     (const uint8_t*)w_scales, bias, seg_off, y, (uint8_t*)y_codes,
                     (uint8_t*)y_scales, n_rows, (int)in_feat, (int)out_feat, (int)n_expert, dtype};
  hipStream_t s = (hipStream_t)stream;
  if (y_codes)      // (the element type then is that of the bias alone, which is read as it comes)
    return act == FMOE_ACT_GELU   ? launch<float, kMxQuantGelu>(a, s)
           : act == FMOE_ACT_RELU ? launch<float, kMxQuantRelu>(a, s)
                                  : launch<float, kMxQuant>(a, s);
  switch (dtype) {
    case FMOE_F32: return launch_y<float>(a, s);
    case FMOE_F16: return launch_y<__half>(a, s);
    default: return launch_y<__hip_bfloat16>(a, s);
  }
}
