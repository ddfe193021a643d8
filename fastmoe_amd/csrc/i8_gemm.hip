// Grouped product of 8-bit rows with 8-bit expert weights on gfx950 (the format: i8.h):
//   y[r][n] = sx[r] sw_e[n] sum_k qx[r][k] qw_e[n][k] + b_e[n],   r in the rows of expert e.
//
// v_mfma_i32_16x16x64_i8 multiplies 16 rows of 64 codes by 16 rows of 64 codes and adds to 32-bit
// integers, which hold every sum exactly (in_feat <= 2^17).  Its operands are 16 bytes a lane like
// those of the 4-bit product and its result lies like that one's, so that both products run in the
// same tiles (quant_gemm.h), features as rows of the result.
//
// Few rows are bound by the weights' bytes (one each), many by the matrix cores; which of two
// kernels and three tile shapes runs: choose_kernel().  Measured: 32768 rows of 8 experts,
// 4096 -> 14336, in bf16 1418 us, 2.72 PFLOP/s (the library's product of 16384^3 in 8-bit integers:
// 2.44); 128 rows of these 89 us, 470 MB at 5.3 TB/s.
#include <algorithm>

#include "quant_gemm.h"

namespace fmoe {

// ------------------------------------------------------------------------- few rows
// Weights straight from memory into registers, since nothing would read them twice: a workgroup's
// 4 waves take 16 rows of an expert, 32 features, and a quarter of K each, whose sums meet in LDS.
// K is split because there are few tiles otherwise: 128 rows of 16 experts, 4096 -> 1024, are 512
// workgroups and take 17.5 us (67 MB at 3.8 TB/s) where 128 x 64 tiles take 28.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void i8_stream_kernel(QuantGemmArgs a) {
  constexpr int kWaves = 4, kCols = 32;
  __shared__ int s_sum[2 * kWaves], s_out[4];
  __shared__ int part[(kWaves - 1) * 8 * kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowTiles<16, kOneHeight, kWaves> tiles;
  tiles.scan(a.seg_off, a.n_expert, s_sum);
  const int n_cols = (a.out_feat + kCols - 1) / kCols;
  if (tiles.rows_f == 0) return;
  const int col = blockIdx.x / tiles.rows_f, v = blockIdx.x - col * tiles.rows_f;
  if (col >= n_cols) return;
  const TileRows t = tiles.find(a.seg_off, v, false, s_out);

  const int m = lane & 15, g = lane >> 4, base = col * kCols;
  const int64_t row_bytes = i8_row_bytes(a.in_feat);
  // rows and features past the end repeat the last one; their results are not stored
  const uint8_t* wc[2];
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const int64_t n = (int64_t)t.e * a.out_feat + min(base + mx_feature(f, m), a.out_feat - 1);
    wc[f] = a.wc + n * row_bytes + g * 16;
  }
  const int64_t r = (int64_t)t.row0 + min(t.m0 + m, t.cnt - 1);
  const uint8_t* const xc = a.xc + r * row_bytes + g * 16;
  const int pairs = (int)(row_bytes / kI8Step), p1 = (wave + 1) * pairs / kWaves;
  i32x4 acc[2] = {i32x4{0, 0, 0, 0}, i32x4{0, 0, 0, 0}};
  for (int p = wave * pairs / kWaves; p < p1; p += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (p + u >= p1) break;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int64_t off = (int64_t)(p + u) * kI8Step + s * 64;
        const i32x4 x = *(const i32x4*)(xc + off);
#pragma unroll
        for (int f = 0; f < 2; ++f)
          acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(wc[f] + off), x, acc[f], 0, 0, 0);
      }
    }
  }
  // the quarters meet in the first wave (as integers, in any order)
  if (wave > 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[((wave - 1) * 8 + j) * kWave + lane] = acc[j >> 2][j & 3];
  }
  __syncthreads();
  if (wave > 0) return;
  const float* const sw = (const float*)a.ws + (int64_t)t.e * a.out_feat;
  const float sx = ((const float*)a.xs)[r];
  float b[8], y[8];
  mx_load_bias(a, mx_bias_rows(a, t.e), base + 8 * g, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int sum = acc[j >> 2][j & 3];
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) sum += part[(w * 8 + j) * kWave + lane];
    y[j] = fmaf((float)sum * sx, sw[min(base + 8 * g + j, a.out_feat - 1)], b[j]);
  }
  const MxOutput<T, MODE> out(a, (int64_t)t.row0 + t.m0, min(16, t.cnt - t.m0));
  out.store(m, base + 8 * g, y);
}

// ------------------------------------------------------------------------- many rows
template <typename T, int TN, int TM, int MODE>
__global__ __launch_bounds__(256, (QuantTile<true, TN, TM>::kGroups)) void i8_tile_kernel(
    QuantGemmArgs a) {
  quant_tiles<true, T, TN, TM, MODE>(a);
}

constexpr int kCus = 256;

// Which kernel: by the mean number of rows per expert, the features and the number of tiles this
// makes.  Measured with several sets of operands in turn (us, bf16), with even loads, which fill the
// tiles (a routed batch's do not: 71.1 below is 95 there, 86.5 is 100), and, behind the slash, with half
// of all rows on one expert:
//   rows  experts  in -> out      stream       128x64       128x128      256x256
//     64   16    1024 -> 4096   16.6 / 17.0  16.5 / 16.2  17.0 / 16.9  21.8 / 21.0
//    128   16    4096 -> 1024   17.5 / 20.5  27.7 / 27.7  28.4 / 28.5  41.4 / 41.6
//      8    1    4096 -> 14336  16.6         27.2         27.7         41.4
//    128    8    4096 -> 14336   106 / 130   89.4 / 87.5  91.1 / 95.5   102 / 99.1
//    512    8    1024 -> 4096   28.0 / 29.8   9.3 / 11.4  10.3 / 12.1  17.4 / 17.0
//   2048   32    2048 -> 1408   67.4 / 77.4  23.6 / 32.8  24.9 / 24.8  28.5 / 30.0
//   4096   32    4096 -> 1024                41.8 / 56.8  40.8 / 43.8  47.9 / 47.6
//  16376  128    2048 -> 1408                 104 / 114   86.5 / 107   92.0 / 115
//    512    1    2048 -> 5632                13.3         12.8         24.0
//   2047    1    2048 -> 5632                34.6         28.7         27.6
//   8192    8     512 -> 2048                20.4 / 21.9  15.2 / 17.6  16.0 / 25.0
//  16384   16    1024 -> 4096                 109 / 108   79.9 / 86.1  71.1 / 84.1
//   8192    2    8192 -> 2048                 193 / 193    131 / 132   98.4 / 98.0
//  32768    8    4096 -> 14336               2494 / 2515  1844 / 1836  1418 / 1483
// Few rows and few tiles: the kernel that splits K.  Many rows: a 256 x 256 tile costs 1.46 times a
// round of two 128 x 128 ones on a CU for twice their work, so that it wins where K is long enough for
// its end not to matter and the chip's rounds are as full with it.
enum I8Kernel { kStream, kTile128x64, kTile128x128, kTile256x256 };
static I8Kernel choose_kernel(const QuantGemmArgs& a) {
  const double live = (double)std::min<int64_t>(a.n_expert, a.n_rows);
  const double mean = (double)a.n_rows / a.n_expert;
  // (of several experts the last tile is half empty on average)
  auto tiles = [&](int tn, int tm) {
    const double rows = live == 1 ? ceil_div(a.n_rows, tm) : (double)a.n_rows / tm + live / 2;
    return std::max(rows, live) * ceil_div(a.out_feat, tn);
  };
  if (mean <= 16 && tiles(128, 64) <= kCus / 2) return kStream;
  if (mean < 56) return kTile128x64;
  if (mean >= 192 && a.in_feat >= 1024 &&
      std::max(tiles(256, 256) / kCus, 1.) <= 0.73 * std::max(tiles(128, 128) / (2 * kCus), 1.))
    return kTile256x256;
  return kTile128x128;
}

template <typename T, int MODE>
static int launch(const QuantGemmArgs& a, hipStream_t s) {
#define FMOE_TILE(TN, TM)                                                                        \
  do {                                                                                           \
    using S = QuantTile<true, TN, TM>;                                                           \
    const int64_t rows = a.n_rows / TM + std::min<int64_t>(a.n_expert, a.n_rows);                \
    FMOE_REQUIRE(rows * ceil_div(a.out_feat, TN) <= INT32_MAX, FMOE_ERR_UNSUPPORTED,             \
                 "i8_linear: too many tiles");                                                   \
    FMOE_SET_DYNAMIC_LDS_ONCE((i8_tile_kernel<T, TN, TM, MODE>), S::kLdsBytes);                  \
    hipLaunchKernelGGL((i8_tile_kernel<T, TN, TM, MODE>), dim3(kCus * S::kGroups), dim3(256),    \
                       S::kLdsBytes, s, a);                                                      \
  } while (0)
  switch (choose_kernel(a)) {
    case kStream: {
      const int64_t rows = a.n_rows / 16 + std::min<int64_t>(a.n_expert, a.n_rows);
      hipLaunchKernelGGL((i8_stream_kernel<T, MODE>),
                         dim3((unsigned)(rows * ceil_div(a.out_feat, 32))), dim3(256), 0, s,
                         a);      // (few tiles, or this kernel is not chosen)
      break;
    }
    case kTile128x64: FMOE_TILE(128, 64); break;
    case kTile128x128: FMOE_TILE(128, 128); break;
    case kTile256x256: FMOE_TILE(256, 256); break;
  }
#undef FMOE_TILE
  FMOE_LAUNCH_CHECK("i8_linear");
  return FMOE_OK;
}

template <typename T> static int launch_y(const QuantGemmArgs& a, hipStream_t s) {
  constexpr int kN = Pack16<T>::kN;
  return a.out_feat % kN == 0 && (uintptr_t)a.y % 16 == 0 ? launch<T, kMxPacked>(a, s)
                                                          : launch<T, kMxAny>(a, s);
}

}  // namespace fmoe

extern "C" int fmoe_i8_linear_fwd(const void* x_codes, const float* x_scales, const void* w_codes,
                                  const float* w_scales, const void* bias, const int32_t* seg_off,
                                  void* y, int64_t n_rows, int64_t in_feat, int64_t out_feat,
                                  int64_t n_expert, int dtype, void* stream) {
  using namespace fmoe;
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && n_expert >= 1 && n_expert < INT32_MAX &&
                   in_feat >= 1 && out_feat >= 1 && in_feat <= FMOE_I8_MAX_FEATURES &&
                   out_feat <= FMOE_I8_MAX_FEATURES,
               FMOE_ERR_INVALID, "i8_linear: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "i8_linear: unsupported dtype %d", dtype);
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(x_codes && x_scales && w_codes && w_scales && seg_off && y, FMOE_ERR_INVALID,
               "i8_linear: null pointer");
  FMOE_REQUIRE(((uintptr_t)x_codes | (uintptr_t)w_codes) % 16 == 0, FMOE_ERR_INVALID,
               "i8_linear: codes must be 16-byte aligned");
  FMOE_REQUIRE(((uintptr_t)x_scales | (uintptr_t)w_scales) % 4 == 0, FMOE_ERR_INVALID,
               "i8_linear: scales must be aligned floats");
  const QuantGemmArgs a{(const uint8_t*)x_codes, (const uint8_t*)x_scales, (const uint8_t*)w_codes,
                        (const uint8_t*)w_scales, bias, seg_off, y, nullptr, nullptr, n_rows,
                        (int)in_feat, (int)out_feat, (int)n_expert, dtype};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FMOE_F32: return launch_y<float>(a, s);
    case FMOE_F16: return launch_y<__half>(a, s);
    default: return launch_y<__hip_bfloat16>(a, s);
  }
}
