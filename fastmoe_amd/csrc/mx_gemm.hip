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
// is stored in 16-byte packs straight from the registers, and the block maximum of the quantising
// epilogue takes two exchanges.
#include <algorithm>

#include "act_math.h"
#include "gemm_tiles.h"
#include "mx.h"

namespace fmoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct MxGemmArgs {
  const uint8_t *xc, *xs, *wc, *ws;
  const void* bias;            // [E, out] or null
  const int32_t* seg_off;
  void* y;                     // [n_rows, out], or null with yc
  uint8_t *yc, *ys;            // rows of `out` features
  int64_t n_rows;
  int in_feat, out_feat, n_expert, act;
};

__device__ __forceinline__ f32x4 mx_mfma(i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
  const i32x8 a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 b8 = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  // 4 = E2M1 in either operand; the scale bytes are the lowest ones of sa and sb
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, sa, 0, sb);
}

// Feature, within its group of 32, of row m of fragment f.
__device__ __forceinline__ int mx_feature(int f, int m) { return 8 * (m >> 2) + 4 * f + (m & 3); }

// Bias, activation and output of 8 consecutive features n0 .. n0 + 7 of row `row` (if `live`).
// All lanes of a wave come here together; lanes l, l ^ 16, l ^ 32 and l ^ 48 hold one block.
template <typename T, bool QUANT>
__device__ __forceinline__ void mx_epilogue(const MxGemmArgs& a, int e, int64_t row, bool live,
                                            int n0, float (&v)[8]) {
  const int n = a.out_feat;
  if (a.bias) {
    const T* b = (const T*)a.bias + (int64_t)e * n;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n0 + i < n) v[i] += Elem<T>::to_acc(b[n0 + i]);
  }
  if (a.act == FMOE_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu_direct(v[i]);
  } else if (a.act == FMOE_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];   // (a NaN stays)
  }
  if (!QUANT) {
    if (!live) return;
    T* out = (T*)a.y + row * n + n0;
    constexpr int kN = Pack16<T>::kN;
    if (n % kN == 0 && n0 + 8 <= n && (uintptr_t)a.y % 16 == 0) {
#pragma unroll
      for (int p = 0; p < 8 / kN; ++p) {
        Pack16<T> o;
#pragma unroll
        for (int i = 0; i < kN; ++i) o.v[i] = Elem<T>::from_acc(v[p * kN + i]);
        *reinterpret_cast<Pack16<T>*>(out + p * kN) = o;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n0 + i < n) out[i] = Elem<T>::from_acc(v[i]);
    }
    return;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (n0 + i >= n) v[i] = 0.f;
    m = max(m, magnitude_bits(v[i]));
  }
  m = max(m, (uint32_t)__shfl_xor((int)m, 16, kWave));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, kWave));
  const int byte = mx_scale_byte(m);
  const uint32_t word = mx_codes(v, byte);
  if (live && n0 < mx_code_bytes(n) * 2) {
    *reinterpret_cast<uint32_t*>(a.yc + row * mx_code_bytes(n) + n0 / 2) = word;
    if ((n0 & 31) == 0) a.ys[row * mx_scale_bytes(n) + n0 / kMxBlock] = (uint8_t)byte;
  }
}

// ------------------------------------------------------------------------- few rows
// Weights straight from memory into registers: a workgroup's 4 waves take 16 NT rows of an expert and
// 32 features each (KS == 1), or the same 32 features and a quarter of K each (KS == 4).
template <typename T, int NT, int KS, bool QUANT>
__global__ __launch_bounds__(256) void mx_stream_kernel(MxGemmArgs a) {
  constexpr int kWaves = 4, kCols = 32 * (kWaves / KS);
  __shared__ int s_sum[2 * kWaves], s_out[4];
  __shared__ float part[KS > 1 ? (KS - 1) * NT * 8 * kWave : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowTiles<16 * NT, kOneHeight, kWaves> tiles;
  tiles.scan(a.seg_off, a.n_expert, s_sum);
  const int n_pad = QUANT ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const int n_cols = (n_pad + kCols - 1) / kCols;
  if (tiles.rows_f == 0) return;
  const int col = blockIdx.x / tiles.rows_f, v = blockIdx.x - col * tiles.rows_f;
  if (col >= n_cols) return;
  const TileRows t = tiles.find(a.seg_off, v, false, s_out);

  const int m = lane & 15, g = lane >> 4;
  const int base = col * kCols + (KS == 1 ? wave * 32 : 0);
  const int64_t code_row = mx_code_bytes(a.in_feat), scale_row = mx_scale_bytes(a.in_feat);
  // rows and features past the end repeat the last one; their results are not stored
  const uint8_t *wc[2], *ws[2], *xc[NT], *xs[NT];
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const int64_t n = (int64_t)t.e * a.out_feat + min(base + mx_feature(f, m), a.out_feat - 1);
    wc[f] = a.wc + n * code_row + g * 16;
    ws[f] = a.ws + n * scale_row;
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int64_t r = t.row0 + min(t.m0 + i * 16 + m, t.cnt - 1);
    xc[i] = a.xc + r * code_row + g * 16;
    xs[i] = a.xs + r * scale_row;
  }
  const int steps = (a.in_feat + kMxStep - 1) / kMxStep, groups = (steps + 3) / 4;
  const int g0 = KS == 1 ? 0 : wave * groups / KS, g1 = KS == 1 ? groups : (wave + 1) * groups / KS;
  f32x4 acc[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int q = g0; q < g1; ++q) {
    i32x4 wsv[2], xsv[NT];
#pragma unroll
    for (int f = 0; f < 2; ++f) wsv[f] = *(const i32x4*)(ws[f] + q * 16);
#pragma unroll
    for (int i = 0; i < NT; ++i) xsv[i] = *(const i32x4*)(xs[i] + q * 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (q * 4 + s >= steps) break;
      const int64_t off = (int64_t)(q * 4 + s) * 64;
      i32x4 w[2], x[NT];
#pragma unroll
      for (int f = 0; f < 2; ++f) w[f] = *(const i32x4*)(wc[f] + off);
#pragma unroll
      for (int i = 0; i < NT; ++i) x[i] = *(const i32x4*)(xc[i] + off);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int f = 0; f < 2; ++f)
          acc[i][f] = mx_mfma(w[f], (int)((uint32_t)wsv[f][s] >> (8 * g)), x[i],
                              (int)((uint32_t)xsv[i][s] >> (8 * g)), acc[i][f]);
    }
  }
  if (KS > 1) {
    // the quarters meet in the first wave, always in the same order
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          part[(((wave - 1) * NT + i) * 8 + j) * kWave + lane] = acc[i][j >> 2][j & 3];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w2 = 0; w2 < KS - 1; ++w2)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[i][j >> 2][j & 3] += part[((w2 * NT + i) * 8 + j) * kWave + lane];
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = acc[i][j >> 2][j & 3];
    const int in_tile = t.m0 + i * 16 + m;
    mx_epilogue<T, QUANT>(a, t.e, t.row0 + in_tile, in_tile < t.cnt, base + 8 * g, r);
  }
}

template <typename T, bool QUANT>
static int launch(const MxGemmArgs& a, hipStream_t s) {
  const int n_pad = QUANT ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const double mean = (double)a.n_rows / a.n_expert;
#define FMOE_CALL(NT, KS)                                                                        \
  do {                                                                                           \
    const int64_t rows = a.n_rows / (16 * NT) + std::min<int64_t>(a.n_expert, a.n_rows);         \
    const int64_t blocks = rows * ceil_div(n_pad, 32 * (4 / KS));                                \
    FMOE_REQUIRE(blocks <= INT32_MAX, FMOE_ERR_UNSUPPORTED, "mx_linear: too many tiles");        \
    hipLaunchKernelGGL((mx_stream_kernel<T, NT, KS, QUANT>), dim3((unsigned)blocks), dim3(256), 0, \
                       s, a);                                                                    \
  } while (0)
  if (mean <= 16) FMOE_CALL(1, 4);
  else FMOE_CALL(4, 1);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("mx_linear");
  return FMOE_OK;
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
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(x_codes && x_scales && w_codes && w_scales && seg_off, FMOE_ERR_INVALID,
               "mx_linear: null pointer");
  FMOE_REQUIRE((y != nullptr) != (y_codes != nullptr) && (y_codes != nullptr) == (y_scales != nullptr),
               FMOE_ERR_INVALID, "mx_linear: either y, or y_codes and y_scales");
  FMOE_REQUIRE(((uintptr_t)x_codes | (uintptr_t)x_scales | (uintptr_t)w_codes |
                (uintptr_t)w_scales | (uintptr_t)y_codes | (uintptr_t)y_scales) % 16 == 0,
               FMOE_ERR_INVALID, "mx_linear: codes and scales must be 16-byte aligned");
  const MxGemmArgs a{(const uint8_t*)x_codes, (const uint8_t*)x_scales, (const uint8_t*)w_codes,
                     (const uint8_t*)w_scales, bias, seg_off, y, (uint8_t*)y_codes,
                     (uint8_t*)y_scales, n_rows, (int)in_feat, (int)out_feat, (int)n_expert, act};
  hipStream_t s = (hipStream_t)stream;
  const bool q = y_codes != nullptr;
  switch (dtype) {
    case FMOE_F32: return q ? launch<float, true>(a, s) : launch<float, false>(a, s);
    case FMOE_F16: return q ? launch<__half, true>(a, s) : launch<__half, false>(a, s);
    default: return q ? launch<__hip_bfloat16, true>(a, s) : launch<__hip_bfloat16, false>(a, s);
  }
}
