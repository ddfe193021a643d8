// The gradient of an 8-bit product's rows:
//   dx[r][k] = sum_n dy[r][n] s_e[n] q_e[n][k],   r in the rows of expert e
// straight from the codes, for few rows and for f32.  (Many 16-bit rows go through weights laid out in
// their type and the other products' backward, which costs 5 bytes of traffic per weight whatever the
// rows; here it is one per 32 or 64 rows of an expert.)
//
// The sum runs over the codes' rows, so that v_mfma_f32_16x16x32_bf16 needs 8 rows' codes of one
// feature in a lane, where memory has 8 features of one row.  A lane loads 8 bytes of 8 rows, and
// byte j of these is its part of the j-th of eight fragments: integers up to 127 are exact in bf16,
// one conversion each and a byte permutation for two.  Codes are the first operand, lane m holding
// features 8 m .. 8 m + 7, so that a result fragment's row i of lane group g is feature
// 8 (4 g + i) + j.
//
// The scales are on the summed axis and go into the other operand: dy s in f32, as a sum of bf16
// numbers, two (relative error 2^-17) for 16-bit rows and three for f32, each with a product of its
// own.  The result is then off by its own rounding alone.
#include <algorithm>

#include "gemm_tiles.h"
#include "i8.h"
#include "rows.h"

namespace fmoe {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kGradWaves = 8;          // share the summed axis
constexpr int kGradCols = 128;         // features: 8 fragments
static_assert(kGradCols == kI8Step, "rows of codes are whole column tiles");

// Mean rows per expert up to which this is the faster way in 16 bits; in f32, whose product by weights
// laid out has a sixteenth of their rate, it always is.  Microseconds here and by weights laid out:
//   rows  experts  in -> out        bf16          f32
//     64   16    1024 -> 4096      20 /  67     22 /  172
//   1024   16    1024 -> 4096      40 /  65     51 /  178
//   2048   16    1024 -> 4096      60 /  70     98 /  220
//   4096   16    1024 -> 4096     113 /  81    200 /  339
//   2048  128    2048 -> 1408     117 / 338    132 /  827
//   8192  128    2048 -> 1408     223 / 347    336 /  838
//  16384  128    2048 -> 1408     410 / 364    638 / 1165
//     16    1    4096 -> 14336     21 / 125     23 /  350
//    128    8    4096 -> 14336     97 / 444    107 / 1080
//    768    8    4096 -> 14336    324 / 444    435 / 1497
// (469 MB at 4.8 TB/s in the last but one; with more rows the split of dy and the conversions, 70 and
// 96 instructions per 16 and 64 rows in a step of 4 KiB, set the time.)
constexpr int64_t kGradFewRows = 96;
constexpr int64_t kGradBlocks = 256;   // one on a CU

struct I8GradArgs {
  const void* dy;
  const uint8_t* wc;
  const float* ws;
  const int32_t* seg_off;
  void* dx;
  float* shares;              // [gridDim.y][n_rows][in_feat], or null where gridDim.y is 1
  int64_t n_rows;
  int in_feat, out_feat, n_expert;
};

__device__ __forceinline__ uint32_t bf16_bits(float v) {
  return __builtin_bit_cast(uint16_t, __float2bfloat16(v));
}

// 8 numbers as PARTS bf16 fragments whose sum they are.
template <int PARTS>
__device__ __forceinline__ void split_bf16(float (&v)[8], u32x4 (&out)[PARTS]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = __builtin_elementwise_maximum(top, __builtin_fabsf(v[i]));
  // (what rounds to an infinity, which less itself would be a NaN: one number is enough then)
  const bool huge = !(top < 0x1.ffp127f);
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      b[i] = bf16_bits(v[i]);
      v[i] -= __uint_as_float(b[i] << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) out[p][i] = p > 0 && huge ? 0u : b[2 * i] | b[2 * i + 1] << 16;
  }
}

// 4 of a row's values from k on, of which it has d.
template <typename T>
__device__ __forceinline__ void store_four(T* to, int k, int d, const float (&v)[4]) {
  T o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = Elem<T>::from_acc(v[j]);
  if (k + 4 <= d) {
    __builtin_memcpy(to, o, sizeof(o));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k + j < d) to[j] = o[j];
  }
}

// A block takes 16 F rows of an expert.
template <typename T, int F>
__global__ __launch_bounds__(kGradWaves* kWave) void i8_grad_kernel(I8GradArgs a, ClearedTail<T> tail) {
  constexpr int kParts = sizeof(T) == 4 ? 3 : 2;
  __shared__ float part[kGradWaves][32][kWave];
  if (blockIdx.y == 0) tail.clear(a.in_feat);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  RowTiles<16 * F, kOneHeight, kGradWaves> tiles;
  int* const s_find = (int*)part;
  tiles.scan(a.seg_off, a.n_expert, s_find);
  const int row_bytes = (int)i8_row_bytes(a.in_feat), n_cols = row_bytes / kGradCols;
  if (tiles.rows_f == 0) return;
  const int col = blockIdx.x / tiles.rows_f, v = blockIdx.x - col * tiles.rows_f;
  if (col >= n_cols) return;
  const TileRows t = tiles.find(a.seg_off, v, false, s_find + 2 * kGradWaves);
  if (!tiles.by_lane) __syncthreads();     // (before that place holds anything else)

  const int m = lane & 15, g = lane >> 4;
  const int rows = min(16 * F, t.cnt - t.m0);
  const T* const dy = (const T*)a.dy + ((int64_t)t.row0 + t.m0) * a.out_feat;
  const float* const scale = a.ws + (int64_t)t.e * a.out_feat;
  const uint8_t* const w = a.wc + (int64_t)t.e * a.out_feat * row_bytes + col * kGradCols + m * 8;
  // the summed axis is dealt to the waves of gridDim.y blocks
  const int steps = (a.out_feat + 31) / 32;
  const int deal = (int)gridDim.y * kGradWaves, at = (int)blockIdx.y * kGradWaves + wave;
  const int s1 = (int)((int64_t)(at + 1) * steps / deal);
  f32x4 acc[F][8];
#pragma unroll
  for (int h = 0; h < F; ++h)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int frags = (rows + 15) / 16;      // that hold rows
  // what a step reads: codes of rows 32 s + 8 g .. + 7 (behind the last: that one's, which meet
  // zeros), these rows' scales and values of dy (rows of dy behind the last repeat it; their results
  // are not stored)
  struct Step {
    uint2 code[8];
    Eight<float> scale;
    Eight<T> dy[F];
  };
  auto fetch = [&](int s, Step& to) {
    const int n = s * 32 + g * 8;
    to.scale.load(scale, n, a.out_feat);
#pragma unroll
    for (int h = 0; h < F; ++h)
      if (h < frags)
        to.dy[h].load(dy + (int64_t)min(h * 16 + m, rows - 1) * a.out_feat, n, a.out_feat);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      to.code[i] = *reinterpret_cast<const uint2*>(w + (int64_t)min(n + i, a.out_feat - 1) * row_bytes);
  };
  int s = (int)((int64_t)at * steps / deal);
  Step now, next;
  if (s < s1) fetch(s, now);
  for (; s < s1; ++s) {
    if (s + 1 < s1) fetch(s + 1, next);
    u32x4 q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = j < 4 ? now.code[2 * i].x : now.code[2 * i].y;
        const uint32_t hi = j < 4 ? now.code[2 * i + 1].x : now.code[2 * i + 1].y;
        const float x = (float)(int8_t)(lo >> (8 * (j & 3))), y = (float)(int8_t)(hi >> (8 * (j & 3)));
        q[j][i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
      }
#pragma unroll
    for (int h = 0; h < F; ++h) {
      if (h >= frags) break;
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = now.dy[h][i] * now.scale[i];
      u32x4 b[kParts];
      split_bf16<kParts>(p, b);
#pragma unroll
      for (int u = 0; u < kParts; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[h][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, q[j]), __builtin_bit_cast(bf16x8, b[u]), acc[h][j], 0, 0, 0);
    }
    now = next;
  }
  // The waves' shares meet in LDS, 16 rows at a time, in the order of the waves: wave u adds up
  // features 8 (4 g + u / 2) + 4 (u % 2) .. + 3 of lane group g.
  const int i0 = wave >> 1, j0 = 4 * (wave & 1);
#pragma unroll
  for (int h = 0; h < F; ++h) {
    if (h >= frags) break;
    if (h > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[wave][i * 8 + j][lane] = acc[h][j][i];
    __syncthreads();
    const int r = h * 16 + m, k = col * kGradCols + 8 * (4 * g + i0) + j0;
    float sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum[j] = 0.f;
#pragma unroll
      for (int u = 0; u < kGradWaves; ++u) sum[j] += part[u][i0 * 8 + j0 + j][lane];
    }
    if (r >= rows) continue;
    const int64_t to = ((int64_t)t.row0 + t.m0 + r) * a.in_feat + k;
    if (a.shares) store_four(a.shares + blockIdx.y * a.n_rows * a.in_feat + to, k, a.in_feat, sum);
    else store_four((T*)a.dx + to, k, a.in_feat, sum);
  }
}

// dx = the sum of `n` shares, in order, of the rows that an expert owns.
template <typename T>
__global__ __launch_bounds__(256) void i8_grad_sum_kernel(const float* __restrict__ shares, int n,
                                                          int64_t size, const int32_t* __restrict__ end,
                                                          int k, T* __restrict__ dx) {
  const int64_t live = min(size, (int64_t)max(*end, 0) * k);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < live; i += (int64_t)gridDim.x * 256) {
    float sum = 0.f;
    for (int u = 0; u < n; ++u) sum += shares[u * size + i];
    dx[i] = Elem<T>::from_acc(sum);
  }
}

// Fragments of 16 rows in a block, and blocks that share the summed axis: so many that there are enough for the chip's memory, while a
// wave keeps two steps.  (4096 -> 14336 for 16 rows of one expert, 32 column tiles: 89 us in one
// block each, 21 in eight.)
struct GradShape {
  int frags, shares;
  GradShape(int64_t n_rows, int64_t in_feat, int64_t out_feat, int64_t n_expert, int dtype) {
    const int64_t live = std::min(n_expert, n_rows), cols = i8_row_bytes(in_feat) / kGradCols;
    auto tiles = [&](int f) { return std::max(n_rows / (16 * f) + live / 2, live) * cols; };
    // Four fragments halve the conversions (384 rows of 8 experts, 4096 -> 14336: 219 -> 157 us),
    // but leave CUs without a block where there were just enough (1024 of 16, 1024 -> 4096: 40 -> 53);
    // f32's do not fit the registers.
    frags = 2;
    if (dtype != FMOE_F32 && n_rows > n_expert * 32 &&
        (tiles(4) >= kGradBlocks || tiles(4) <= kGradBlocks / 2))
      frags = 4;
    const int64_t steps = (out_feat + 31) / 32;
    shares = (int)std::max<int64_t>(
        std::min({kGradBlocks / tiles(frags), steps / (2 * kGradWaves), (int64_t)16}), 1);
  }
};

template <typename T>
static int launch_grad(const I8GradArgs& a, const GradShape& shape, hipStream_t s) {
  const int frags = shape.frags, shares = shape.shares;
  const int64_t rows = a.n_rows / (16 * frags) + std::min<int64_t>(a.n_expert, a.n_rows);
  const int64_t blocks = rows * (i8_row_bytes(a.in_feat) / kGradCols);
  FMOE_REQUIRE(blocks * (kGradWaves * kWave) <= UINT32_MAX, FMOE_ERR_UNSUPPORTED,
               "i8_linear_dx: too many tiles");
  const ClearedTail<T> tail{a.seg_off + a.n_expert, (T*)a.dx, a.n_rows};
  const dim3 grid((unsigned)blocks, shares), block(kGradWaves * kWave);
  if constexpr (sizeof(T) == 2) {
    if (frags == 4) hipLaunchKernelGGL((i8_grad_kernel<T, 4>), grid, block, 0, s, a, tail);
  }
  if (frags == 2) hipLaunchKernelGGL((i8_grad_kernel<T, 2>), grid, block, 0, s, a, tail);
  FMOE_LAUNCH_CHECK("i8_linear_dx");
  if (shares > 1) {
    const int64_t size = a.n_rows * a.in_feat;
    hipLaunchKernelGGL((i8_grad_sum_kernel<T>), dim3((unsigned)std::min<int64_t>((size + 255) / 256, 2048)),
                       dim3(256), 0, s, a.shares, shares, size, a.seg_off + a.n_expert, a.in_feat,
                       (T*)a.dx);
    FMOE_LAUNCH_CHECK("i8_linear_dx");
  }
  return FMOE_OK;
}

}  // namespace fmoe

extern "C" int fmoe_i8_few_rows(int64_t n_rows, int64_t n_expert, int dtype) {
  return dtype == FMOE_F32 || n_rows <= n_expert * fmoe::kGradFewRows;
}

extern "C" int64_t fmoe_i8_dx_workspace_bytes(int64_t n_rows, int64_t in_feat, int64_t out_feat,
                                              int64_t n_expert, int dtype) {
  using namespace fmoe;
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && n_expert >= 1 && n_expert < INT32_MAX &&
                   in_feat >= 1 && out_feat >= 1 && in_feat <= FMOE_I8_MAX_FEATURES &&
                   out_feat <= FMOE_I8_MAX_FEATURES,
               FMOE_ERR_INVALID, "i8_linear_dx: bad sizes");
  if (n_rows == 0) return 0;
  const int shares = GradShape(n_rows, in_feat, out_feat, n_expert, dtype).shares;
  return shares > 1 ? (int64_t)sizeof(float) * shares * n_rows * in_feat : 0;
}

extern "C" int fmoe_i8_linear_dx(const void* dy, const void* w_codes, const float* w_scales,
                                 const int32_t* seg_off, void* dx, int64_t n_rows, int64_t in_feat,
                                 int64_t out_feat, int64_t n_expert, void* workspace,
                                 int64_t workspace_bytes, int dtype, void* stream) {
  using namespace fmoe;
  const int64_t need = fmoe_i8_dx_workspace_bytes(n_rows, in_feat, out_feat, n_expert, dtype);
  if (need < 0) return (int)need;
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "i8_linear_dx: unsupported dtype %d", dtype);
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(dy && w_codes && w_scales && seg_off && dx, FMOE_ERR_INVALID,
               "i8_linear_dx: null pointer");
  FMOE_REQUIRE((uintptr_t)w_codes % 16 == 0 && (uintptr_t)w_scales % 4 == 0, FMOE_ERR_INVALID,
               "i8_linear_dx: codes must be 16-byte aligned, scales aligned floats");
  FMOE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
               FMOE_ERR_WORKSPACE, "i8_linear_dx: a workspace of %lld bytes, 16-byte aligned, is needed",
               (long long)need);
  const I8GradArgs a{dy, (const uint8_t*)w_codes, w_scales, seg_off, dx,
                     need ? (float*)workspace : nullptr, n_rows,
                     (int)in_feat, (int)out_feat, (int)n_expert};
  const GradShape shape(n_rows, in_feat, out_feat, n_expert, dtype);
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FMOE_F32: return launch_grad<float>(a, shape, s);
    case FMOE_F16: return launch_grad<__half>(a, shape, s);
    default: return launch_grad<__hip_bfloat16>(a, shape, s);
  }
}
