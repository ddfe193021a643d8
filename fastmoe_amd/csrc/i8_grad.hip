// The gradient of an 8-bit product's rows:
//   dx[r][k] = sum_n dy[r][n] s_e[n] q_e[n][k],   r in the rows of expert e
// straight from the codes, for few rows and for f32, and for many 16-bit rows by way of the other
// products' backward, which costs 5 bytes of traffic per weight whatever the rows; from the codes it
// is one per 32 or 64 rows of an expert.  Either way the result is off by its own rounding and hardly
// more: the error does not depend on which of the two runs.
//
// From the codes:
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
// own.
//
// Many rows: see "many rows" below.
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

// Mean rows per expert up to which the codes are the faster way in 16 bits, bf16 and f16 (whose product
// is twice as long); in f32, whose product has a sixteenth of their rate, they always are.  Microseconds
// from the codes and by the product, rows dealt to experts at random (f32: evenly, and weights laid out
// in f32):
//   rows  experts  in -> out         bf16           f16            f32
//   1024   16    1024 -> 4096      66 /   74      64 /  171      51 /  178
//   2048   16    1024 -> 4096     100 /   94      99 /  208      98 /  220
//   4096   16    1024 -> 4096     151 /  120     150 /  258     200 /  339
//  16384   16    1024 -> 4096     440 /  267     445 /  457
//  12288  128    2048 -> 1408     393 /  409     393 /  681
//  16384  128    2048 -> 1408     446 /  446     444 /  735     638 / 1165
//  32768  128    2048 -> 1408     808 /  590     810 /  969
//    128    1    2048 -> 5632      23 /   63      23 /  101
//   2048    1    2048 -> 5632     149 /   90     146 /  149
//    768    8    4096 -> 14336    321 /  469     321 /  814     435 / 1497
//   1536    8    4096 -> 14336    620 /  556     620 / 1018
//   4096    8    4096 -> 14336   1428 /  812    1427 / 1458
//  32768    8    4096 -> 14336  11638 / 3843   11699 / 7087
//   1536   16    4096 -> 1024      88 /   76      88 /  135
//   8192   16    4096 -> 1024     314 /  164     311 /  257
// (From the codes, few rows are bound by the codes' bytes: 128 of 8 experts, 4096 -> 14336, take 97 us,
// 469 MB at 4.8 TB/s; with more the split of dy and the conversions, 70 and 96 instructions per 16 and
// 64 rows in a step of 4 KiB, set the time.)
constexpr int64_t kGradFewRows = 96, kGradFewRowsF16 = 512;
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

// ------------------------------------------------------------------------- many rows
// The codes are exact in f16, too, so that the scales again go to the rows: v = dy s in f32, times a
// power of two u of the row's own, in f16; the f16 product of these with the codes' 128th parts; and
// its result times 128 / u.  With u the largest power of two for which sum |v| u < 2^15, no sum leaves
// f16's range (2^15 < 65504), and what v u loses to f16's smallest step is below 2^-39 of sum |v|.
//
// bf16: v u is rounded to f16 once (2^-11), the product's result once (2^-11), dx once (2^-8).  In mean
// squares the first two add 1 / 64 each to the last one's, and that, of numbers with 3 bits more, is
// 1 + 2 / 64: dx is off by sqrt(1 + 4 / 64) = 1.031 times its own rounding (8192 x top-2 rows, 1024 ->
// 4096: 0.00171 of the norm, 0.00166 for the rounding alone; weights rounded to bf16 gave 0.00235).
// f16: v u is a sum of two f16 numbers, behind one another along the summed axis, and the codes are
// laid out twice; the product's rounding is dx's own, as 128 / u is a power of two (a subnormal dx
// is rounded once more, to the steps there).
//
// A row with a v that is not finite keeps those alone, the finite ones being nothing beside them, and
// has u = 1: every element is an infinity or a NaN, as the formula has it.
//
// Both axes are padded to whole 16-byte packs with zeros, so that the product runs on the matrix cores
// whatever the features.
constexpr int kRowHeld = 4;            // chunks of a row in registers

// The power of two u for a row: sum of the magnitudes and the largest's bits, finite.
__device__ __forceinline__ int row_exponent(float sum, uint32_t top) {
  const uint32_t bits = __float_as_uint(sum);
  // (a sum that overflows: at most 2^17 magnitudes below twice the largest's power of two)
  const int e = bits < 0x7f800000u ? (int)(bits >> 23) - 127 : (int)(top >> 23) - 127 + 18;
  return min(max(14 - e, -120), 126);  // (so that 128 / u is a number; what is cut off needs no more)
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// parts[r] = v u of row r as PARTS f16 numbers, [PARTS][pitch], zeros behind the last feature; undo[r] =
// 128 / u.  A block of W waves takes a row.  (Two and four rows that share the scales: within 5 % of
// this either way.)
template <typename T, int PARTS, int W>
__global__ __launch_bounds__(W * kWave) void i8_scaled_rows_kernel(
    const T* __restrict__ dy, const float* __restrict__ scales, const int32_t* __restrict__ seg_off,
    int n_expert, int64_t n_rows, int out_feat, int pitch, __half* __restrict__ parts,
    float* __restrict__ undo) {
  constexpr int kSpan = W * kWave * 8;
  __shared__ float s_sum[2][W];
  __shared__ uint32_t s_top[2][W];
  const int at = threadIdx.x * 8;
  const int64_t live = min(n_rows, (int64_t)seg_off[n_expert]);
  int turn = 0;
  for (int64_t r = blockIdx.x; r < live; r += gridDim.x, turn ^= 1) {
    int lo = 0, hi = n_expert;         // the row's expert: seg_off[lo] <= r < seg_off[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (seg_off[mid] <= r) lo = mid;
      else hi = mid;
    }
    const T* const row = dy + r * out_feat;
    const float* const scale = scales + (int64_t)lo * out_feat;
    auto values = [&](int c, float (&v)[8]) {
      Eight<T> d;
      Eight<float> s;
      d.load(row, c + at, out_feat);
      s.load(scale, c + at, out_feat);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = d[i] * s[i];
    };
    float held[kRowHeld][8], sum = 0.f;
    uint32_t top = 0;
    auto count = [&](const float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum += __builtin_fabsf(v[i]);
        top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      }
    };
#pragma unroll
    for (int h = 0; h < kRowHeld; ++h) {
      if (h * kSpan >= out_feat) break;
      values(h * kSpan, held[h]);
      count(held[h]);
    }
    for (int c = kRowHeld * kSpan; c < out_feat; c += kSpan) {
      float v[8];
      values(c, v);
      count(v);
    }
    sum = wave_sum(sum);
    top = wave_max(top);
    if constexpr (W > 1) {
      if ((threadIdx.x & (kWave - 1)) == 0) {
        s_sum[turn][threadIdx.x / kWave] = sum;
        s_top[turn][threadIdx.x / kWave] = top;
      }
      __syncthreads();                 // (the turn after next is the first to write there again)
      sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        sum += s_sum[turn][w];
        top = max(top, s_top[turn][w]);
      }
    }
    const bool finite = top < 0x7f800000u;
    const int e = finite ? row_exponent(sum, top) : 0;
    const float unit = power_of_two(e);
    if (threadIdx.x == 0) undo[r] = power_of_two(7 - e);
    __half* const out = parts + r * PARTS * pitch;
    auto put = [&](int c, float (&v)[8]) {
      if (c + at >= pitch) return;
      float low[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool keep = finite || !(__builtin_fabsf(v[i]) < INFINITY);
        v[i] = keep ? v[i] * unit : 0.f;
        low[i] = finite ? v[i] - __half2float(__float2half(v[i])) : 0.f;
      }
      Eight<__half>::store(out, c + at, pitch, v);
      if constexpr (PARTS == 2) Eight<__half>::store(out + pitch, c + at, pitch, low);
    };
#pragma unroll
    for (int h = 0; h < kRowHeld; ++h) {
      if (h * kSpan >= out_feat) break;
      put(h * kSpan, held[h]);
    }
    for (int c = kRowHeld * kSpan; c < out_feat; c += kSpan) {
      float v[8];
      values(c, v);
      put(c, v);
    }
  }
}

// Chunks of 512 values of rows of k, numbered row by row: a wave takes U at a time, first
// `read(u, row, first value)` of all and then `write(u, row, first value)`, for a lane's 8.  I: what
// numbers the chunks.
template <int U, typename I, typename R, typename W>
__device__ __forceinline__ void for_chunks(I n_rows, int k, R&& read, W&& write) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int chunks = (k + kWave * 8 - 1) / (kWave * 8);
  const I items = n_rows * chunks, waves = (I)(blockDim.x / kWave * U);
  for (I it = blockIdx.x * waves + wave * U; it < items; it += gridDim.x * waves) {
    I row[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = (it + u) / (I)chunks;
      at[u] = it + u < items ? (int)(it + u - row[u] * chunks) * kWave * 8 + lane * 8 : k;
      if (at[u] < k) read(u, row[u], at[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at[u] < k) write(u, row[u], at[u]);
  }
}
constexpr int kChunksAtOnce = 4;
static unsigned chunk_blocks(int64_t n_rows, int k) {
  const int64_t items = n_rows * ((k + kWave * 8 - 1) / (kWave * 8)), block = 4 * kChunksAtOnce;
  return (unsigned)std::max<int64_t>(std::min<int64_t>((items + block - 1) / block, 256 * 64), 1);
}

// The 128th parts of the experts' codes (blockIdx.y), each expert's `copies` times: w [n_expert]
// [copies][rows][pitch], of whose rows the first out_feat are codes and the others zeros.
__global__ __launch_bounds__(256) void i8_codes_f16_kernel(const uint8_t* __restrict__ codes,
                                                           int out_feat, int rows, int in_feat,
                                                           int pitch, int copies,
                                                           __half* __restrict__ w) {
  const int64_t row_bytes = i8_row_bytes(in_feat);
  codes += (int64_t)blockIdx.y * out_feat * row_bytes;
  w += (int64_t)blockIdx.y * copies * rows * pitch;
  uint2 c[kChunksAtOnce];
  for_chunks<kChunksAtOnce>(
      (uint32_t)rows, pitch,
      [&](int u, uint32_t row, int k) {                // (codes reach to the next 128 features)
        c[u] = row < (uint32_t)out_feat ? *reinterpret_cast<const uint2*>(codes + row * row_bytes + k)
                                        : make_uint2(0, 0);
      },
      [&](int u, uint32_t row, int k) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = (float)(int8_t)((i < 4 ? c[u].x : c[u].y) >> (8 * (i & 3))) * 0x1p-7f;
        for (int j = 0; j < copies; ++j)
          Eight<__half>::store(w + ((int64_t)j * rows + row) * pitch, k, pitch, v);
      });
}

// dx[r] = undo[r] times row r of the f16 product (of `pitch` values; it may lie in dx's place); zeros
// from row *end on.
template <typename T>
__global__ __launch_bounds__(256) void i8_undo_kernel(const __half* product, int pitch,
                                                      const float* __restrict__ undo,
                                                      const int32_t* __restrict__ end, int64_t n_rows,
                                                      int in_feat, T* dx) {
  const int64_t live = *end;
  Eight<__half> in[kChunksAtOnce];
  float by[kChunksAtOnce];
  for_chunks<kChunksAtOnce>(
      n_rows, in_feat,
      [&](int u, int64_t row, int k) {
        if (row >= live) return;
        in[u].load(product + row * pitch, k, pitch);
        by[u] = undo[row];
      },
      [&](int u, int64_t row, int k) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = row < live ? in[u][i] * by[u] : 0.f;
        Eight<T>::store(dx + row * in_feat, k, in_feat, v);
      });
}

// What a call keeps in its workspace: the rows, the weights, a float a row and, where it does not fit in
// dx's place, the product.
struct ManyRows {
  int parts, rows, pitch;              // rows of the weights and their length, whole packs
  int64_t at_w, at_undo, at_product, bytes;
  ManyRows(int64_t n_rows, int64_t in_feat, int64_t out_feat, int64_t n_expert, int dtype) {
    parts = dtype == FMOE_F16 ? 2 : 1;
    rows = (int)(out_feat + 7) / 8 * 8;
    pitch = (int)(in_feat + 7) / 8 * 8;
    auto whole = [](int64_t b) { return (b + 255) / 256 * 256; };
    at_w = whole(2 * n_rows * parts * rows);
    at_undo = at_w + whole(2 * n_expert * parts * rows * pitch);
    at_product = at_undo + whole(4 * n_rows);
    bytes = at_product + (pitch == in_feat ? 0 : whole(2 * n_rows * pitch));
  }
};

template <typename T, int PARTS>
static int launch_many(const I8GradArgs& a, const ManyRows& m, char* work, hipStream_t s) {
  __half* const rows = (__half*)work;
  __half* const w = (__half*)(work + m.at_w);
  float* const undo = (float*)(work + m.at_undo);
  // (a lane reads the 8 values that it then writes)
  __half* const product = m.pitch == a.in_feat ? (__half*)a.dx : (__half*)(work + m.at_product);
  // (as many waves as hold a row, up to four; what is longer is read twice)
  auto scale_rows = [&](auto waves) {
    constexpr int W = decltype(waves)::value;
    const unsigned blocks = (unsigned)std::min<int64_t>(a.n_rows, 256 * 32 / W);
    hipLaunchKernelGGL((i8_scaled_rows_kernel<T, PARTS, W>), dim3(blocks), dim3(W * kWave), 0, s,
                       (const T*)a.dy, a.ws, a.seg_off, a.n_expert, a.n_rows, a.out_feat, m.rows, rows,
                       undo);
  };
  constexpr int kHeld = kWave * 8 * kRowHeld;
  if (a.out_feat <= kHeld) scale_rows(std::integral_constant<int, 1>{});
  else if (a.out_feat <= 2 * kHeld) scale_rows(std::integral_constant<int, 2>{});
  else scale_rows(std::integral_constant<int, 4>{});
  FMOE_LAUNCH_CHECK("i8_linear_dx_many");
  hipLaunchKernelGGL(i8_codes_f16_kernel, dim3(chunk_blocks(m.rows, m.pitch), a.n_expert), dim3(256), 0,
                     s, a.wc, a.out_feat, m.rows, a.in_feat, m.pitch, PARTS, w);
  FMOE_LAUNCH_CHECK("i8_linear_dx_many");
  const int rc = fmoe_grouped_linear_bwd(rows, rows, w, a.seg_off, product, nullptr, nullptr, a.n_rows,
                                         m.pitch, (int64_t)PARTS * m.rows, a.n_expert, FMOE_F16, s);
  if (rc) return rc;
  hipLaunchKernelGGL((i8_undo_kernel<T>), dim3(chunk_blocks(a.n_rows, a.in_feat)), dim3(256), 0, s,
                     product, m.pitch, undo, a.seg_off + a.n_expert, a.n_rows, a.in_feat, (T*)a.dx);
  FMOE_LAUNCH_CHECK("i8_linear_dx_many");
  return FMOE_OK;
}

}  // namespace fmoe

extern "C" int fmoe_i8_few_rows(int64_t n_rows, int64_t n_expert, int dtype) {
  return dtype == FMOE_F32 ||
         n_rows <= n_expert * (dtype == FMOE_F16 ? fmoe::kGradFewRowsF16 : fmoe::kGradFewRows);
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

extern "C" int64_t fmoe_i8_dx_many_workspace_bytes(int64_t n_rows, int64_t in_feat, int64_t out_feat,
                                                   int64_t n_expert, int dtype) {
  using namespace fmoe;
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && n_expert >= 1 && n_expert <= 65535 &&
                   in_feat >= 1 && out_feat >= 1 && in_feat <= FMOE_I8_MAX_FEATURES &&
                   out_feat <= FMOE_I8_MAX_FEATURES,
               FMOE_ERR_INVALID, "i8_linear_dx_many: bad sizes");
  return n_rows == 0 ? 0 : ManyRows(n_rows, in_feat, out_feat, n_expert, dtype).bytes;
}

extern "C" int fmoe_i8_linear_dx_many(const void* dy, const void* w_codes, const float* w_scales,
                                      const int32_t* seg_off, void* dx, int64_t n_rows,
                                      int64_t in_feat, int64_t out_feat, int64_t n_expert,
                                      void* workspace, int64_t workspace_bytes, int dtype,
                                      void* stream) {
  using namespace fmoe;
  const int64_t need = fmoe_i8_dx_many_workspace_bytes(n_rows, in_feat, out_feat, n_expert, dtype);
  if (need < 0) return (int)need;
  FMOE_REQUIRE(dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "i8_linear_dx_many: unsupported dtype %d", dtype);
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(dy && w_codes && w_scales && seg_off && dx, FMOE_ERR_INVALID,
               "i8_linear_dx_many: null pointer");
  FMOE_REQUIRE((uintptr_t)w_codes % 16 == 0 && (uintptr_t)w_scales % 4 == 0, FMOE_ERR_INVALID,
               "i8_linear_dx_many: codes must be 16-byte aligned, scales aligned floats");
  FMOE_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0,
               FMOE_ERR_WORKSPACE,
               "i8_linear_dx_many: a workspace of %lld bytes, 16-byte aligned, is needed",
               (long long)need);
  const I8GradArgs a{dy, (const uint8_t*)w_codes, w_scales, seg_off, dx, nullptr, n_rows,
                     (int)in_feat, (int)out_feat, (int)n_expert};
  const ManyRows m(n_rows, in_feat, out_feat, n_expert, dtype);
  hipStream_t s = (hipStream_t)stream;
  return dtype == FMOE_F16 ? launch_many<__half, 2>(a, m, (char*)workspace, s)
                           : launch_many<__hip_bfloat16, 1>(a, m, (char*)workspace, s);
}
