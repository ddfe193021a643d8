// Quantisation of rows to 8-bit integers and back on gfx950 (the format: i8.h).
//
// Both directions are bound by HBM: a value costs its own 2 or 4 bytes plus one.  The scale needs
// the whole row before the first code, so a wave, or four, keeps a row in registers between the two
// (up to 4096 or 16384 values; what is longer is read a second time, from L2 as a rule).
//
// A code is one multiply-add: t = x (127 / a) + 1.5 * 2^23 rounds the product to an integer whose
// low byte is the code.  That is wrong at most for products within 2^-15 of a half-way point (the
// quotient's error is 2^-24 of at most 127); a lane that holds one decides it exactly, by the sign
// of 127 |x| - (k + 1/2) a, whose terms have at most 19 bits for 16-bit x (32 for f32, where the
// sign is taken in f64).
#include <algorithm>

#include "i8.h"
#include "rows.h"

namespace fmoe {

constexpr int kI8Threads = 256;
constexpr int kI8Waves = kI8Threads / kWave;
constexpr int kI8Chunk = kWave * 8;          // values that a wave takes at once
constexpr int kI8Held = 8;                   // chunks of a row in a wave's registers

// What turns a row's values into codes.
struct I8Row {
  float unit;       // power of two that keeps everything below in range
  float top;        // the largest magnitude, times unit
  float inv;        // 127 / top
  float scale;      // 0 for a row of zeros, NaN for one that is not finite
  bool finite;

  __device__ __forceinline__ explicit I8Row(uint32_t top_bits) {
    finite = top_bits < 0x7f800000u;
    const float a = __uint_as_float(finite ? top_bits : 0u);
    unit = a < 0x1p-60f ? 0x1p64f : a > 0x1p60f ? 0x1p-64f : 1.f;
    top = a * unit;
    inv = top > 0.f ? 127.f / top : 0.f;
    scale = finite ? a / 127.f : __uint_as_float(0x7fc00000u);
  }
};

constexpr float kI8Magic = 12582912.f;       // 1.5 * 2^23: a float there has integers as its steps

// The codes of 8 values, v[0] in the lowest byte.  EXACT: f32 for 16-bit values, f64 for f32.
template <typename EXACT>
__device__ __forceinline__ uint2 i8_codes(const float (&v)[8], const I8Row& row) {
  float t[8], off = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = v[i] * row.unit;
    t[i] = fmaf(x, row.inv, kI8Magic);
    off = fmaxf(off, fabsf(fmaf(x, row.inv, kI8Magic - t[i])));
  }
  if (off > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = fabsf(v[i] * row.unit);
      const float k = floorf(x * row.inv);
      const EXACT side = fma(-((EXACT)k + (EXACT)0.5), (EXACT)row.top, (EXACT)127 * (EXACT)x);
      const bool odd = (int)k & 1;
      const float q = side > 0 || (side == 0 && odd) ? k + 1.f : k;
      t[i] = copysignf(q, v[i]) + kI8Magic;
    }
  }
  auto four = [&](int i) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[i + 1]), __float_as_uint(t[i]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[i + 3]), __float_as_uint(t[i + 2]), 0x04000c0cu);
    return lo | hi;
  };
  return row.finite ? make_uint2(four(0), four(4)) : make_uint2(0, 0);
}

__device__ __forceinline__ void i8_values(uint2 codes, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = (float)(int8_t)((i < 4 ? codes.x : codes.y) >> (8 * (i & 3))) * scale;
    // (an f32 product, always: left alone, the compiler makes it and a conversion to f16 one
    // instruction with one rounding, here and there)
    asm("" : "+v"(v[i]));
  }
}

// The largest magnitude's bits (NaN > infinity > numbers) among the waves of a row.
template <int W>
__device__ __forceinline__ uint32_t row_max(uint32_t m) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, kWave));
  if constexpr (W > 1) {
    __shared__ uint32_t part[W];
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) m = max(m, part[w]);
  }
  return m;
}

// inv == nullptr: row r goes to row r, and rows from *n_rows_dev on (if given) are skipped; else
// row t goes to the rows inv[t * top_k + j] that are not -1.  W waves take a row.
template <typename T, int N, int W>
__global__ __launch_bounds__(kI8Threads) void i8_quantize_kernel(
    const T* __restrict__ x, int64_t n_rows, int k, const int32_t* __restrict__ n_rows_dev,
    const int32_t* __restrict__ inv, int top_k, uint8_t* __restrict__ codes,
    float* __restrict__ scales, SegmentsOut segments) {
  static_assert(W == 1 || W == kI8Waves, "rows do not share a block's barrier");
  using Exact = std::conditional_t<sizeof(T) == 4, double, float>;
  if (segments.seg_off && blockIdx.x == 0 && threadIdx.x < kWave)
    write_segments(segments, n_rows, threadIdx.x);
  const int at = (threadIdx.x & (W * kWave - 1)) * 8;      // first value of the thread's in a chunk
  const int64_t r = (int64_t)blockIdx.x * (kI8Waves / W) + (W > 1 ? 0 : threadIdx.x / kWave);
  int64_t rows = n_rows;
  if (n_rows_dev) rows = min(rows, (int64_t)*n_rows_dev);
  if (r >= rows) return;
  constexpr int kSpan = W * kI8Chunk;
  const T* const src = x + r * k;
  float v[kI8Held][8];
  uint32_t m = 0;
  auto widest = [&](const float (&u)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(u[i]) & 0x7fffffffu);
  };
#pragma unroll
  for (int c = 0; c < kI8Held; ++c)
    if (c * kSpan < k) load8<T, N>(src, c * kSpan + at, k, v[c]);
#pragma unroll
  for (int c = 0; c < kI8Held; ++c)
    if (c * kSpan < k) widest(v[c]);
  for (int c = kI8Held * kSpan; c < k; c += kSpan) {
    float u[8];
    load8<T, N>(src, c + at, k, u);
    widest(u);
  }
  const I8Row row(row_max<W>(m));
  const int64_t row_bytes = i8_row_bytes(k);
  auto put = [&](int c, const float (&u)[8]) {
    if (c + at >= row_bytes) return;
    const uint2 w = i8_codes<Exact>(u, row);
    if (inv == nullptr) {
      *reinterpret_cast<uint2*>(codes + r * row_bytes + c + at) = w;
    } else {
      for (int j = 0; j < top_k; ++j) {
        const int64_t to = inv[r * top_k + j];
        if (to >= 0) *reinterpret_cast<uint2*>(codes + to * row_bytes + c + at) = w;
      }
    }
  };
#pragma unroll
  for (int c = 0; c < kI8Held; ++c)
    if (c * kSpan < k) put(c * kSpan, v[c]);
  for (int c = kI8Held * kSpan; c < k; c += kSpan) {
    float u[8];
    load8<T, N>(src, c + at, k, u);
    put(c, u);
  }
  if (at != 0) return;
  if (inv == nullptr) {
    scales[r] = row.scale;
  } else {
    for (int j = 0; j < top_k; ++j) {
      const int64_t to = inv[r * top_k + j];
      if (to >= 0) scales[to] = row.scale;
    }
  }
}

// The chunks of all rows are numbered row by row; a wave takes U consecutive ones at a time.
template <typename T, int N, int U>
__global__ __launch_bounds__(kI8Threads) void i8_dequantize_kernel(
    const uint8_t* __restrict__ codes, const float* __restrict__ scales, int64_t n_rows, int k,
    T* __restrict__ out, ClearedTail<T> tail) {
  if (tail.p) tail.clear(k);
  const int lane = threadIdx.x & (kWave - 1);
  const int chunks = (k + kI8Chunk - 1) / kI8Chunk;
  const int64_t row_bytes = i8_row_bytes(k);
  const int64_t items = n_rows * chunks, stride = (int64_t)gridDim.x * kI8Waves * U;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  for (int64_t it = ((int64_t)blockIdx.x * kI8Waves + wave) * U; it < items; it += stride) {
    uint2 w[U];
    float s[U];
    int64_t row[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t number = min(it + u, items - 1);
      row[u] = number / chunks;
      at[u] = (int)(number - row[u] * chunks) * kI8Chunk + lane * 8;
      if (it + u >= items) at[u] = k;
      w[u] = make_uint2(0, 0);
      if (at[u] < k) w[u] = *reinterpret_cast<const uint2*>(codes + row[u] * row_bytes + at[u]);
      s[u] = scales[row[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] >= k) continue;
      float v[8];
      i8_values(w[u], s[u], v);
      store8<T, N>(out + row[u] * k, at[u], k, v);
    }
  }
}

#define FMOE_RUNS(CALL)                                             \
  do {                                                              \
    constexpr int kMost = 16 / (int)sizeof(T);                      \
    if (run == 8) CALL(kMost);                                      \
    else if (run == 4) CALL(4);                                     \
    else if (run == 2) CALL(2);                                     \
    else CALL(1);                                                   \
  } while (0)

// One wave a row where rows are enough to fill the chip and short enough for its registers.
constexpr int64_t kI8ManyRows = 256 * 16;

template <typename T>
static int launch_quantize(const void* x, int64_t n_rows, int k, const int32_t* n_rows_dev,
                           const int32_t* inv, int top_k, uint8_t* codes, float* scales,
                           const SegmentsOut& segments, hipStream_t s) {
  const int run = run_length<T>(x, k);
  const bool one = k <= kI8Chunk || (n_rows >= kI8ManyRows && k <= kI8Held * kI8Chunk);
  const dim3 grid((unsigned)std::max<int64_t>(one ? (n_rows + kI8Waves - 1) / kI8Waves : n_rows, 1));
#define FMOE_CALL(N)                                                                             \
  do {                                                                                           \
    if (one)                                                                                     \
      hipLaunchKernelGGL((i8_quantize_kernel<T, N, 1>), grid, dim3(kI8Threads), 0, s,            \
                         (const T*)x, n_rows, k, n_rows_dev, inv, top_k, codes, scales, segments); \
    else                                                                                         \
      hipLaunchKernelGGL((i8_quantize_kernel<T, N, kI8Waves>), grid, dim3(kI8Threads), 0, s,     \
                         (const T*)x, n_rows, k, n_rows_dev, inv, top_k, codes, scales, segments); \
  } while (0)
  FMOE_RUNS(FMOE_CALL);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("i8_quantize");
  return FMOE_OK;
}

// Four chunks at a time where that leaves every CU several waves.
constexpr int64_t kI8ManyItems = 256 * 32;

template <typename T>
static int launch_dequantize(const uint8_t* codes, const float* scales, int64_t n_rows, int k,
                             void* out, const int32_t* tail_end, void* tail, int64_t tail_rows,
                             hipStream_t s) {
  const int run = run_length<T>(out, k);
  const int64_t items = n_rows * ((k + kI8Chunk - 1) / kI8Chunk);
  const bool many = items >= kI8ManyItems;
  const int64_t per_block = kI8Waves * (many ? 4 : 1);
  const dim3 grid((unsigned)std::max<int64_t>(std::min<int64_t>((items + per_block - 1) / per_block, 256 * 64), 1));
  const ClearedTail<T> cleared{tail_end, (T*)tail, tail_rows};
#define FMOE_CALL(N)                                                                            \
  do {                                                                                          \
    if (many)                                                                                   \
      hipLaunchKernelGGL((i8_dequantize_kernel<T, N, 4>), grid, dim3(kI8Threads), 0, s, codes,  \
                         scales, n_rows, k, (T*)out, cleared);                                  \
    else                                                                                        \
      hipLaunchKernelGGL((i8_dequantize_kernel<T, N, 1>), grid, dim3(kI8Threads), 0, s, codes,  \
                         scales, n_rows, k, (T*)out, cleared);                                  \
  } while (0)
  FMOE_RUNS(FMOE_CALL);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("i8_dequantize");
  return FMOE_OK;
}

static int i8_quantize(const void* x, int64_t n_rows, int64_t k, const int32_t* n_rows_dev,
                       const int32_t* inv, int64_t top_k, void* codes, float* scales, int dtype,
                       hipStream_t s, const SegmentsOut& segments = {}) {
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && k >= 1 && k <= FMOE_I8_MAX_FEATURES,
               FMOE_ERR_INVALID, "i8_quantize: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "i8_quantize: unsupported dtype %d", dtype);
  if (n_rows == 0 && !segments.seg_off) return FMOE_OK;
  FMOE_REQUIRE((x && codes && scales) || n_rows == 0, FMOE_ERR_INVALID, "i8_quantize: null pointer");
  FMOE_REQUIRE((uintptr_t)codes % 16 == 0, FMOE_ERR_INVALID,
               "i8_quantize: codes must be 16-byte aligned");
  uint8_t* const c = (uint8_t*)codes;
  switch (dtype) {
    case FMOE_F32:
      return launch_quantize<float>(x, n_rows, (int)k, n_rows_dev, inv, (int)top_k, c, scales, segments, s);
    case FMOE_F16:
      return launch_quantize<__half>(x, n_rows, (int)k, n_rows_dev, inv, (int)top_k, c, scales, segments, s);
    default:
      return launch_quantize<__hip_bfloat16>(x, n_rows, (int)k, n_rows_dev, inv, (int)top_k, c, scales, segments, s);
  }
}

static int i8_dequantize(const void* codes, const float* scales, int64_t n_rows, int64_t k, void* out,
                         const int32_t* tail_end, void* tail, int64_t tail_rows, int dtype,
                         hipStream_t s) {
  FMOE_REQUIRE(n_rows >= 0 && k >= 1 && k <= FMOE_I8_MAX_FEATURES, FMOE_ERR_INVALID,
               "i8_dequantize: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "i8_dequantize: unsupported dtype %d", dtype);
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(codes && scales && out, FMOE_ERR_INVALID, "i8_dequantize: null pointer");
  FMOE_REQUIRE((uintptr_t)codes % 16 == 0, FMOE_ERR_INVALID,
               "i8_dequantize: codes must be 16-byte aligned");
  const uint8_t* const c = (const uint8_t*)codes;
  switch (dtype) {
    case FMOE_F32:
      return launch_dequantize<float>(c, scales, n_rows, (int)k, out, tail_end, tail, tail_rows, s);
    case FMOE_F16:
      return launch_dequantize<__half>(c, scales, n_rows, (int)k, out, tail_end, tail, tail_rows, s);
    default:
      return launch_dequantize<__hip_bfloat16>(c, scales, n_rows, (int)k, out, tail_end, tail, tail_rows, s);
  }
}

}  // namespace fmoe

extern "C" int64_t fmoe_i8_row_bytes(int64_t features) {
  FMOE_REQUIRE(features >= 0 && features <= FMOE_I8_MAX_FEATURES, FMOE_ERR_INVALID,
               "i8: bad feature count");
  return fmoe::i8_row_bytes(features);
}

extern "C" int fmoe_i8_quantize(const void* x, int64_t n_rows, int64_t features,
                                const int32_t* n_rows_dev, void* codes, float* scales, int dtype,
                                void* stream) {
  return fmoe::i8_quantize(x, n_rows, features, n_rows_dev, nullptr, 1, codes, scales, dtype,
                           (hipStream_t)stream);
}

extern "C" int fmoe_i8_quantize_counted(const void* x, int64_t n_rows, int64_t features,
                                        const int64_t* expert_count, int64_t n_expert,
                                        int32_t* seg_off, void* codes, float* scales, int dtype,
                                        void* stream) {
  FMOE_REQUIRE((expert_count || n_expert == 1) && seg_off && n_expert >= 1 && n_expert < INT32_MAX,
               FMOE_ERR_INVALID, "i8_quantize_counted: bad counts");
  return fmoe::i8_quantize(x, n_rows, features, nullptr, nullptr, 1, codes, scales, dtype,
                           (hipStream_t)stream, {expert_count, (int)n_expert, seg_off});
}

extern "C" int fmoe_i8_quantize_tokens(const void* x, const int32_t* inv, int64_t n_tokens,
                                       int64_t top_k, int64_t features, void* codes, float* scales,
                                       int dtype, void* stream) {
  FMOE_REQUIRE(top_k >= 1 && n_tokens >= 0 && n_tokens <= INT32_MAX / top_k, FMOE_ERR_INVALID,
               "i8_quantize_tokens: bad sizes");
  FMOE_REQUIRE(n_tokens == 0 || inv, FMOE_ERR_INVALID, "i8_quantize_tokens: null pointer");
  return fmoe::i8_quantize(x, n_tokens, features, nullptr, inv, top_k, codes, scales, dtype,
                           (hipStream_t)stream);
}

extern "C" int fmoe_i8_dequantize(const void* codes, const float* scales, int64_t n_rows,
                                  int64_t features, void* out, int dtype, void* stream) {
  return fmoe::i8_dequantize(codes, scales, n_rows, features, out, nullptr, nullptr, 0, dtype,
                             (hipStream_t)stream);
}

extern "C" int fmoe_i8_dequantize_bwd(const void* w_codes, const float* w_scales,
                                      const int32_t* seg_off, void* w, void* dx, int64_t n_rows,
                                      int64_t in_feat, int64_t out_feat, int64_t n_expert,
                                      int dtype, void* stream) {
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && n_expert >= 1 && n_expert < INT32_MAX &&
                   out_feat >= 1 && out_feat <= FMOE_I8_MAX_FEATURES,
               FMOE_ERR_INVALID, "i8_dequantize_bwd: bad sizes");
  FMOE_REQUIRE(seg_off && (dx || n_rows == 0), FMOE_ERR_INVALID, "i8_dequantize_bwd: null pointer");
  return fmoe::i8_dequantize(w_codes, w_scales, n_expert * out_feat, in_feat, w, seg_off + n_expert,
                             n_rows ? dx : nullptr, n_rows, dtype, (hipStream_t)stream);
}
