// Quantisation of rows to 8-bit integers and back on gfx950 (the format: i8.h).
//
// Both directions are bound by HBM: a value costs its own 2 or 4 bytes plus one.  The scale needs
// the whole row before the first code, so up to eight waves keep a row in registers between the two
// (4 KiB each; what is longer is read a second time, from L2 as a rule), and the next row is on its
// way meanwhile.  Measured: 114688 x 4096 in bf16 to 8 bits 240 us, 1.41 GB at 5.9 TB/s, and back 238,
// at 5.9 (a large copy reaches 5.2); 1000 x 300 in f32 3.8 and 3.0, a launch alone 2.1.
//
// A code is one multiply-add: t = x (127 / a) + 1.5 * 2^23 rounds the product, taken exactly, to an
// integer whose low byte is the code.  The quotient is off by up to 2^-23 of itself, and so is the
// product r = 127 x / a near a half-way point k + 1/2.  The distance there is |254 x - (2 k + 1) a| /
// (2 a): with x and a of m bits, it is zero or at least 2^-m / 254 of r, so that for 16-bit types
// (m = 8, 11) only exact ties can go wrong.  254 x = (2 k + 1) a needs 127 to divide 2 k + 1, which
// is k = 63, or the digits of a.  The first goes to the even 64 if the quotient is rounded up, which
// it is; rows with the second, 1 in 128, decide every code by the sign of 127 |x| - (k + 1/2) a,
// whose terms have at most 19 bits.  f32 values do so, in f64, where a product is within 2^-15 of a
// half-way point.  (Looking for
// products near a half-way point in 16-bit rows as well, where every x = a / 2 is one: 306 us in place
// of 250 for 114688 x 4096.)
#include <algorithm>

#include "i8.h"
#include "rows.h"

namespace fmoe {

constexpr int kI8Threads = 256;              // of a block that dequantises
constexpr int kI8Chunk = kWave * 8;          // values that a wave takes at once
constexpr int kI8HeldBytes = 4096;           // of a row in a wave's registers
constexpr float kI8Magic = 12582912.f;       // 1.5 * 2^23: a float there has integers as its steps

// What turns a row's values into codes.
struct I8Row {
  float unit;       // power of two that keeps everything below in range
  float top;        // the largest magnitude, times unit
  float inv;        // 127 / top, rounded up
  float scale;      // 0 for a row of zeros, NaN for one that is not finite
  bool finite;
  bool ties;        // of 16-bit values: there may be ties other than top / 2

  __device__ __forceinline__ explicit I8Row(uint32_t top_bits) {
    finite = top_bits < 0x7f800000u;
    const float a = __uint_as_float(finite ? top_bits : 0u);
    unit = a < 0x1p-60f ? 0x1p64f : a > 0x1p60f ? 0x1p-64f : 1.f;
    top = a * unit;
    inv = 127.f / top;
    if (fmaf(inv, top, -127.f) < 0.f) inv = __uint_as_float(__float_as_uint(inv) + 1);
    if (!(top > 0.f)) inv = 0.f;
    ties = ((__float_as_uint(top) & 0x7fffffu) | 0x800000u) % 127 == 0;
    scale = finite ? a / 127.f : __uint_as_float(0x7fc00000u);
  }

  // The code of x, as a float, decided exactly.
  template <typename EXACT> __device__ __forceinline__ float decide(float x) const {
    const float k = floorf(fabsf(x) * inv);
    const EXACT side = fma(-((EXACT)k + (EXACT)0.5), (EXACT)top, (EXACT)127 * (EXACT)fabsf(x));
    const bool odd = (int)k & 1;
    return copysignf(side > 0 || (side == 0 && odd) ? k + 1.f : k, x);
  }

  // The codes of 8 values, v[0] in the lowest byte.
  template <typename T> __device__ __forceinline__ uint2 codes(const Eight<T>& from) const {
    float v[8], t[8];
    from.widen(v);
    if (unit != 1.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= unit;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = fmaf(v[i], inv, kI8Magic);
    if constexpr (sizeof(T) == 2) {
      if (ties) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = decide<float>(v[i]) + kI8Magic;
      }
    } else {
      float off = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) off = fmaxf(off, fabsf(fmaf(v[i], inv, kI8Magic - t[i])));
      if (off > 0.5f - 0x1p-15f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = decide<double>(v[i]) + kI8Magic;
      }
    }
    auto four = [&](int i) {
      const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[i + 1]), __float_as_uint(t[i]), 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[i + 3]), __float_as_uint(t[i + 2]), 0x04000c0cu);
      return lo | hi;
    };
    return finite ? make_uint2(four(0), four(4)) : make_uint2(0, 0);
  }
};

// The maximum of m over the waves of a block; `part` is not the one of the call before.
template <int W> __device__ __forceinline__ uint32_t row_max(uint32_t m, uint32_t* part) {
  m = wave_max(m);
  if constexpr (W > 1) {
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) m = max(m, part[w]);
  }
  return m;
}

// Row r goes to row r, and rows from *n_rows_dev on (if given) are skipped; or, PLACED, row t to the
// rows inv[t * top_k + j] that are not -1.  A block of W waves takes row after row, the next one's
// loads under way while it works on one's values.
template <typename T, int W, bool PLACED>
__global__ __launch_bounds__(W * kWave) void i8_quantize_kernel(
    const T* __restrict__ x, int64_t n_rows, int k, const int32_t* __restrict__ n_rows_dev,
    const int32_t* __restrict__ inv, int top_k, uint8_t* __restrict__ codes,
    float* __restrict__ scales, SegmentsOut segments) {
  constexpr int kHeld = kI8HeldBytes / (8 * kWave * (int)sizeof(T));     // chunks in registers
  constexpr int kSpan = W * kI8Chunk;
  __shared__ uint32_t part[2][W];
  if (segments.seg_off && blockIdx.x == 0 && threadIdx.x < kWave)
    write_segments(segments, n_rows, threadIdx.x);
  const int at = threadIdx.x * 8;                      // first value of the thread's in a chunk
  const bool odd = threadIdx.x & 1;
  const int row_bytes = (int)i8_row_bytes(k);
  int64_t rows = n_rows;
  if (n_rows_dev) rows = min(rows, (int64_t)*n_rows_dev);
  Eight<T> held[kHeld];
  auto fetch = [&](int64_t row) {
    const T* const src = x + row * k;
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      if ((c + 1) * kSpan <= k) held[c].template load<true>(src + c * kSpan + at);
      else if (c * kSpan < k) held[c].template load<true>(src, c * kSpan + at, k);
    }
  };
  int64_t r = blockIdx.x;
  if (r < rows) fetch(r);
  for (int turn = 0; r < rows; r += gridDim.x, turn ^= 1) {
    Eight<T> v[kHeld];
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      if (c * kSpan >= k) break;
      m = held[c].widest(m);
      v[c] = held[c];
    }
    if (r + gridDim.x < rows) fetch(r + gridDim.x);
    for (int c = kHeld * kSpan; c < k; c += kSpan) {
      Eight<T> u;
      u.load(x + r * k, c + at, k);
      m = u.widest(m);
    }
    const I8Row row(row_max<W>(Eight<T>::f32_bits(m), part[turn]));
    // The codes of the chunks from c and c + kSpan on: neighbouring lanes exchange halves, so that
    // a lane stores 16 bytes of one of the two.
    auto put = [&](int c, const Eight<T>& a, const Eight<T>& b, bool second) {
      const uint2 ca = row.codes(a), cb = second ? row.codes(b) : make_uint2(0, 0);
      const uint32_t s0 = odd ? ca.x : cb.x, s1 = odd ? ca.y : cb.y;
      const uint32_t g0 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)s0, 0xb1, 0xf, 0xf, false);
      const uint32_t g1 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)s1, 0xb1, 0xf, 0xf, false);
      const uint4 w = odd ? make_uint4(g0, g1, cb.x, cb.y) : make_uint4(ca.x, ca.y, g0, g1);
      const int to = c + (odd ? kSpan : 0) + (at & ~15);
      if (to >= row_bytes) return;
      if constexpr (!PLACED) {
        *reinterpret_cast<uint4*>(codes + r * row_bytes + to) = w;
      } else {
        for (int j = 0; j < top_k; ++j) {
          const int64_t place = inv[r * top_k + j];
          if (place >= 0) *reinterpret_cast<uint4*>(codes + place * row_bytes + to) = w;
        }
      }
    };
#pragma unroll
    for (int c = 0; c < kHeld; c += 2) {
      if (c * kSpan >= k) break;
      put(c * kSpan, v[c], v[c + 1], (c + 1) * kSpan < k);
    }
    for (int c = kHeld * kSpan; c < k; c += 2 * kSpan) {
      Eight<T> a, b;
      a.load(x + r * k, c + at, k);
      b.load(x + r * k, c + kSpan + at, k);
      put(c, a, b, c + kSpan < k);
    }
    if (threadIdx.x != 0) continue;
    if constexpr (!PLACED) {
      scales[r] = row.scale;
    } else {
      for (int j = 0; j < top_k; ++j) {
        const int64_t place = inv[r * top_k + j];
        if (place >= 0) scales[place] = row.scale;
      }
    }
  }
}

// The chunks of all rows are numbered row by row; a wave takes U consecutive ones at a time, a lane 16
// bytes of values, N, of each of a chunk's 8 / N parts.  ONCE: nobody reads them at once.
template <typename T, int U, bool ONCE>
__global__ __launch_bounds__(kI8Threads) void i8_dequantize_kernel(
    const uint8_t* __restrict__ codes, const float* __restrict__ scales, int64_t n_rows, int k,
    T* __restrict__ out, ClearedTail<T> tail) {
  constexpr int kWaves = kI8Threads / kWave, N = 16 / (int)sizeof(T), kParts = 8 / N;
  if (tail.p) tail.clear(k);
  const int lane = threadIdx.x & (kWave - 1);
  const int chunks = (k + kI8Chunk - 1) / kI8Chunk;
  const int64_t row_bytes = i8_row_bytes(k);
  const int64_t items = n_rows * chunks, stride = (int64_t)gridDim.x * kWaves * U;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  for (int64_t it = ((int64_t)blockIdx.x * kWaves + wave) * U; it < items; it += stride) {
    uint32_t w[U][kParts][N / 4];
    float s[U];
    int64_t row[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t number = min(it + u, items - 1);
      row[u] = number / chunks;
      at[u] = (int)(number - row[u] * chunks) * kI8Chunk + lane * N;
      if (it + u >= items) at[u] = k;
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
        const int from = at[u] + q * kWave * N;        // (codes reach to the next 128 features)
        if (from < k) __builtin_memcpy(w[u][q], codes + row[u] * row_bytes + from, N);
      }
      s[u] = scales[row[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] >= k) continue;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = (float)(int8_t)(w[u][i / N][i % N / 4] >> (8 * (i & 3))) * s[u];
        // (an f32 product, always: left alone, the compiler makes it and a conversion to f16 one
        // instruction with one rounding, here and there)
        asm("" : "+v"(v[i]));
      }
      Eight<T>::template store<ONCE>(out + row[u] * k, at[u], k, v, kWave * N);
    }
  }
}

// Waves of a row: as many as hold it, or, where rows are few, as many as find a chunk in it (2047 x
// 2048 in bf16: 5.9 us, otherwise 6.9; 4000 x 4096: 18.2, otherwise 13.8).
constexpr int64_t kI8FewRows = 2048;
constexpr int64_t kI8Waves = 256 * 16;     // as many as their registers allow on the chip

template <typename T, int W>
static void start_quantize(const void* x, int64_t n_rows, int k, const int32_t* n_rows_dev,
                           const int32_t* inv, int top_k, uint8_t* codes, float* scales,
                           const SegmentsOut& segments, hipStream_t s) {
  const dim3 grid((unsigned)std::max<int64_t>(std::min(n_rows, kI8Waves / W), 1));
  if (inv)
    hipLaunchKernelGGL((i8_quantize_kernel<T, W, true>), grid, dim3(W * kWave), 0, s, (const T*)x,
                       n_rows, k, n_rows_dev, inv, top_k, codes, scales, segments);
  else
    hipLaunchKernelGGL((i8_quantize_kernel<T, W, false>), grid, dim3(W * kWave), 0, s, (const T*)x,
                       n_rows, k, n_rows_dev, inv, top_k, codes, scales, segments);
}

template <typename T>
static int launch_quantize(const void* x, int64_t n_rows, int k, const int32_t* n_rows_dev,
                           const int32_t* inv, int top_k, uint8_t* codes, float* scales,
                           const SegmentsOut& segments, hipStream_t s) {
  const int64_t need = n_rows < kI8FewRows
                           ? ((int64_t)k + kI8Chunk - 1) / kI8Chunk
                           : ((int64_t)k * (int)sizeof(T) + kI8HeldBytes - 1) / kI8HeldBytes;
#define FMOE_START(W) \
  start_quantize<T, W>(x, n_rows, k, n_rows_dev, inv, top_k, codes, scales, segments, s)
  if (need <= 1) FMOE_START(1);
  else if (need <= 2) FMOE_START(2);
  else if (need <= 4) FMOE_START(4);
  else FMOE_START(8);
#undef FMOE_START
  FMOE_LAUNCH_CHECK("i8_quantize");
  return FMOE_OK;
}

// Four chunks at a time where that leaves every CU several waves (114688 x 4096 in bf16: 243 us, one at
// a time 291; 16376 x 2048 23 and 21).
constexpr int64_t kI8ManyItems = 256 * 32;

template <typename T, bool ONCE>
static int launch_dequantize(const uint8_t* codes, const float* scales, int64_t n_rows, int k,
                             void* out, const ClearedTail<T>& cleared, hipStream_t s) {
  const int64_t items = n_rows * ((k + kI8Chunk - 1) / kI8Chunk);
  const bool many = items >= kI8ManyItems;
  const int64_t per_block = kI8Threads / kWave * (many ? 4 : 1);
  const dim3 grid((unsigned)std::max<int64_t>(std::min<int64_t>((items + per_block - 1) / per_block, 256 * 64), 1));
  if (many)
    hipLaunchKernelGGL((i8_dequantize_kernel<T, 4, ONCE>), grid, dim3(kI8Threads), 0, s, codes, scales,
                       n_rows, k, (T*)out, cleared);
  else
    hipLaunchKernelGGL((i8_dequantize_kernel<T, 1, ONCE>), grid, dim3(kI8Threads), 0, s, codes, scales,
                       n_rows, k, (T*)out, cleared);
  FMOE_LAUNCH_CHECK("i8_dequantize");
  return FMOE_OK;
}

// (weights that a product reads next stay in the caches, others pass them by: 232 in place of 243 us)
template <typename T>
static int launch_dequantize(const uint8_t* codes, const float* scales, int64_t n_rows, int k,
                             void* out, const int32_t* tail_end, void* tail, int64_t tail_rows,
                             hipStream_t s) {
  const ClearedTail<T> cleared{tail_end, (T*)tail, tail_rows};
  return tail_end ? launch_dequantize<T, false>(codes, scales, n_rows, k, out, cleared, s)
                  : launch_dequantize<T, true>(codes, scales, n_rows, k, out, cleared, s);
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
