// Quantisation of rows to MXFP4 and back on gfx950 (the format: mx.h).
//
// Both directions are bound by HBM: a value costs its own 2 or 4 bytes plus 17/32 of a byte.
// Four lanes share a block of 32 values, 8 each (one 16-byte load of a 16-bit type), so a
// wave's load covers 1 KiB of a row and its store 256 bytes; the block's largest magnitude is
// two DPP steps inside the four lanes, taken on the bits as integers (NaN > infinity > numbers),
// and the codes come from the conversion instruction that divides by the power of two itself.
// The form for tokens writes a row to its top_k places in expert order, which makes the
// dispatch of a 4-bit layer part of this pass: 4.25 bits written per value and place.
#include <algorithm>

#include "mx.h"

namespace fmoe {

constexpr int kMxThreads = 256;
constexpr int kMxWaves = kMxThreads / kWave;
constexpr int kMxChunk = kWave * 8;          // values of a row that a wave takes at once
static_assert(kMxChunk == kMxGroup, "a chunk's scales are one 16-byte pack");

// 8 values of a row from element k on, as f32; zeros from k_total on.  VEC: 16-byte packs.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int k, int k_total, float (&v)[8]) {
  if (VEC) {
    constexpr int kN = Pack16<T>::kN;
#pragma unroll
    for (int p = 0; p < 8 / kN; ++p) {
      if (k + p * kN < k_total) {
        const Pack16<T> x = *reinterpret_cast<const Pack16<T>*>(row + k + p * kN);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[p * kN + i] = Elem<T>::to_acc(x.v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[p * kN + i] = 0.f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < k_total ? Elem<T>::to_acc(row[k + i]) : 0.f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int k, int k_total, const float (&v)[8]) {
  if (VEC) {
    constexpr int kN = Pack16<T>::kN;
#pragma unroll
    for (int p = 0; p < 8 / kN; ++p) {
      if (k + p * kN >= k_total) break;
      Pack16<T> x;
#pragma unroll
      for (int i = 0; i < kN; ++i) x.v[i] = Elem<T>::from_acc(v[p * kN + i]);
      *reinterpret_cast<Pack16<T>*>(row + k + p * kN) = x;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < k_total) row[k + i] = Elem<T>::from_acc(v[i]);
  }
}

// Maximum over the four lanes of a block, in each of them.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));  // 1 0 3 2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));  // 2 3 0 1
  return v;
}

// Row counts of experts as segment bounds, for the call's first workgroup to leave behind.
struct MxSegments {
  const int64_t* count = nullptr;
  int n_expert = 0;
  int32_t* seg_off = nullptr;
};

// seg_off = exclusive prefix of the counts, by one wave.  Counts on the device nobody has looked
// at: negative ones count as zero, and what lies beyond the rows there are is cut off.
__device__ __forceinline__ void write_segments(const MxSegments& sg, int64_t n_rows, int lane) {
  int64_t carry = 0;
  for (int e0 = 0; e0 < sg.n_expert; e0 += kWave) {
    const int64_t c = e0 + lane < sg.n_expert ? min(max(sg.count[e0 + lane], (int64_t)0), n_rows) : 0;
    int64_t sum = c;
    for (int d = 1; d < kWave; d <<= 1) {
      const int64_t o = __shfl_up(sum, d, kWave);
      if (lane >= d) sum += o;
    }
    if (e0 + lane < sg.n_expert) sg.seg_off[e0 + lane] = (int32_t)min(carry + sum - c, n_rows);
    carry += __shfl(sum, kWave - 1, kWave);
  }
  if (lane == 0) sg.seg_off[sg.n_expert] = (int32_t)min(carry, n_rows);
}

// One wave takes `U` chunks of a row at a time.  inv == nullptr: row r goes to row r, and rows
// from *n_rows_dev on (if given) are skipped; else row t goes to the rows inv[t * top_k + j]
// that are not -1.
template <typename T, bool VEC, int U>
__global__ __launch_bounds__(kMxThreads) void mx_quantize_kernel(
    const T* __restrict__ x, int64_t n_rows, int k, const int32_t* __restrict__ n_rows_dev,
    const int32_t* __restrict__ inv, int top_k, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ scales, MxSegments segments) {
  const int lane = threadIdx.x & (kWave - 1);
  if (segments.seg_off && blockIdx.x == 0 && threadIdx.x < kWave) write_segments(segments, n_rows, lane);
  const int chunks = (k + kMxChunk - 1) / kMxChunk, runs = (chunks + U - 1) / U;
  const int64_t code_row = mx_code_bytes(k), scale_row = mx_scale_bytes(k);
  int64_t rows = n_rows;
  if (n_rows_dev) rows = min(rows, (int64_t)*n_rows_dev);
  const int64_t items = rows * runs, n_waves = (int64_t)gridDim.x * kMxWaves;
  for (int64_t it = (int64_t)blockIdx.x * kMxWaves + threadIdx.x / kWave; it < items;
       it += n_waves) {
    const int64_t row = it / runs;
    const int c0 = (int)(it - row * runs) * U;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
      load8<T, VEC>(x + row * k, (c0 + u) * kMxChunk + lane * 8, k, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + u >= chunks) break;
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, magnitude_bits(v[u][i]));
      const int byte = mx_scale_byte(quad_max(m));
      const uint32_t word = mx_codes(v[u], byte);
      const int64_t at = (int64_t)(c0 + u) * (kMxChunk / 2) + lane * 4;
      const int64_t sat = (int64_t)(c0 + u) * 16 + (lane >> 2);
      if (inv == nullptr) {
        if (at < code_row) *reinterpret_cast<uint32_t*>(codes + row * code_row + at) = word;
        if ((lane & 3) == 0) scales[row * scale_row + sat] = (uint8_t)byte;
      } else {
        for (int j = 0; j < top_k; ++j) {
          const int64_t to = inv[row * top_k + j];
          if (to < 0) continue;
          if (at < code_row) *reinterpret_cast<uint32_t*>(codes + to * code_row + at) = word;
          if ((lane & 3) == 0) scales[to * scale_row + sat] = (uint8_t)byte;
        }
      }
    }
  }
}

template <typename T, bool VEC, int U>
__global__ __launch_bounds__(kMxThreads) void mx_dequantize_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n_rows, int k,
    T* __restrict__ out) {
  const int lane = threadIdx.x & (kWave - 1);
  const int chunks = (k + kMxChunk - 1) / kMxChunk, runs = (chunks + U - 1) / U;
  const int64_t code_row = mx_code_bytes(k), scale_row = mx_scale_bytes(k);
  const int64_t items = n_rows * runs, n_waves = (int64_t)gridDim.x * kMxWaves;
  for (int64_t it = (int64_t)blockIdx.x * kMxWaves + threadIdx.x / kWave; it < items;
       it += n_waves) {
    const int64_t row = it / runs;
    const int c0 = (int)(it - row * runs) * U;
    uint32_t word[U];
    int byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (int64_t)(c0 + u) * (kMxChunk / 2) + lane * 4;
      const bool in = at < code_row;       // (the row's scales reach at least as far)
      word[u] = in ? *reinterpret_cast<const uint32_t*>(codes + row * code_row + at) : 0;
      byte[u] = in ? scales[row * scale_row + (int64_t)(c0 + u) * 16 + (lane >> 2)] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = (c0 + u) * kMxChunk + lane * 8;
      if (at >= k) break;
      float v[8];
      mx_values(word[u], byte[u], v);
      store8<T, VEC>(out + row * k, at, k, v);
    }
  }
}

// Chunks that a wave takes at once: one where the rows are too few to fill the GPU with waves
// of four.
constexpr int kMxManyItems = 256 * 32;

template <typename T>
static int launch_quantize(const void* x, int64_t n_rows, int k, const int32_t* n_rows_dev,
                           const int32_t* inv, int top_k, uint8_t* codes, uint8_t* scales,
                           const MxSegments& segments, hipStream_t s) {
  const bool vec = k % Pack16<T>::kN == 0 && (uintptr_t)x % 16 == 0;
  const int64_t chunks = ceil_div(k, kMxChunk);
  const bool many = chunks >= 4 && n_rows * (chunks / 4) >= kMxManyItems;
  const int64_t items = n_rows * (many ? (chunks + 3) / 4 : chunks);
  const dim3 grid((unsigned)std::min<int64_t>(std::max<int64_t>((items + kMxWaves - 1) / kMxWaves, 1), 256 * 64));
#define FMOE_CALL(VEC, U)                                                                        \
  hipLaunchKernelGGL((mx_quantize_kernel<T, VEC, U>), grid, dim3(kMxThreads), 0, s, (const T*)x, \
                     n_rows, k, n_rows_dev, inv, top_k, codes, scales, segments)
  if (vec && many) FMOE_CALL(true, 4);
  else if (vec) FMOE_CALL(true, 1);
  else FMOE_CALL(false, 1);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("mx_quantize");
  return FMOE_OK;
}

template <typename T>
static int launch_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t n_rows, int k,
                             void* out, hipStream_t s) {
  const bool vec = k % Pack16<T>::kN == 0 && (uintptr_t)out % 16 == 0;
  const int64_t chunks = ceil_div(k, kMxChunk);
  const bool many = chunks >= 4 && n_rows * (chunks / 4) >= kMxManyItems;
  const int64_t items = n_rows * (many ? (chunks + 3) / 4 : chunks);
  const dim3 grid((unsigned)std::min<int64_t>((items + kMxWaves - 1) / kMxWaves, 256 * 64));
#define FMOE_CALL(VEC, U)                                                                      \
  hipLaunchKernelGGL((mx_dequantize_kernel<T, VEC, U>), grid, dim3(kMxThreads), 0, s, codes,   \
                     scales, n_rows, k, (T*)out)
  if (vec && many) FMOE_CALL(true, 4);
  else if (vec) FMOE_CALL(true, 1);
  else FMOE_CALL(false, 1);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("mx_dequantize");
  return FMOE_OK;
}

static int quantize(const void* x, int64_t n_rows, int64_t k, const int32_t* n_rows_dev,
                    const int32_t* inv, int64_t top_k, void* codes, void* scales, int dtype,
                    hipStream_t s, const MxSegments& segments = {}) {
  FMOE_REQUIRE(n_rows >= 0 && k >= 1 && k <= FMOE_MX_MAX_FEATURES, FMOE_ERR_INVALID,
               "mx_quantize: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "mx_quantize: unsupported dtype %d", dtype);
  if (n_rows == 0 && !segments.seg_off) return FMOE_OK;
  FMOE_REQUIRE((x && codes && scales) || n_rows == 0, FMOE_ERR_INVALID, "mx_quantize: null pointer");
  FMOE_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, FMOE_ERR_INVALID,
               "mx_quantize: codes and scales must be 16-byte aligned");
  uint8_t *c = (uint8_t*)codes, *sc = (uint8_t*)scales;
  switch (dtype) {
    case FMOE_F32:
      return launch_quantize<float>(x, n_rows, (int)k, n_rows_dev, inv, (int)top_k, c, sc, segments, s);
    case FMOE_F16:
      return launch_quantize<__half>(x, n_rows, (int)k, n_rows_dev, inv, (int)top_k, c, sc, segments, s);
    default:
      return launch_quantize<__hip_bfloat16>(x, n_rows, (int)k, n_rows_dev, inv, (int)top_k, c, sc, segments, s);
  }
}

}  // namespace fmoe

extern "C" int64_t fmoe_mx_code_bytes(int64_t features) {
  FMOE_REQUIRE(features >= 0 && features <= FMOE_MX_MAX_FEATURES, FMOE_ERR_INVALID,
               "mx: bad feature count");
  return fmoe::mx_code_bytes(features);
}

extern "C" int64_t fmoe_mx_scale_bytes(int64_t features) {
  FMOE_REQUIRE(features >= 0 && features <= FMOE_MX_MAX_FEATURES, FMOE_ERR_INVALID,
               "mx: bad feature count");
  return fmoe::mx_scale_bytes(features);
}

extern "C" int fmoe_mx_quantize(const void* x, int64_t n_rows, int64_t features,
                                const int32_t* n_rows_dev, void* codes, void* scales, int dtype,
                                void* stream) {
  return fmoe::quantize(x, n_rows, features, n_rows_dev, nullptr, 1, codes, scales, dtype,
                        (hipStream_t)stream);
}

extern "C" int fmoe_mx_quantize_counted(const void* x, int64_t n_rows, int64_t features,
                                        const int64_t* expert_count, int64_t n_expert,
                                        int32_t* seg_off, void* codes, void* scales, int dtype,
                                        void* stream) {
  FMOE_REQUIRE(expert_count && seg_off && n_expert >= 1 && n_expert < INT32_MAX, FMOE_ERR_INVALID,
               "mx_quantize_counted: bad counts");
  return fmoe::quantize(x, n_rows, features, nullptr, nullptr, 1, codes, scales, dtype,
                        (hipStream_t)stream, {expert_count, (int)n_expert, seg_off});
}

extern "C" int fmoe_mx_quantize_tokens(const void* x, const int32_t* inv, int64_t n_tokens,
                                       int64_t top_k, int64_t features, void* codes, void* scales,
                                       int dtype, void* stream) {
  FMOE_REQUIRE(top_k >= 1 && n_tokens >= 0 && n_tokens <= INT32_MAX / top_k, FMOE_ERR_INVALID,
               "mx_quantize_tokens: bad sizes");
  FMOE_REQUIRE(n_tokens == 0 || inv, FMOE_ERR_INVALID, "mx_quantize_tokens: null pointer");
  return fmoe::quantize(x, n_tokens, features, nullptr, inv, top_k, codes, scales, dtype,
                        (hipStream_t)stream);
}

extern "C" int fmoe_mx_dequantize(const void* codes, const void* scales, int64_t n_rows,
                                  int64_t features, void* out, int dtype, void* stream) {
  using namespace fmoe;
  FMOE_REQUIRE(n_rows >= 0 && features >= 1 && features <= FMOE_MX_MAX_FEATURES, FMOE_ERR_INVALID,
               "mx_dequantize: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "mx_dequantize: unsupported dtype %d", dtype);
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(codes && scales && out, FMOE_ERR_INVALID, "mx_dequantize: null pointer");
  FMOE_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, FMOE_ERR_INVALID,
               "mx_dequantize: codes and scales must be 16-byte aligned");
  const uint8_t *c = (const uint8_t*)codes, *sc = (const uint8_t*)scales;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FMOE_F32: return launch_dequantize<float>(c, sc, n_rows, (int)features, out, s);
    case FMOE_F16: return launch_dequantize<__half>(c, sc, n_rows, (int)features, out, s);
    default: return launch_dequantize<__hip_bfloat16>(c, sc, n_rows, (int)features, out, s);
  }
}
