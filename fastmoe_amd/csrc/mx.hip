// Quantisation of rows to MXFP4 and back on gfx950 (the format: mx.h).
//
// Both directions are bound by HBM: a value costs its own 2 or 4 bytes plus 17/32 of a byte.
// Four lanes share a block of 32 values, 8 each (one 16-byte load of a 16-bit type), so a
// wave's load covers 1 KiB of a row and its store 256 bytes; the block's largest magnitude is
// two DPP steps inside the four lanes, taken on the bits as integers (NaN > infinity > numbers),
// and the codes come from the conversion instruction that divides by the power of two itself.
// The form for tokens writes a row to its top_k places in expert order, which makes the
// dispatch of a 4-bit layer part of this pass: 4.25 bits written per value and place.
// With many rows a wave takes four chunks of 512 values, so that codes are stored 16 bytes a lane.
// Measured: 114688 x 4096 in bf16 to 4 bits and back in 446 us, 2.38 GB at 5.3 TB/s (a large copy
// reaches 5.2); 1000 x 300 in f32 2.7 us either way, a launch alone 2.1.
#include <algorithm>

#include "mx.h"

namespace fmoe {

constexpr int kMxThreads = 256;
constexpr int kMxWaves = kMxThreads / kWave;
constexpr int kMxChunk = kWave * 8;          // values of a row that a wave takes at once
static_assert(kMxChunk == kMxGroup, "a chunk's scales are one 16-byte pack");

// N values, moved as one.
template <typename T, int N> struct alignas(sizeof(T) * N) Run { T v[N]; };

// 8 values of a row from element k on, as f32; zeros from k_total on.  Rows are moved in runs of N
// values, of which they hold whole ones.
template <typename T, int N>
__device__ __forceinline__ void load8(const T* row, int k, int k_total, float (&v)[8]) {
#pragma unroll
  for (int p = 0; p < 8; p += N) {
    Run<T, N> x;
    const bool in = k + p < k_total;
    if (in) x = *reinterpret_cast<const Run<T, N>*>(row + k + p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[p + i] = in ? Elem<T>::to_acc(x.v[i]) : 0.f;
  }
}

template <typename T, int N>
__device__ __forceinline__ void store8(T* row, int k, int k_total, const float (&v)[8]) {
#pragma unroll
  for (int p = 0; p < 8; p += N) {
    if (k + p >= k_total) break;
    Run<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = Elem<T>::from_acc(v[p + i]);
    *reinterpret_cast<Run<T, N>*>(row + k + p) = x;
  }
}

// Maximum over the four lanes of a block, in each of them.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));  // 1 0 3 2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));  // 2 3 0 1
  return v;
}

// w[u] of lane i to w[i] of lane u among every four lanes: four words of a block, one in each
// lane, for four blocks become a block's 16 bytes in one lane, so that four chunks take one store
// of 1 KiB instead of four of 256 bytes.
__device__ __forceinline__ void transpose_quad(uint32_t (&w)[4], int lane) {
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const bool up = lane & d;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u & d) continue;
      const uint32_t send = up ? w[u] : w[u | d];
      const uint32_t got = (uint32_t)(d == 1 ? __builtin_amdgcn_update_dpp(0, (int)send, 0xb1, 0xf, 0xf, false)
                                             : __builtin_amdgcn_update_dpp(0, (int)send, 0x4e, 0xf, 0xf, false));
      w[u] = up ? got : w[u];
      w[u | d] = up ? w[u | d] : got;
    }
  }
}

__device__ __forceinline__ int of_four(const int (&v)[4], int i) {
  return i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3];
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

// The chunks of all rows are numbered row by row; a wave takes U consecutive ones at a time.
struct MxChunk {
  int64_t row;
  int k;                  // first value
  __device__ __forceinline__ MxChunk(int64_t number, int chunks) {
    row = number / chunks;
    k = (int)(number - row * chunks) * kMxChunk;
  }
};

// inv == nullptr: row r goes to row r, and rows from *n_rows_dev on (if given) are skipped; else
// row t goes to the rows inv[t * top_k + j] that are not -1.
template <typename T, int N, int U>
__global__ __launch_bounds__(kMxThreads) void mx_quantize_kernel(
    const T* __restrict__ x, int64_t n_rows, int k, const int32_t* __restrict__ n_rows_dev,
    const int32_t* __restrict__ inv, int top_k, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ scales, MxSegments segments) {
  static_assert(U == 1 || U == 4, "the lanes of a block share the chunks between them");
  const int lane = threadIdx.x & (kWave - 1);
  if (segments.seg_off && blockIdx.x == 0 && threadIdx.x < kWave) write_segments(segments, n_rows, lane);
  const int chunks = (k + kMxChunk - 1) / kMxChunk;
  const int64_t code_row = mx_code_bytes(k), scale_row = mx_scale_bytes(k);
  int64_t rows = n_rows;
  if (n_rows_dev) rows = min(rows, (int64_t)*n_rows_dev);
  const int64_t items = rows * chunks, stride = (int64_t)gridDim.x * kMxWaves * U;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  for (int64_t it = ((int64_t)blockIdx.x * kMxWaves + wave) * U; it < items; it += stride) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const MxChunk c(min(it + u, items - 1), chunks);
      load8<T, N>(x + c.row * k, c.k + lane * 8, k, v[u]);
    }
    uint32_t word[U];
    int byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, magnitude_bits(v[u][i]));
      byte[u] = mx_scale_byte(quad_max(m));
      word[u] = mx_codes(v[u], byte[u]);
    }
    if constexpr (U == 4) {
      // lane j of a block's four lanes gets the whole block of chunk j
      transpose_quad(word, lane);
      byte[0] = of_four(byte, lane & 3);
    }
    const int64_t mine = it + (U == 4 ? lane & 3 : 0);
    if (mine >= items) continue;
    const MxChunk c(mine, chunks);
    const int at = c.k / 2 + (U == 4 ? (lane >> 2) * 16 : lane * 4);
    const int sat = c.k / kMxBlock + (lane >> 2);
    auto put = [&](int64_t to) {
      uint8_t* const p = codes + to * code_row + at;
      if (at < code_row) {
        if constexpr (U == 4) *reinterpret_cast<uint4*>(p) = make_uint4(word[0], word[1], word[2], word[3]);
        else *reinterpret_cast<uint32_t*>(p) = word[0];
      }
      if (U == 4 || (lane & 3) == 0) scales[to * scale_row + sat] = (uint8_t)byte[0];
    };
    if (inv == nullptr) {
      put(c.row);
    } else {
      for (int j = 0; j < top_k; ++j) {
        const int64_t to = inv[c.row * top_k + j];
        if (to >= 0) put(to);
      }
    }
  }
}

// The rows of a gradient that no expert owns, for mx_dequantize_kernel to clear in passing: rows
// *end .. n_rows - 1 of k values at p.
template <typename T> struct MxTail {
  const int32_t* end = nullptr;
  T* p = nullptr;
  int64_t n_rows = 0;

  __device__ __forceinline__ void clear(int k) const {
    const int64_t stride = (int64_t)gridDim.x * kMxThreads;
    for (int64_t i = (int64_t)max(*end, 0) * k + (int64_t)blockIdx.x * kMxThreads + threadIdx.x;
         i < n_rows * k; i += stride)
      p[i] = Elem<T>::from_acc(0.f);
  }
};

template <typename T, int N, int U>
__global__ __launch_bounds__(kMxThreads) void mx_dequantize_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n_rows, int k,
    T* __restrict__ out, MxTail<T> tail) {
  if (tail.p) tail.clear(k);
  const int lane = threadIdx.x & (kWave - 1);
  const int chunks = (k + kMxChunk - 1) / kMxChunk;
  const int64_t code_row = mx_code_bytes(k), scale_row = mx_scale_bytes(k);
  const int64_t items = n_rows * chunks, stride = (int64_t)gridDim.x * kMxWaves * U;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  for (int64_t it = ((int64_t)blockIdx.x * kMxWaves + wave) * U; it < items; it += stride) {
    // the way of mx_quantize_kernel backwards: lane j fetches the block of chunk j
    const MxChunk c(min(it + (U == 4 ? lane & 3 : 0), items - 1), chunks);
    const int at = c.k / 2 + (U == 4 ? (lane >> 2) * 16 : lane * 4);
    const uint8_t* const p = codes + c.row * code_row + at;
    uint32_t word[U] = {};
    int byte = 0;
    if (at < code_row) {                  // (the row's scales reach at least as far)
      if constexpr (U == 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        word[0] = w.x; word[1] = w.y; word[2] = w.z; word[3] = w.w;
      } else {
        word[0] = *reinterpret_cast<const uint32_t*>(p);
      }
      byte = scales[c.row * scale_row + c.k / kMxBlock + (lane >> 2)];
    }
    if constexpr (U == 4) transpose_quad(word, lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (it + u >= items) break;
      const MxChunk d(it + u, chunks);
      const int first = d.k + lane * 8;
      const int b = U == 4 ? __shfl(byte, (lane & ~3) + u, kWave) : byte;
      float v[8];
      mx_values(word[u], b, v);
      if (first < k) store8<T, N>(out + d.row * k, first, k, v);
    }
  }
}

// Four chunks at a time where that leaves every CU several waves.
constexpr int64_t kMxManyItems = 256 * 32;
struct MxGrid {
  bool many;
  unsigned blocks;
  MxGrid(int64_t rows, int k) {
    const int64_t items = rows * ((k + kMxChunk - 1) / kMxChunk);
    many = items >= kMxManyItems;
    const int64_t per_block = kMxWaves * (many ? 4 : 1);
    blocks = (unsigned)std::max<int64_t>(std::min<int64_t>((items + per_block - 1) / per_block, 256 * 64), 1);
  }
};

// The longest run (of at most 16 bytes) that every row holds a whole number of, at its alignment.
template <typename T> static int run_length(const void* p, int k) {
  int n = 16 / (int)sizeof(T);
  while (n > 1 && (k % n || (uintptr_t)p % (n * sizeof(T)))) n /= 2;
  return n;
}
#define FMOE_RUN(CALL, N)          \
  do {                             \
    if (g.many) CALL(N, 4);        \
    else CALL(N, 1);               \
  } while (0)
#define FMOE_RUNS(CALL)                                             \
  do {                                                              \
    constexpr int kMost = 16 / (int)sizeof(T);                      \
    if (run == 8) FMOE_RUN(CALL, kMost);                            \
    else if (run == 4) FMOE_RUN(CALL, 4);                           \
    else if (run == 2) FMOE_RUN(CALL, 2);                           \
    else FMOE_RUN(CALL, 1);                                         \
  } while (0)

template <typename T>
static int launch_quantize(const void* x, int64_t n_rows, int k, const int32_t* n_rows_dev,
                           const int32_t* inv, int top_k, uint8_t* codes, uint8_t* scales,
                           const MxSegments& segments, hipStream_t s) {
  const int run = run_length<T>(x, k);
  const MxGrid g(n_rows, k);
  const dim3 grid(g.blocks);
#define FMOE_CALL(N, U)                                                                          \
  hipLaunchKernelGGL((mx_quantize_kernel<T, N, U>), grid, dim3(kMxThreads), 0, s, (const T*)x, \
                     n_rows, k, n_rows_dev, inv, top_k, codes, scales, segments)
  FMOE_RUNS(FMOE_CALL);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("mx_quantize");
  return FMOE_OK;
}

template <typename T>
static int launch_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t n_rows, int k,
                             void* out, const int32_t* tail_end, void* tail, int64_t tail_rows,
                             hipStream_t s) {
  const int run = run_length<T>(out, k);
  const MxGrid g(n_rows, k);
  const dim3 grid(g.blocks);
#define FMOE_CALL(N, U)                                                                        \
  hipLaunchKernelGGL((mx_dequantize_kernel<T, N, U>), grid, dim3(kMxThreads), 0, s, codes,   \
                     scales, n_rows, k, (T*)out, MxTail<T>{tail_end, (T*)tail, tail_rows})
  FMOE_RUNS(FMOE_CALL);
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

static int dequantize(const void* codes, const void* scales, int64_t n_rows, int64_t k, void* out,
                      const int32_t* tail_end, void* tail, int64_t tail_rows, int dtype,
                      hipStream_t s) {
  FMOE_REQUIRE(n_rows >= 0 && k >= 1 && k <= FMOE_MX_MAX_FEATURES, FMOE_ERR_INVALID,
               "mx_dequantize: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "mx_dequantize: unsupported dtype %d", dtype);
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(codes && scales && out, FMOE_ERR_INVALID, "mx_dequantize: null pointer");
  FMOE_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, FMOE_ERR_INVALID,
               "mx_dequantize: codes and scales must be 16-byte aligned");
  const uint8_t *c = (const uint8_t*)codes, *sc = (const uint8_t*)scales;
  switch (dtype) {
    case FMOE_F32:
      return launch_dequantize<float>(c, sc, n_rows, (int)k, out, tail_end, tail, tail_rows, s);
    case FMOE_F16:
      return launch_dequantize<__half>(c, sc, n_rows, (int)k, out, tail_end, tail, tail_rows, s);
    default:
      return launch_dequantize<__hip_bfloat16>(c, sc, n_rows, (int)k, out, tail_end, tail, tail_rows, s);
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
  return fmoe::dequantize(codes, scales, n_rows, features, out, nullptr, nullptr, 0, dtype,
                          (hipStream_t)stream);
}

extern "C" int fmoe_mx_dequantize_bwd(const void* w_codes, const void* w_scales,
                                      const int32_t* seg_off, void* w, void* dx, int64_t n_rows,
                                      int64_t in_feat, int64_t out_feat, int64_t n_expert,
                                      int dtype, void* stream) {
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && n_expert >= 1 && n_expert < INT32_MAX &&
                   out_feat >= 1 && out_feat <= FMOE_MX_MAX_FEATURES,
               FMOE_ERR_INVALID, "mx_dequantize_bwd: bad sizes");
  FMOE_REQUIRE(seg_off && (dx || n_rows == 0), FMOE_ERR_INVALID, "mx_dequantize_bwd: null pointer");
  return fmoe::dequantize(w_codes, w_scales, n_expert * out_feat, in_feat, w, seg_off + n_expert,
                          n_rows ? dx : nullptr, n_rows, dtype, (hipStream_t)stream);
}
