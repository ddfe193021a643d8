// Tokens sorted by expert and back where a truth value per (token, expert) says who takes whom, so
// that a token may go to any number of experts (experts that choose their tokens, thresholds):
//   rows are numbered expert by expert, an expert's in token order;
//   expand  rows[r(t, e)] = w[t][e] x[t]               (dw[t][e] = <x[t], given[r]>)
//   reduce  y[t] = sum_e w[t][e] rows[r(t, e)]          (dw[t][e] = <given[t], rows[r]>)
// Each is the other's gradient, the product for dw taken while the row is at hand.
//
// Both move rows and are bound by HBM.  They go token by token, along a list of each token's
// (row, expert) pairs, so that x[t] is read once for all its rows and a sum needs no atomics: its
// order is that of the experts, always.
#include <algorithm>

#include "gemm_tiles.h"
#include "rows.h"

namespace fmoe {

constexpr int kMapThreads = 256;
constexpr int kMapWaves = kMapThreads / kWave;

// ------------------------------------------------------------------------- plan
// Two launches, or one for up to kMapUnit tokens: a histogram per block of tokens, then, in every
// block, the sums of the histograms in front of its own and of all (16-bit counts, 16 bytes a load:
// 16384 tokens of 128 experts are 64 KiB a block, from L2) and the places of its own tokens.
constexpr int kMapUnit = 64;           // tokens of the smallest block
constexpr int kMapBlocks = 256;        // at most; more tokens make larger blocks
constexpr int kMapStage = 4096;        // bytes of truth values a wave holds in LDS
static_assert(FMOE_MAP_MAX_EXPERTS <= 1024 && FMOE_MAP_MAX_EXPERTS <= kMapStage, "a token's fit");

struct MapBlocks {
  int per_block, per_wave, blocks;     // tokens of a block and of a wave; blocks
  __host__ __device__ explicit MapBlocks(int64_t n_tokens) {
    const int64_t units = (n_tokens + kMapUnit - 1) / kMapUnit;
    per_block = (int)((units + kMapBlocks - 1) / kMapBlocks) * kMapUnit;
    if (per_block == 0) per_block = kMapUnit;
    per_wave = per_block / kMapWaves;
    blocks = (int)((n_tokens + per_block - 1) / per_block);
  }
};
__host__ __device__ inline int map_hist_row(int n_expert) { return (n_expert + 7) & ~7; }

// A wave's truth values, `batch` tokens at a time, through its own LDS.
struct MapStage {
  const uint8_t* map;
  uint8_t* lds;
  int n_expert, batch;
  int64_t end;                         // one behind the wave's last token
  int64_t at = -1;                     // first token held

  // (whole wave) the tokens t .. held() - 1
  __device__ __forceinline__ void hold(int64_t t, int lane) {
    if (t == at) return;
    at = t;
    const int bytes = (int)(min(t + batch, end) - t) * n_expert;
    const uint8_t* const src = map + t * n_expert;
    for (int i = lane * 16; i < bytes; i += kWave * 16) {
      if (i + 16 <= bytes) {
        uint4 v;
        __builtin_memcpy(&v, src + i, 16);
        *reinterpret_cast<uint4*>(lds + i) = v;
      } else {
        for (int j = i; j < bytes; ++j) lds[j] = src[j];
      }
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __device__ __forceinline__ int64_t held() const { return min(at + batch, end); }
  __device__ __forceinline__ bool takes(int64_t t, int e) const {
    return e < n_expert && lds[(int)(t - at) * n_expert + e] != 0;
  }
};

// Tokens that the wave's experts take, counted into cnt[0 .. n_expert - 1].
__device__ __forceinline__ void map_count(MapStage& st, int64_t first, int32_t* cnt, int lane) {
  for (int e = lane; e < st.n_expert; e += kWave) cnt[e] = 0;
  for (int64_t t = first; t < st.end; t = st.held()) {
    st.hold(t, lane);
    const int64_t stop = st.held();
    for (int e = lane; e < st.n_expert; e += kWave) {
      int c = 0;
      for (int64_t u = t; u < stop; ++u) c += st.takes(u, e);
      cnt[e] += c;
    }
  }
}

__device__ __forceinline__ MapStage map_stage(const uint8_t* map, uint8_t* lds, int64_t n_tokens,
                                              int n_expert, const MapBlocks& b, int wave,
                                              int64_t& first) {
  first = min((int64_t)blockIdx.x * b.per_block + wave * b.per_wave, n_tokens);
  MapStage st;
  st.map = map;
  st.lds = lds + wave * kMapStage;
  st.n_expert = n_expert;
  st.batch = kMapStage / n_expert;
  st.end = min(first + b.per_wave, n_tokens);
  return st;
}

__global__ __launch_bounds__(kMapThreads) void map_count_kernel(const uint8_t* __restrict__ map,
                                                                int64_t n_tokens, int n_expert,
                                                                uint16_t* __restrict__ hist) {
  __shared__ __align__(16) uint8_t stage[kMapWaves * kMapStage];
  extern __shared__ int32_t cnt[];     // [waves][n_expert]
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const MapBlocks b(n_tokens);
  int64_t first;
  MapStage st = map_stage(map, stage, n_tokens, n_expert, b, wave, first);
  map_count(st, first, cnt + wave * n_expert, lane);
  __syncthreads();
  const int row = map_hist_row(n_expert);
  for (int e = threadIdx.x; e < row; e += kMapThreads) {
    int c = 0;
    if (e < n_expert)
      for (int w = 0; w < kMapWaves; ++w) c += cnt[w * n_expert + e];
    hist[(int64_t)blockIdx.x * row + e] = (uint16_t)c;
  }
}

__global__ __launch_bounds__(kMapThreads) void map_place_kernel(
    const uint8_t* __restrict__ map, int64_t n_tokens, int n_expert, int max_rows,
    const uint16_t* __restrict__ hist, int64_t* __restrict__ counts, int32_t* __restrict__ seg_off,
    int32_t* __restrict__ token_off, int2* __restrict__ pairs) {
  __shared__ __align__(16) uint8_t stage[kMapWaves * kMapStage];
  extern __shared__ int32_t lds[];
  const int row = map_hist_row(n_expert);
  int32_t* const cnt = lds;                          // [waves][n_expert]
  int32_t* const total = cnt + kMapWaves * n_expert; // [row] tokens of an expert
  int32_t* const before = total + row;               // [row] of those, in blocks in front
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const MapBlocks b(n_tokens);
  int64_t first;
  MapStage st = map_stage(map, stage, n_tokens, n_expert, b, wave, first);

  for (int e = threadIdx.x; e < row; e += kMapThreads) total[e] = before[e] = 0;
  map_count(st, first, cnt + wave * n_expert, lane);
  __syncthreads();
  if (hist == nullptr) {
    for (int e = threadIdx.x; e < n_expert; e += kMapThreads)
      for (int w = 0; w < kMapWaves; ++w) total[e] += cnt[w * n_expert + e];
  } else {
    const int packs = row / 8;                       // (at most 128)
    const int p = threadIdx.x % packs, from = threadIdx.x / packs, step = kMapThreads / packs;
    int32_t all[8] = {}, mine[8] = {};
    if (from < step) {
#pragma unroll 4
      for (int k = from; k < b.blocks; k += step) {
        const uint4 v = *reinterpret_cast<const uint4*>(hist + (int64_t)k * row + p * 8);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        const bool in_front = k < (int)blockIdx.x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t c = (int32_t)((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
          all[i] += c;
          mine[i] += in_front ? c : 0;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {                  // (integers: any order)
        atomicAdd(&total[p * 8 + i], all[i]);
        atomicAdd(&before[p * 8 + i], mine[i]);
      }
    }
  }
  __syncthreads();
  // first row of every expert, in total's place; all waves need them, one makes them
  if (wave == 0) {
    int carry = 0;
    for (int e0 = 0; e0 < n_expert; e0 += kWave) {
      const int e = e0 + lane, c = e < n_expert ? total[e] : 0;
      const int incl = wave_inclusive_sum(c);
      const int start = carry + incl - c;
      if (e < n_expert) {
        total[e] = start;
        if (blockIdx.x == 0) {
          seg_off[e] = min(start, max_rows);
          counts[e] = min(c, max(max_rows - start, 0));
        }
      }
      carry += __builtin_amdgcn_readlane(incl, kWave - 1);
    }
    if (blockIdx.x == 0 && lane == 0) seg_off[n_expert] = min(carry, max_rows);
  }
  __syncthreads();
  // The next row of the wave's experts, in LDS too (by the lane that alone uses it), and the number
  // of pairs of the tokens in front of the wave's.  Rows from max_rows on are nobody's.
  int32_t* const next = cnt + wave * n_expert;
  int pairs_before = 0;
  for (int e = lane; e < n_expert; e += kWave) {
    int c = before[e];
    for (int w = 0; w < wave; ++w) c += cnt[w * n_expert + e];
    pairs_before += min(c, max(max_rows - total[e], 0));
    before[row * (wave + 1) + e] = total[e] + c;     // (others still read cnt)
  }
  int at = __builtin_amdgcn_readlane(wave_inclusive_sum(pairs_before), kWave - 1);
  __syncthreads();
  for (int e = lane; e < n_expert; e += kWave) next[e] = before[row * (wave + 1) + e];
  const unsigned long long below = (1ull << lane) - 1;
  for (int64_t t = first; t < st.end;) {
    st.hold(t, lane);
    const int64_t stop = st.held();
    for (; t < stop; ++t) {
      if (lane == 0) token_off[t] = at;
      for (int e0 = 0; e0 < n_expert; e0 += kWave) {
        const int e = e0 + lane;
        const bool takes = st.takes(t, e);
        int r = 0;
        if (takes) {
          r = next[e];
          next[e] = r + 1;
        }
        const bool kept = takes && r < max_rows;
        const unsigned long long all = __ballot(kept);
        if (kept) pairs[at + __popcll(all & below)] = make_int2(r, e);
        at += __popcll(all);
      }
    }
  }
  if (lane == 0 && st.end == n_tokens && first < n_tokens) token_off[n_tokens] = at;
}

// ------------------------------------------------------------------------- rows
// 8 values of a row from k on (zeros behind its end), rows of any alignment.
template <typename T>
__device__ __forceinline__ void load_any(const T* row, int k, int d, T (&v)[8]) {
  if (k + 8 <= d) {
    __builtin_memcpy(v, row + k, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < d ? row[k + i] : Elem<T>::from_acc(0.f);
  }
}
template <typename T>
__device__ __forceinline__ void store_any(T* row, int k, int d, const float (&v)[8]) {
  T o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = Elem<T>::from_acc(v[i]);
  if (k + 8 <= d) {
    __builtin_memcpy(row + k, o, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < d) row[k + i] = o[i];
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int s = kWave / 2; s > 0; s >>= 1) v += __shfl_xor(v, s, kWave);
  return v;
}

struct MapMoveArgs {
  const void *one, *many, *weight;     // [tokens, d], [rows, d], [tokens, experts] or null (ones)
  const int32_t* token_off;
  const int2* pairs;
  void *out, *dweight;
  int64_t n_tokens;
  int d, n_expert;
};

// EXPAND: out[r] = w one[t] for a token's rows; else out[t] = sum of w many[r].  DOT: also
// dweight[t][e] = <one[t], many[r]>, zero where the token has no row.  G threads take a token,
// `H` chunks of 8 G values of its row at a time; without DOT a row's pieces of H chunks may be
// different blocks' (blockIdx.y).
template <typename T, typename W, int G, int H, bool EXPAND, bool DOT>
__global__ __launch_bounds__(kMapThreads) void map_move_kernel(MapMoveArgs a, ClearedTail<T> tail) {
  if (EXPAND && tail.p && blockIdx.y == 0) tail.clear(a.d);
  extern __shared__ float s_dot[];                   // [waves][n_expert]
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t t = (int64_t)blockIdx.x * (kMapThreads / G) + (G == kWave ? wave : 0);
  // (with G = 64 no barrier follows; with G = 256 the whole block leaves)
  if (t >= a.n_tokens) return;
  const T* const one = (const T*)a.one + t * a.d;
  const T* const many = (const T*)a.many;
  const W* const weight = (const W*)a.weight;
  T* const out = (T*)a.out;
  const int p0 = a.token_off[t], p1 = a.token_off[t + 1];
  float* const dot = s_dot + wave * a.n_expert;
  if constexpr (DOT)
    for (int e = lane; e < a.n_expert; e += kWave) dot[e] = 0.f;
  constexpr int kSpan = G * 8, kPiece = kSpan * H;
  const int at = (threadIdx.x & (G - 1)) * 8;
  for (int k0 = blockIdx.y * kPiece; k0 < a.d; k0 += gridDim.y * kPiece) {
    float x[H][8], sum[H][8];
    if constexpr (EXPAND || DOT) {
      T raw[H][8];
#pragma unroll
      for (int h = 0; h < H; ++h) load_any(one, k0 + h * kSpan + at, a.d, raw[h]);
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[h][i] = Elem<T>::to_acc(raw[h][i]);
    }
    if constexpr (!EXPAND) {
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[h][i] = 0.f;
    }
    for (int b = p0; b < p1; b += kWave) {
      // a lane fetches a pair and its weight
      int2 pair = make_int2(0, 0);
      float w = 1.f;
      if (b + lane < p1) {
        pair = a.pairs[b + lane];
        if (weight) w = Elem<W>::to_acc(weight[t * a.n_expert + pair.y]);
      }
      const int n = min(p1 - b, kWave);
      constexpr int U = EXPAND ? (DOT ? 2 : 1) : 8 / H;       // rows under way at a time
      for (int j = 0; j < n; j += U) {
        T raw[U][H][8];
        if constexpr (!EXPAND || DOT) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int64_t r = __builtin_amdgcn_readlane(pair.x, min(j + u, n - 1));
#pragma unroll
            for (int h = 0; h < H; ++h) load_any(many + r * a.d, k0 + h * kSpan + at, a.d, raw[u][h]);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (j + u >= n) break;
          const int64_t r = __builtin_amdgcn_readlane(pair.x, j + u);
          const float wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), j + u));
          if constexpr (DOT) {
            float s = 0.f;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
              for (int i = 0; i < 8; ++i) s = fmaf(x[h][i], Elem<T>::to_acc(raw[u][h][i]), s);
            s = wave_sum(s);
            if (lane == 0) dot[__builtin_amdgcn_readlane(pair.y, j + u)] += s;
          }
#pragma unroll
          for (int h = 0; h < H; ++h) {
            if constexpr (EXPAND) {
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = x[h][i] * wj;
              store_any(out + r * a.d, k0 + h * kSpan + at, a.d, v);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                sum[h][i] = fmaf(Elem<T>::to_acc(raw[u][h][i]), wj, sum[h][i]);
            }
          }
        }
      }
    }
    if constexpr (!EXPAND) {
#pragma unroll
      for (int h = 0; h < H; ++h) store_any(out + t * a.d, k0 + h * kSpan + at, a.d, sum[h]);
    }
  }
  if constexpr (DOT) {
    W* const dw = (W*)a.dweight + t * a.n_expert;
    if constexpr (G == kWave) {
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int e = lane; e < a.n_expert; e += kWave) dw[e] = Elem<W>::from_acc(dot[e]);
    } else {
      __syncthreads();
      for (int e = threadIdx.x; e < a.n_expert; e += kMapThreads) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kMapWaves; ++w) s += s_dot[w * a.n_expert + e];
        dw[e] = Elem<W>::from_acc(s);
      }
    }
  }
}

// A wave takes a token where there are enough of them, a block otherwise.
constexpr int64_t kMapManyTokens = 256 * 8;

template <typename T, typename W, bool EXPAND, bool DOT>
static int launch_move(const MapMoveArgs& a, const ClearedTail<T>& tail, hipStream_t s) {
  const size_t lds = DOT ? sizeof(float) * kMapWaves * a.n_expert : 0;
  const bool wave = a.n_tokens >= kMapManyTokens;
  constexpr int kHWave = 4, kHBlock = 2;
  const int piece = wave ? kWave * 8 * kHWave : kMapThreads * 8 * kHBlock;
  const dim3 grid((unsigned)(wave ? (a.n_tokens + kMapWaves - 1) / kMapWaves : a.n_tokens),
                  DOT ? 1 : (unsigned)((a.d + piece - 1) / piece));
  if (wave)
    hipLaunchKernelGGL((map_move_kernel<T, W, kWave, kHWave, EXPAND, DOT>), grid, dim3(kMapThreads),
                       lds, s, a, tail);
  else
    hipLaunchKernelGGL((map_move_kernel<T, W, kMapThreads, kHBlock, EXPAND, DOT>), grid,
                       dim3(kMapThreads), lds, s, a, tail);
  FMOE_LAUNCH_CHECK(EXPAND ? "map_expand" : "map_reduce");
  return FMOE_OK;
}

template <typename T, typename W, bool EXPAND>
static int launch_dot(const MapMoveArgs& a, const ClearedTail<T>& tail, hipStream_t s) {
  return a.dweight ? launch_move<T, W, EXPAND, true>(a, tail, s)
                   : launch_move<T, W, EXPAND, false>(a, tail, s);
}

template <typename T, bool EXPAND>
static int launch_weight(const MapMoveArgs& a, bool wide, const ClearedTail<T>& tail, hipStream_t s) {
  return wide ? launch_dot<T, float, EXPAND>(a, tail, s) : launch_dot<T, T, EXPAND>(a, tail, s);
}

template <bool EXPAND>
static int move(const MapMoveArgs& a, int dtype, int weight_dtype, const int32_t* n_rows_dev,
                int64_t max_rows, hipStream_t s) {
  const char* const name = EXPAND ? "map_expand" : "map_reduce";
  FMOE_REQUIRE(a.n_tokens >= 0 && a.n_tokens < INT32_MAX && a.d >= 1 && a.n_expert >= 1 &&
                   a.n_expert <= FMOE_MAP_MAX_EXPERTS && max_rows >= 0 && max_rows < INT32_MAX,
               FMOE_ERR_INVALID, "%s: bad sizes", name);
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "%s: unsupported dtype %d", name, dtype);
  FMOE_REQUIRE(weight_dtype == FMOE_F32 || weight_dtype == dtype, FMOE_ERR_UNSUPPORTED,
               "%s: weights must be f32 or of the rows' dtype", name);
  if (a.n_tokens == 0) return FMOE_OK;
  // (rows of a plan without any may be null)
  FMOE_REQUIRE(a.token_off && (a.pairs || max_rows == 0) &&
                   (EXPAND ? a.one && (a.out || max_rows == 0) : (a.many || max_rows == 0) && a.out),
               FMOE_ERR_INVALID, "%s: null pointer", name);
  FMOE_REQUIRE(!a.dweight || (a.weight && a.one && (a.many || max_rows == 0)), FMOE_ERR_INVALID,
               "%s: a gradient of weights needs them, the tokens and the rows", name);
  const bool wide = weight_dtype == FMOE_F32;
  void* const cleared = EXPAND && n_rows_dev && max_rows ? a.out : nullptr;
  switch (dtype) {
    case FMOE_F32:
      return launch_dot<float, float, EXPAND>(a, {n_rows_dev, (float*)cleared, max_rows}, s);
    case FMOE_F16:
      return launch_weight<__half, EXPAND>(a, wide, {n_rows_dev, (__half*)cleared, max_rows}, s);
    default:
      return launch_weight<__hip_bfloat16, EXPAND>(a, wide, {n_rows_dev, (__hip_bfloat16*)cleared, max_rows}, s);
  }
}

}  // namespace fmoe

extern "C" int64_t fmoe_map_workspace_bytes(int64_t n_tokens, int32_t n_expert) {
  using namespace fmoe;
  FMOE_REQUIRE(n_tokens >= 0 && n_expert >= 1 && n_expert <= FMOE_MAP_MAX_EXPERTS &&
                   n_tokens <= INT32_MAX / n_expert,
               FMOE_ERR_INVALID, "map: bad sizes");
  const MapBlocks b(n_tokens);
  return b.blocks <= 1 ? 0 : (int64_t)b.blocks * map_hist_row(n_expert) * (int64_t)sizeof(uint16_t);
}

extern "C" int fmoe_map_plan(const uint8_t* map, int64_t n_tokens, int32_t n_expert,
                             int64_t max_rows, int64_t* counts, int32_t* seg_off,
                             int32_t* token_off, int32_t* pairs, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  using namespace fmoe;
  const int64_t need = fmoe_map_workspace_bytes(n_tokens, n_expert);
  if (need < 0) return (int)need;
  FMOE_REQUIRE(max_rows >= 0 && max_rows < INT32_MAX, FMOE_ERR_INVALID, "map_plan: bad sizes");
  FMOE_REQUIRE(n_tokens >= 1, FMOE_ERR_INVALID, "map_plan: no tokens");
  FMOE_REQUIRE(map && counts && seg_off && token_off && (pairs || max_rows == 0), FMOE_ERR_INVALID,
               "map_plan: null pointer");
  FMOE_REQUIRE((uintptr_t)pairs % 8 == 0, FMOE_ERR_INVALID, "map_plan: pairs must be 8-byte aligned");
  FMOE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
               FMOE_ERR_WORKSPACE, "map_plan: a workspace of %lld bytes, 16-byte aligned, is needed",
               (long long)need);
  hipStream_t s = (hipStream_t)stream;
  const MapBlocks b(n_tokens);
  const int row = map_hist_row(n_expert);
  uint16_t* const hist = b.blocks > 1 ? (uint16_t*)workspace : nullptr;
  const size_t counters = sizeof(int32_t) * kMapWaves * n_expert;
  if (hist)
    hipLaunchKernelGGL(map_count_kernel, dim3(b.blocks), dim3(kMapThreads), counters, s, map,
                       n_tokens, n_expert, hist);
  FMOE_LAUNCH_CHECK("map_count");
  hipLaunchKernelGGL(map_place_kernel, dim3(b.blocks), dim3(kMapThreads),
                     counters + sizeof(int32_t) * row * (2 + kMapWaves), s, map, n_tokens, n_expert,
                     (int)max_rows, hist, counts, seg_off, token_off, (int2*)pairs);
  FMOE_LAUNCH_CHECK("map_place");
  return FMOE_OK;
}

extern "C" int fmoe_map_expand(const void* tokens, const void* given, const void* weight,
                               const int32_t* token_off, const int32_t* pairs,
                               const int32_t* n_rows_dev, void* rows, void* dweight,
                               int64_t n_tokens, int64_t d, int32_t n_expert, int64_t max_rows,
                               int dtype, int weight_dtype, void* stream) {
  FMOE_REQUIRE(d >= 1 && d < INT32_MAX / 2, FMOE_ERR_INVALID, "map_expand: bad sizes");
  return fmoe::move<true>({tokens, given, weight, token_off, (const int2*)pairs, rows, dweight,
                           n_tokens, (int)d, n_expert},
                          dtype, weight_dtype, n_rows_dev, max_rows, (hipStream_t)stream);
}

extern "C" int fmoe_map_reduce(const void* rows, const void* given, const void* weight,
                               const int32_t* token_off, const int32_t* pairs, void* tokens,
                               void* dweight, int64_t n_tokens, int64_t d, int32_t n_expert,
                               int64_t max_rows, int dtype, int weight_dtype, void* stream) {
  FMOE_REQUIRE(d >= 1 && d < INT32_MAX / 2, FMOE_ERR_INVALID, "map_reduce: bad sizes");
  return fmoe::move<false>({given, rows, weight, token_off, (const int2*)pairs, tokens, dweight,
                            n_tokens, (int)d, n_expert},
                           dtype, weight_dtype, nullptr, max_rows, (hipStream_t)stream);
}
