// Tokens sorted by expert and back where a truth value per (token, expert) says who takes whom, so
// that a token may go to any number of experts (experts that choose their tokens, thresholds):
//   rows are numbered expert by expert, an expert's in token order;
//   expand  rows[r(t, e)] = w[t][e] x[t]               (dw[t][e] = <x[t], given[r]>)
//   reduce  y[t] = sum_e w[t][e] rows[r(t, e)]          (dw[t][e] = <given[t], rows[r]>)
// Each is the other's gradient, the product for dw taken while the row is at hand.
//
// Both move rows and are bound by HBM (131072 rows of 16384 tokens, 2048 in bf16: summed up 103 us,
// 604 MB at 5.9 TB/s; expanded with the weights' gradient 204, 1.15 GB at 5.6; that gradient alone
// 94).  They go token by token, along a list of each token's (row, expert) pairs, so that x[t] is read
// once for all its rows and a sum needs no atomics: its order is that of the experts, always.
#include <algorithm>

#include "gemm_tiles.h"
#include "rows.h"

namespace fmoe {

// ------------------------------------------------------------------------- plan
// Two launches, or one for up to 64 tokens: a histogram per block of tokens, then, in every block,
// the sums of the histograms in front of its own and of all, and the places of its own tokens.
//
// A wave takes up to 16 tokens in a round.  Their truth values pass through LDS into one 16-bit mask
// per expert, which a lane holds; from there on a token's row is the expert's first one plus the bits
// below the token's in the mask, and its place in the token's list the bits below the lane's in a
// ballot, so that no step waits for the one before (a counter per expert in LDS, advanced token by
// token, took 11 us for 8192 tokens of 16 experts where this takes 7.8).
constexpr int kMapThreads = 1024;
constexpr int kMapWaves = kMapThreads / kWave;
constexpr int kMapRound = 16;          // most tokens of a wave at a time
constexpr int kMapUnit = 64;           // tokens of the smallest block, 4 for each wave
constexpr int kMapBlocks = 256;        // at most; more tokens make more rounds
constexpr int kMapStage = 2048;        // bytes of truth values a wave holds in LDS
constexpr int64_t kMapMostTokens = (int64_t)1 << 23;    // a block's counts have 16 bits
constexpr int64_t kMapMostPieces = (int64_t)1 << 26;
static_assert(FMOE_MAP_MAX_EXPERTS <= kMapStage, "a token's truth values fit");
static_assert(kMapMostTokens / kMapBlocks < 65536, "counts fit");

struct MapBlocks {
  int per_block, per_wave, blocks;     // tokens of a block and of a wave; blocks
  explicit MapBlocks(int64_t n_tokens) {
    const int64_t units = std::max<int64_t>((n_tokens + kMapUnit - 1) / kMapUnit, 1);
    const int64_t waves = std::min<int64_t>(units, kMapBlocks) * kMapWaves;
    per_wave = std::max((int)((n_tokens + waves - 1) / waves), 1);
    per_block = per_wave * kMapWaves;
    blocks = (int)((n_tokens + per_block - 1) / per_block);
  }
};
__host__ __device__ inline int map_hist_row(int n_expert) { return (n_expert + 7) & ~7; }

// A wave's tokens and its part of LDS.
struct MapWave {
  const uint8_t* map;
  uint8_t* stage;                      // [kMapStage]
  uint16_t* mask;                      // [n_expert]: the round's tokens that an expert takes
  int n_expert, lane;
  int first, end;                      // its tokens

  __device__ __forceinline__ MapWave(const uint8_t* map_, int n_tokens, int n_expert_,
                                     const MapBlocks& b, uint8_t* stages, uint16_t* masks) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    map = map_;
    stage = stages + wave * kMapStage;
    mask = masks + wave * n_expert_;
    n_expert = n_expert_;
    lane = threadIdx.x & (kWave - 1);
    first = min((int)blockIdx.x * b.per_block + wave * b.per_wave, n_tokens);
    end = min(first + b.per_wave, n_tokens);
  }

  // The masks of tokens t .. t + n - 1 (n <= kMapRound).
  __device__ __forceinline__ void round(int t, int n) {
    const int batch = min(kMapStage / n_expert, n);
    for (int at = 0; at < n; at += batch) {
      const int tokens = min(batch, n - at), bytes = tokens * n_expert;
      const uint8_t* const src = map + (int64_t)(t + at) * n_expert;
      for (int i = lane * 16; i < bytes; i += kWave * 16) {
        if (i + 16 <= bytes) {
          uint4 v;
          __builtin_memcpy(&v, src + i, 16);
          *reinterpret_cast<uint4*>(stage + i) = v;
        } else {
          for (int j = i; j < bytes; ++j) stage[j] = src[j];
        }
      }
      wave_fence();
      for (int e = lane; e < n_expert; e += kWave) {
        uint32_t m = at == 0 ? 0 : mask[e];
#pragma unroll
        for (int i = 0; i < kMapRound; ++i) {
          if (i >= tokens) break;
          m |= (uint32_t)(stage[i * n_expert + e] != 0) << (at + i);
        }
        mask[e] = (uint16_t)m;
      }
      wave_fence();
    }
  }
  // (a wave's LDS accesses run in order; this keeps the compiler's order, too)
  static __device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
};

__global__ __launch_bounds__(kMapThreads) void map_count_kernel(const uint8_t* __restrict__ map,
                                                                int n_tokens, int n_expert,
                                                                MapBlocks b,
                                                                uint16_t* __restrict__ hist) {
  extern __shared__ __align__(16) uint8_t lds[];
  uint16_t* const masks = (uint16_t*)(lds + kMapWaves * kMapStage);
  const int row = map_hist_row(n_expert);
  int32_t* const count = (int32_t*)(masks + kMapWaves * row);
  MapWave w(map, n_tokens, n_expert, b, lds, masks);
  for (int e = threadIdx.x; e < row; e += kMapThreads) count[e] = 0;
  __syncthreads();
  for (int t = w.first; t < w.end; t += kMapRound) {
    w.round(t, min(kMapRound, w.end - t));
    for (int e = w.lane; e < n_expert; e += kWave)
      if (const int c = __popc(w.mask[e])) atomicAdd(&count[e], c);       // (integers: any order)
  }
  __syncthreads();
  for (int e = threadIdx.x; e < row; e += kMapThreads)
    hist[(int64_t)blockIdx.x * row + e] = (uint16_t)count[e];
}

__global__ __launch_bounds__(kMapThreads) void map_place_kernel(
    const uint8_t* __restrict__ map, int n_tokens, int n_expert, int max_rows, MapBlocks b,
    const uint16_t* __restrict__ hist, int64_t* __restrict__ counts, int32_t* __restrict__ seg_off,
    int32_t* __restrict__ token_off, int2* __restrict__ pairs) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int row = map_hist_row(n_expert);
  uint16_t* const masks = (uint16_t*)(lds + kMapWaves * kMapStage);
  uint16_t* const taken = masks + kMapWaves * row;             // [waves][n_expert]
  int32_t* const total = (int32_t*)(taken + kMapWaves * row);  // [row] tokens of an expert
  int32_t* const before = total + row;                         // [row] of those, in earlier blocks
  MapWave w(map, n_tokens, n_expert, b, lds, masks);
  const int lane = w.lane, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  uint16_t* const mine = taken + wave * n_expert;

  for (int e = threadIdx.x; e < row; e += kMapThreads) total[e] = before[e] = 0;
  for (int e = lane; e < n_expert; e += kWave) mine[e] = 0;
  for (int t = w.first; t < w.end; t += kMapRound) {
    w.round(t, min(kMapRound, w.end - t));
    for (int e = lane; e < n_expert; e += kWave) mine[e] += (uint16_t)__popc(w.mask[e]);
  }
  __syncthreads();
  if (hist) {
    const int packs = row / 8;                       // (at most 128)
    const int p = threadIdx.x % packs, from = threadIdx.x / packs, step = kMapThreads / packs;
    int32_t all[8] = {}, front[8] = {};
    if (from < step) {
#pragma unroll 8
      for (int k = from; k < b.blocks; k += step) {
        const uint4 v = *reinterpret_cast<const uint4*>(hist + (int64_t)k * row + p * 8);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
        const bool in_front = k < (int)blockIdx.x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t c = (int32_t)((u[i >> 1] >> (16 * (i & 1))) & 0xffffu);
          all[i] += c;
          front[i] += in_front ? c : 0;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {                  // (integers: any order)
        if (all[i]) atomicAdd(&total[p * 8 + i], all[i]);
        if (front[i]) atomicAdd(&before[p * 8 + i], front[i]);
      }
    }
  }
  // every wave's counts become those of the waves in front of it
  for (int e = threadIdx.x; e < n_expert; e += kMapThreads) {
    int c[kMapWaves], sum = 0;
#pragma unroll
    for (int k = 0; k < kMapWaves; ++k) c[k] = taken[k * n_expert + e];
#pragma unroll
    for (int k = 0; k < kMapWaves; ++k) {
      taken[k * n_expert + e] = (uint16_t)sum;
      sum += c[k];
    }
    if (!hist) total[e] = sum;
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
  // pairs of the tokens in front of the wave's (rows from max_rows on are nobody's)
  int pairs_before = 0;
  for (int e = lane; e < n_expert; e += kWave)
    pairs_before += min(before[e] + mine[e], max(max_rows - total[e], 0));
  int at = __builtin_amdgcn_readlane(wave_inclusive_sum(pairs_before), kWave - 1);
  const unsigned long long below = (1ull << lane) - 1;
  const bool one_round = w.end - w.first <= kMapRound;
  for (int t = w.first; t < w.end; t += kMapRound) {
    const int n = min(kMapRound, w.end - t);
    if (!one_round) w.round(t, n);
    // lane i: pairs of token i
    int tokens = 0;
    for (int e0 = 0; e0 < n_expert; e0 += kWave) {
      const int e = e0 + lane;
      uint32_t m = 0;
      if (e < n_expert) {
        m = w.mask[e];
        const int fit = max(max_rows - (total[e] + before[e] + mine[e]), 0);
        if (__popc(m) > fit) {                       // the last ones are cut off
          while (__popc(m) > fit) m &= ~(1u << (31 - __clz(m)));
          w.mask[e] = (uint16_t)m;
        }
      }
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int c = __popcll(__ballot((m >> i) & 1));
        tokens += lane == i ? c : 0;
      }
    }
    const int incl = wave_inclusive_sum(tokens);
    int start = at + incl - tokens;
    if (lane < n) token_off[t + lane] = start;
    at += __builtin_amdgcn_readlane(incl, kWave - 1);
    for (int e0 = 0; e0 < n_expert; e0 += kWave) {
      const int e = e0 + lane;
      uint32_t m = 0;
      int r = 0;
      if (e < n_expert) {
        m = w.mask[e];
        r = total[e] + before[e] + mine[e];
        mine[e] += (uint16_t)__popc(m);
      }
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const bool takes = (m >> i) & 1;
        const unsigned long long all = __ballot(takes);
        const int to = __builtin_amdgcn_readlane(start, i) + __popcll(all & below);
        if (takes) pairs[to] = make_int2(r + __popc(m & ((1u << i) - 1)), e);
        start += lane == i ? __popcll(all) : 0;
      }
    }
  }
  if (lane == 0 && w.end == n_tokens && w.first < n_tokens) token_off[n_tokens] = at;
}

constexpr size_t map_lds(int n_expert, bool place) {
  const int row = (n_expert + 7) & ~7;
  return kMapWaves * kMapStage + (size_t)row * (place ? 2 * kMapWaves * 2 + 8 : kMapWaves * 2 + 4);
}

// ------------------------------------------------------------------------- rows
struct MapMoveArgs {
  const void *one, *many, *weight;     // [tokens, d], [rows, d], [tokens, experts] or null (ones)
  const int32_t* token_off;
  const int2* pairs;
  void *out, *dweight;
  int64_t n_tokens;
  int d, n_expert;
};

// EXPAND: out[r] = w one[t] for a token's rows; else out[t] = sum of w many[r].  DOT: also
// dweight[t][e] = <one[t], many[r]>, zero where the token has no row; out may be null then.
//
// A lane holds 8 values of a piece of a row, and U rows are under way at a time.  Without DOT a wave takes 512
// values of a token's rows, whatever their length; with it a block of G threads takes a token,
// H times 8 G values at a time, and its waves' shares of the products meet in LDS.
template <typename T, typename W, int G, int H, bool EXPAND, bool DOT>
__global__ __launch_bounds__(DOT ? G : 256) void map_move_kernel(MapMoveArgs a, ClearedTail<T> tail) {
  static_assert(DOT || (G == kWave && H == 1), "pieces of 512 values");
  if (EXPAND && tail.p) tail.clear(a.d);
  extern __shared__ float s_dot[];                   // [waves][n_expert]
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  constexpr int kSpan = G * 8, kPiece = kSpan * H;
  int64_t t = blockIdx.x;
  int k0 = 0;
  if constexpr (!DOT) {
    const int pieces = (a.d + kPiece - 1) / kPiece;
    const uint32_t item = blockIdx.x * (256 / kWave) + wave;      // (below 2^26)
    t = item / (uint32_t)pieces;
    k0 = (int)(item - (uint32_t)t * pieces) * kPiece;
    if (t >= a.n_tokens) return;
  }
  const T* const one = (const T*)a.one + t * a.d;
  const T* const many = (const T*)a.many;
  const W* const weight = (const W*)a.weight;
  T* const out = (T*)a.out;
  const bool wanted = !DOT || out != nullptr;
  const int p0 = a.token_off[t], p1 = a.token_off[t + 1];
  float* const dot = s_dot + wave * a.n_expert;
  if constexpr (DOT)
    for (int e = lane; e < a.n_expert; e += kWave) dot[e] = 0.f;
  // (a lane's values are runs of 16 bytes, so that a wave's stores are whole lines in f32, too)
  constexpr int kGap = G * Eight<T>::N;
  const int at = (threadIdx.x & (G - 1)) * Eight<T>::N;
  const int k_end = DOT ? a.d : k0 + 1;
  for (; k0 < k_end; k0 += kPiece) {
    float x[H][8], sum[H][8];
    if constexpr (EXPAND || DOT) {
      Eight<T> raw[H];
#pragma unroll
      for (int h = 0; h < H; ++h) raw[h].load(one, k0 + h * kSpan + at, a.d, kGap);
#pragma unroll
      for (int h = 0; h < H; ++h) raw[h].widen(x[h]);
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
      constexpr int U = EXPAND && !DOT ? 1 : 16 / (int)sizeof(T) / H;     // rows under way
      for (int j = 0; j < n; j += U) {
        Eight<T> raw[U][H];
        if constexpr (!EXPAND || DOT) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (j + u >= n) break;
            const int64_t r = __builtin_amdgcn_readlane(pair.x, j + u);
#pragma unroll
            for (int h = 0; h < H; ++h)
              raw[u][h].template load<true>(many + r * a.d, k0 + h * kSpan + at, a.d, kGap);
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
              for (int i = 0; i < 8; ++i) s = fmaf(x[h][i], raw[u][h][i], s);
            s = wave_sum(s);
            const int e = __builtin_amdgcn_readlane(pair.y, j + u);
            if (lane == 0) dot[e] = k0 == 0 ? s : dot[e] + s;
          }
#pragma unroll
          for (int h = 0; h < H; ++h) {
            if constexpr (EXPAND) {
              if (!wanted) continue;
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                v[i] = x[h][i] * wj;
                // (an f32 product, always: with the conversion to f16 the compiler would make it one
                // instruction with one rounding, here and there, and a gradient's bits would depend on
                // which others are wanted)
                if constexpr (std::is_same<T, __half>::value) asm("" : "+v"(v[i]));
              }
              Eight<T>::template store<true>(out + r * a.d, k0 + h * kSpan + at, a.d, v, kGap);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                sum[h][i] = fmaf(raw[u][h][i], wj, sum[h][i]);
            }
          }
        }
      }
    }
    if (!EXPAND && wanted) {
#pragma unroll
      for (int h = 0; h < H; ++h) Eight<T>::store(out + t * a.d, k0 + h * kSpan + at, a.d, sum[h], kGap);
    }
  }
  if constexpr (DOT) {
    __syncthreads();
    W* const dw = (W*)a.dweight + t * a.n_expert;
    for (int e = threadIdx.x; e < a.n_expert; e += G) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < G / kWave; ++w) s += s_dot[w * a.n_expert + e];
      dw[e] = Elem<W>::from_acc(s);
    }
  }
}

template <typename T, typename W, int G, int H, bool EXPAND, bool DOT>
static void start_move(const MapMoveArgs& a, const ClearedTail<T>& tail, hipStream_t s) {
  const int64_t waves = a.n_tokens * ((a.d + kWave * 8 - 1) / (kWave * 8));
  const dim3 grid((unsigned)(DOT ? a.n_tokens : (waves + 3) / 4)), block(DOT ? G : 256);
  const size_t lds = DOT ? sizeof(float) * (G / kWave) * a.n_expert : 0;
  hipLaunchKernelGGL((map_move_kernel<T, W, G, H, EXPAND, DOT>), grid, block, lds, s, a, tail);
}

template <typename T, typename W, bool EXPAND, bool DOT>
static int launch_move(const MapMoveArgs& a, const ClearedTail<T>& tail, hipStream_t s) {
  if constexpr (DOT) {
    if (a.d <= 512) start_move<T, W, 64, 1, EXPAND, true>(a, tail, s);
    else if (a.d <= 1024) start_move<T, W, 128, 1, EXPAND, true>(a, tail, s);
    else if (a.d <= 2048) start_move<T, W, 256, 1, EXPAND, true>(a, tail, s);
    else start_move<T, W, 256, 2, EXPAND, true>(a, tail, s);
  } else {
    start_move<T, W, 64, 1, EXPAND, false>(a, tail, s);
  }
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
  FMOE_REQUIRE(a.n_tokens >= 0 && a.n_tokens <= kMapMostTokens && a.d >= 1 && a.n_expert >= 1 &&
                   a.n_expert <= FMOE_MAP_MAX_EXPERTS && max_rows >= 0 && max_rows < INT32_MAX,
               FMOE_ERR_INVALID, "%s: bad sizes", name);
  // (a wave for each piece of 512 values, and fewer than 2^32 threads in a launch; with dweight it is a
  // block for each token)
  FMOE_REQUIRE(a.dweight || a.n_tokens * ((a.d + 511) / 512) < kMapMostPieces, FMOE_ERR_UNSUPPORTED,
               "%s: %lld tokens of %d features: tokens times ceil(features / 512) must be below 2^26",
               name, (long long)a.n_tokens, a.d);
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "%s: unsupported dtype %d", name, dtype);
  FMOE_REQUIRE(weight_dtype == FMOE_F32 || weight_dtype == dtype, FMOE_ERR_UNSUPPORTED,
               "%s: weights must be f32 or of the rows' dtype", name);
  if (a.n_tokens == 0) return FMOE_OK;
  // (rows of a plan without any may be null)
  FMOE_REQUIRE(a.token_off && (a.pairs || max_rows == 0) &&
                   (EXPAND ? a.one && (a.out || a.dweight || max_rows == 0)
                           : (a.many || max_rows == 0) && (a.out || a.dweight)),
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
  FMOE_REQUIRE(n_tokens >= 0 && n_tokens <= kMapMostTokens && n_expert >= 1 &&
                   n_expert <= FMOE_MAP_MAX_EXPERTS && n_tokens <= INT32_MAX / n_expert,
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
  uint16_t* const hist = b.blocks > 1 ? (uint16_t*)workspace : nullptr;
  FMOE_SET_DYNAMIC_LDS_ONCE(map_count_kernel, map_lds(FMOE_MAP_MAX_EXPERTS, false));
  FMOE_SET_DYNAMIC_LDS_ONCE(map_place_kernel, map_lds(FMOE_MAP_MAX_EXPERTS, true));
  if (hist)
    hipLaunchKernelGGL(map_count_kernel, dim3(b.blocks), dim3(kMapThreads), map_lds(n_expert, false),
                       s, map, (int)n_tokens, n_expert, b, hist);
  FMOE_LAUNCH_CHECK("map_count");
  hipLaunchKernelGGL(map_place_kernel, dim3(b.blocks), dim3(kMapThreads), map_lds(n_expert, true), s,
                     map, (int)n_tokens, n_expert, (int)max_rows, b, hist, counts, seg_off, token_off,
                     (int2*)pairs);
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
