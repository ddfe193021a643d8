// Scored top-k routing on gfx950: scores of the gate's logits, a choice biased and limited to
// the best groups of experts, the k chosen scores renormalised, and the gradient of the logits.
//
//   s = sigmoid(l)  or  softmax(l),   v = s + bias
//   the best `top_group` of `n_group` equal groups stay (value: the sum of a group's 1 or 2
//   best v); idx = the k best v of those, ties to the lower index
//   w_j = scale s_j / (sum of the chosen s + 1e-20),  or  scale s_j
// An expert whose v is -inf (a masked logit under sigmoid has the score 0, so the mask is taken
// from the logit itself) is never chosen; a slot with nobody left is -1 with weight 0.
//
// The arrays are a few MiB at most, so what counts is launch latency and the number of
// instructions per token.  16 lanes share a token (32 above 256 experts; all 64 with few tokens,
// see FMOE_SCORE_SHAPES), so a wave serves four; they hold all v in registers as 64-bit keys that
// order first by v, then by index: the f32 v widened to a double, whose 29 free mantissa bits
// take the index.  One v_max_f64 then is an arg-max with its tie rule, and a round of the
// selection is one such maximum per register, four rotations within the 16 lanes, and one
// comparison per register that drops the winner.
// Measured: 16384 tokens of 128 experts in f32, the best 3 of 8 groups, 10.8 us forward (the
// 10 MB it moves take 1.9; the rest is instructions) and 4.2 us backward; 64 tokens 4.8 and
// 2.5 us, of which an empty launch is 2.1.
#include <algorithm>

#include "common.h"

namespace fmoe {

constexpr int kScoreThreads = 256;
constexpr int kScoreMaxExperts = 512;
constexpr int kScoreMaxGroups = 64;
constexpr float kScoreEps = 1e-20f;

struct ScoreArgs {
  int64_t n_tokens;
  int n_expert, top_k, n_group, top_group, group_best;
  int softmax, renorm;
  float scale;
};

// ---- order keys -------------------------------------------------------------------------
// Larger is better, all keys of a token differ, -inf means "not there".  A NaN is better than
// every number, as torch.sort ranks it.
__device__ __forceinline__ double order_key(float v, int index) {
  constexpr uint32_t kLast = (1u << 29) - 1;
  if (v == -INFINITY) return -INFINITY;
  const double d = (double)(v + 0.f);              // (-0 and 0 are equal)
  uint64_t bits = __builtin_bit_cast(uint64_t, d);
  if (v != v) bits = 0x7fe0000000000000ull;
  else if (v == INFINITY) bits = 0x7fd0000000000000ull;
  // a larger mantissa is a larger positive number and a smaller negative one
  bits |= (bits >> 63) ? (uint32_t)index : kLast - (uint32_t)index;
  return __builtin_bit_cast(double, bits);
}
__device__ __forceinline__ int key_index(double key) {
  constexpr uint32_t kLast = (1u << 29) - 1;
  const uint64_t bits = __builtin_bit_cast(uint64_t, key);
  const uint32_t low = (uint32_t)bits & kLast;
  return (int)((bits >> 63) ? low : kLast - low);
}

// ---- reductions over the 16 lanes of a DPP row (and both rows of 32 lanes) --------------
template <int CTRL> __device__ __forceinline__ float rotate(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL> __device__ __forceinline__ double rotate(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
struct MaxOp {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const {
    return a > b ? a : b;
  }
  __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
};
struct SumOp {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
// op of a lane's value and the one 32 (FAR) or 16 lanes away
template <bool FAR> __device__ __forceinline__ void swap_rows(uint32_t a, uint32_t (&r)[2]) {
  const auto p = FAR ? __builtin_amdgcn_permlane32_swap(a, a, false, false)
                     : __builtin_amdgcn_permlane16_swap(a, a, false, false);
  r[0] = p[0];
  r[1] = p[1];
}
template <bool FAR, typename Op> __device__ __forceinline__ float op_swapped(float v, Op op) {
  uint32_t r[2];
  swap_rows<FAR>(__float_as_uint(v), r);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <bool FAR, typename Op> __device__ __forceinline__ double op_swapped(double v, Op op) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  uint32_t lo[2], hi[2];
  swap_rows<FAR>((uint32_t)b, lo);
  swap_rows<FAR>((uint32_t)(b >> 32), hi);
  return op(__builtin_bit_cast(double, ((uint64_t)hi[0] << 32) | lo[0]),
            __builtin_bit_cast(double, ((uint64_t)hi[1] << 32) | lo[1]));
}
// f(all lanes of the token), in every lane; the same bits in each (rotations by 8, 4, 2, 1 pair
// the same operands everywhere up to their order)
template <int LANES, typename V, typename Op>
__device__ __forceinline__ V over_lanes(V v, Op op) {
  v = op(v, rotate<0x128>(v));
  v = op(v, rotate<0x124>(v));
  v = op(v, rotate<0x122>(v));
  v = op(v, rotate<0x121>(v));
  if (LANES >= 32) v = op_swapped<false>(v, op);
  if (LANES == 64) v = op_swapped<true>(v, op);
  return v;
}

// The scores of a token, C registers per lane (expert u * LANES + g), as elementary torch
// operations give them: sigmoid as 1 / (1 + exp(-l)); softmax as exp(l - max) over their sum,
// which is taken in 64 bits so that it does not depend on the order of the additions.  Equal
// scores (and with them the choice) then are equal however they were computed.
template <int LANES, int C>
__device__ __forceinline__ void scores(const float (&l)[C], int n_expert, int g, bool softmax,
                                       float (&s)[C]) {
  if (!softmax) {
#pragma unroll
    for (int u = 0; u < C; ++u) s[u] = 1.f / (1.f + expf(-l[u]));
    return;
  }
  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < C; ++u) {
    m = fmaxf(m, l[u]);
    nan |= l[u] != l[u];
  }
  m = over_lanes<LANES>(m, MaxOp());
  double sum = nan ? NAN : 0.;
#pragma unroll
  for (int u = 0; u < C; ++u) {
    // (a row without an unmasked logit has m = -inf: no score at all)
    s[u] = u * LANES + g < n_expert && l[u] != -INFINITY ? expf(l[u] - m) : 0.f;
    sum += (double)s[u];
  }
  const float total = (float)over_lanes<LANES>(sum, SumOp());
#pragma unroll
  for (int u = 0; u < C; ++u) s[u] = total == 0.f ? 0.f : s[u] / total;
}

template <typename T, int LANES, int C>
__device__ __forceinline__ void load_logits(const T* logits, int64_t t, bool live, int n_expert,
                                            int g, float (&l)[C]) {
  const T* row = logits + t * n_expert;
#pragma unroll
  for (int u = 0; u < C; ++u) {
    const int e = u * LANES + g;
    l[u] = live && e < n_expert ? Elem<T>::to_acc(row[e]) : -INFINITY;
  }
}

// LDS per token: scores [n_expert], with groups also v [n_expert], the groups' keys and whether
// they stay
template <typename T, int LANES, int C>
__global__ __launch_bounds__(kScoreThreads) void score_topk_fwd_kernel(
    const T* __restrict__ logits, const float* __restrict__ bias, ScoreArgs a,
    int64_t* __restrict__ idx, T* __restrict__ weight) {
  extern __shared__ double score_lds[];
  constexpr int kTokens = kScoreThreads / LANES;
  const int g = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  const int64_t t = (int64_t)blockIdx.x * kTokens + slot;
  const bool live = t < a.n_tokens;
  const bool grouped = a.n_group > 1 && a.top_group < a.n_group;
  double* group_keys = score_lds + slot * a.n_group;
  float* s_row = (float*)(score_lds + (grouped ? kTokens * a.n_group : 0)) + slot * a.n_expert;
  float* v_row = s_row + kTokens * a.n_expert;
  uint8_t* stays = (uint8_t*)(score_lds + kTokens * (a.n_group + a.n_expert)) + slot * a.n_group;

  float l[C], s[C], v[C];
  load_logits<T, LANES, C>(logits, t, live, a.n_expert, g, l);
  scores<LANES, C>(l, a.n_expert, g, a.softmax, s);
#pragma unroll
  for (int u = 0; u < C; ++u) {
    const int e = u * LANES + g;
    v[u] = -INFINITY;
    if (e < a.n_expert) {
      if (l[u] != -INFINITY) v[u] = bias ? s[u] + bias[e] : s[u];
      s_row[e] = s[u];
      if (grouped) v_row[e] = v[u];
    }
  }
  __syncthreads();
  if (grouped) {
    const int size = a.n_expert / a.n_group;
    // `parts` lanes share a group (one if there are more groups than half the lanes)
    int parts = 1;
    while (2 * parts * a.n_group <= LANES) parts *= 2;
    for (int q = g / parts; q < a.n_group; q += LANES / parts) {
      float best = -INFINITY, second = -INFINITY;
      bool nan = false;
      auto take = [&](float x) {
        nan |= x != x;
        second = fmaxf(second, fminf(x, best));        // (a NaN is no part of either)
        best = fmaxf(best, x);
      };
#pragma unroll 4
      for (int i = g % parts; i < size; i += parts) take(v_row[q * size + i]);
      for (int d = 1; d < parts; d *= 2) {
        const float b = __shfl_xor(best, d, kWave), s2 = __shfl_xor(second, d, kWave);
        nan |= (bool)__shfl_xor((int)nan, d, kWave);
        take(b);
        take(s2);
      }
      float value = best;
      if (a.group_best == 2 && second != -INFINITY) value += second;
      if (g % parts == 0) group_keys[q] = order_key(nan ? NAN : value, q);
    }
    __syncthreads();
    for (int q = g; q < a.n_group; q += LANES) {
      const double mine = group_keys[q];
      int better = 0;
#pragma unroll 4
      for (int o = 0; o < a.n_group; ++o) better += group_keys[o] > mine;
      stays[q] = better < a.top_group;
    }
    __syncthreads();
    const float per_size = 1.f / (float)size;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int e = u * LANES + g;
      if (!stays[min((int)(((float)e + 0.5f) * per_size), a.n_group - 1)]) v[u] = -INFINITY;
    }
  }

  double key[C];
#pragma unroll
  for (int u = 0; u < C; ++u) key[u] = order_key(v[u], u * LANES + g);
  double mine = -INFINITY;                 // the key of this lane's slot
  double last = INFINITY;
  for (int j = 0; j < a.top_k; ++j) {
    double best = -INFINITY;
#pragma unroll
    for (int u = 0; u < C; ++u) best = fmax(best, key[u] < last ? key[u] : -INFINITY);
    best = over_lanes<LANES>(best, MaxOp());
    if (g == j) mine = best;
    last = best;
  }
  const bool found = mine != -INFINITY && g < a.top_k;
  const int e = found ? key_index(mine) : 0;
  float w = found ? s_row[e] : 0.f;
  if (a.renorm) {
    const float total = over_lanes<LANES>(w, SumOp());
    w = w / (total + kScoreEps);
  }
  if (live && g < a.top_k) {
    idx[t * a.top_k + g] = found ? e : -1;
    weight[t * a.top_k + g] = Elem<T>::from_acc(found ? w * a.scale : 0.f);
  }
}

// Lane j of a token takes its slot j: with S = sum of the chosen s + 1e-20,
//   ds_j = scale / S (dw_j - sum_i dw_i s_i / S)   or   scale dw_j
//   sigmoid: dl_j = ds_j s_j (1 - s_j), zero elsewhere
//   softmax: dl_e = s_e (ds_e - sum_i ds_i s_i) for every expert
// The row of ds (sigmoid: of dl) meets in LDS; a chosen expert occurs once in a token's slots.
template <typename T, int LANES, int C>
__global__ __launch_bounds__(kScoreThreads) void score_topk_bwd_kernel(
    const T* __restrict__ dweight, const T* __restrict__ logits, const int64_t* __restrict__ idx,
    ScoreArgs a, T* __restrict__ dlogits) {
  extern __shared__ double score_lds[];
  constexpr int kTokens = kScoreThreads / LANES;
  const int g = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  const int64_t t = (int64_t)blockIdx.x * kTokens + slot;
  const bool live = t < a.n_tokens;
  float* row = (float*)score_lds + slot * a.n_expert;

  float dw = 0.f, sj = 0.f;
  int e_mine = -1;
  if (live && g < a.top_k) {
    const int64_t e = idx[t * a.top_k + g];
    if (e >= 0 && e < a.n_expert) {
      e_mine = (int)e;
      dw = Elem<T>::to_acc(dweight[t * a.top_k + g]);
    }
  }
  float l[C], s[C];
  if (a.softmax) {
    load_logits<T, LANES, C>(logits, t, live, a.n_expert, g, l);
    scores<LANES, C>(l, a.n_expert, g, true, s);
#pragma unroll
    for (int u = 0; u < C; ++u)
      if (u * LANES + g < a.n_expert) row[u * LANES + g] = s[u];
    __syncthreads();
    if (e_mine >= 0) sj = row[e_mine];
    __syncthreads();
  } else if (e_mine >= 0) {
    sj = 1.f / (1.f + expf(-Elem<T>::to_acc(logits[t * a.n_expert + e_mine])));
  }
  float ds = a.scale * dw;
  if (a.renorm) {
    const float total = over_lanes<LANES>(sj, SumOp()) + kScoreEps;
    const float dot = over_lanes<LANES>(dw * sj, SumOp());
    ds = (a.scale / total) * (dw - dot / total);
  }
  if (e_mine < 0) ds = 0.f;
  float dot = 0.f;
  if (a.softmax) dot = over_lanes<LANES>(ds * sj, SumOp());
  else ds = ds * sj * (1.f - sj);
#pragma unroll
  for (int u = 0; u < C; ++u)
    if (u * LANES + g < a.n_expert) row[u * LANES + g] = 0.f;
  __syncthreads();
  if (e_mine >= 0) row[e_mine] = ds;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < C; ++u) {
    const int e = u * LANES + g;
    if (!live || e >= a.n_expert) continue;
    const float x = row[e];
    dlogits[t * a.n_expert + e] = Elem<T>::from_acc(a.softmax ? s[u] * (x - dot) : x);
  }
}

static int check_args(const ScoreArgs& a, int dtype) {
  FMOE_REQUIRE(a.n_tokens >= 0 && a.n_expert >= 1, FMOE_ERR_INVALID, "score_topk: bad sizes");
  FMOE_REQUIRE(a.top_k >= 1 && a.top_k <= a.n_expert, FMOE_ERR_INVALID,
               "score_topk: top_k %d of %d experts", a.top_k, a.n_expert);
  FMOE_REQUIRE(a.n_group >= 1 && a.n_expert % a.n_group == 0, FMOE_ERR_INVALID,
               "score_topk: %d groups do not divide %d experts", a.n_group, a.n_expert);
  FMOE_REQUIRE(a.top_group >= 1 && a.top_group <= a.n_group, FMOE_ERR_INVALID,
               "score_topk: top_group %d of %d groups", a.top_group, a.n_group);
  FMOE_REQUIRE(a.top_k <= (int64_t)a.top_group * (a.n_expert / a.n_group), FMOE_ERR_INVALID,
               "score_topk: %d groups hold fewer than top_k %d experts", a.top_group, a.top_k);
  FMOE_REQUIRE(a.group_best == 1 || a.group_best == 2, FMOE_ERR_INVALID,
               "score_topk: a group's value is its best 1 or 2 experts, not %d", a.group_best);
  FMOE_REQUIRE(a.n_expert <= kScoreMaxExperts, FMOE_ERR_UNSUPPORTED,
               "score_topk: %d experts, at most %d", a.n_expert, kScoreMaxExperts);
  FMOE_REQUIRE(a.top_k <= FMOE_MAX_GATE_TOP_K, FMOE_ERR_UNSUPPORTED,
               "score_topk: top_k %d above FMOE_MAX_GATE_TOP_K", a.top_k);
  FMOE_REQUIRE(a.n_group <= kScoreMaxGroups, FMOE_ERR_UNSUPPORTED,
               "score_topk: %d groups, at most %d", a.n_group, kScoreMaxGroups);
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "score_topk: unsupported dtype %d", dtype);
  return FMOE_OK;
}

// LANES lanes hold a token's n_expert <= LANES * C values: f<T, LANES, C>().  With few tokens
// what counts is how long one takes, so a wave has one; with many, how many instructions all of
// them take, and the steps over the lanes are shared by four (two above 256 experts).  Measured
// (us, a launch alone takes 2.1):
//   tokens  experts, of groups     16 or 32 lanes   64 lanes
//       64  256, 4 of 8                  10.8           5.8
//       64  128                           5.0           3.5
//     2048  128                           5.3           4.4
//     2048   64                           3.7           3.6
//     4096  256, 4 of 8                  11.0           9.1
//     4096  128                           5.4           6.2
//     8192  256, 4 of 8                  13.1          14.0
//    16384  128, 3 of 8                  10.9          20.7
#define FMOE_SCORE_SHAPES(T, CALL)                                       \
  do {                                                                   \
    const bool few = a.n_tokens <= (a.n_expert > 128 ? 4096 : 2048);     \
    if (a.n_expert <= 16) CALL(T, 16, 1);                                \
    else if (a.n_expert <= 32) CALL(T, 16, 2);                           \
    else if (a.n_expert <= 64 && few) CALL(T, 64, 1);                    \
    else if (a.n_expert <= 64) CALL(T, 16, 4);                           \
    else if (a.n_expert <= 128 && few) CALL(T, 64, 2);                   \
    else if (a.n_expert <= 128) CALL(T, 16, 8);                          \
    else if (a.n_expert <= 256 && few) CALL(T, 64, 4);                   \
    else if (a.n_expert <= 256) CALL(T, 16, 16);                         \
    else if (few) CALL(T, 64, 8);                                        \
    else CALL(T, 32, 16);                                                \
  } while (0)

template <typename T>
static int launch_fwd(const void* logits, const float* bias, const ScoreArgs& a, int64_t* idx,
                      void* weight, hipStream_t s) {
  const bool grouped = a.n_group > 1 && a.top_group < a.n_group;
#define FMOE_CALL(T, LANES, C)                                                                  \
  hipLaunchKernelGGL((score_topk_fwd_kernel<T, LANES, C>),                                      \
                     dim3(ceil_div(a.n_tokens, kScoreThreads / LANES)), dim3(kScoreThreads),    \
                     (kScoreThreads / LANES) *                                                  \
                         ((grouped ? 2 : 1) * a.n_expert * 4 + (grouped ? a.n_group * 9 : 0)),  \
                     s, (const T*)logits, bias, a, idx, (T*)weight)
  FMOE_SCORE_SHAPES(T, FMOE_CALL);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("score_topk_fwd");
  return FMOE_OK;
}

template <typename T>
static int launch_bwd(const void* dweight, const void* logits, const int64_t* idx,
                      const ScoreArgs& a, void* dlogits, hipStream_t s) {
#define FMOE_CALL(T, LANES, C)                                                                  \
  hipLaunchKernelGGL((score_topk_bwd_kernel<T, LANES, C>),                                      \
                     dim3(ceil_div(a.n_tokens, kScoreThreads / LANES)), dim3(kScoreThreads),    \
                     (kScoreThreads / LANES) * a.n_expert * 4, s, (const T*)dweight,            \
                     (const T*)logits, idx, a, (T*)dlogits)
  FMOE_SCORE_SHAPES(T, FMOE_CALL);
#undef FMOE_CALL
  FMOE_LAUNCH_CHECK("score_topk_bwd");
  return FMOE_OK;
}

}  // namespace fmoe

extern "C" int fmoe_score_topk_fwd(const void* logits, const float* bias, int64_t n_tokens,
                                   int32_t n_expert, int32_t top_k, int32_t n_group,
                                   int32_t top_group, int32_t group_best, int score,
                                   int renormalize, float scale, int64_t* idx, void* weight,
                                   int dtype, void* stream) {
  using namespace fmoe;
  FMOE_REQUIRE(score == FMOE_SCORE_SIGMOID || score == FMOE_SCORE_SOFTMAX, FMOE_ERR_INVALID,
               "score_topk: unknown score %d", score);
  const ScoreArgs a{n_tokens, n_expert, top_k, n_group, top_group, group_best,
                    score == FMOE_SCORE_SOFTMAX, renormalize != 0, scale};
  if (const int rc = check_args(a, dtype)) return rc;
  if (n_tokens == 0) return FMOE_OK;
  FMOE_REQUIRE(logits && idx && weight, FMOE_ERR_INVALID, "score_topk: null pointer");
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FMOE_F32: return launch_fwd<float>(logits, bias, a, idx, weight, s);
    case FMOE_F16: return launch_fwd<__half>(logits, bias, a, idx, weight, s);
    default: return launch_fwd<__hip_bfloat16>(logits, bias, a, idx, weight, s);
  }
}

extern "C" int fmoe_score_topk_bwd(const void* dweight, const void* logits, const int64_t* idx,
                                   int64_t n_tokens, int32_t n_expert, int32_t top_k, int score,
                                   int renormalize, float scale, void* dlogits, int dtype,
                                   void* stream) {
  using namespace fmoe;
  FMOE_REQUIRE(score == FMOE_SCORE_SIGMOID || score == FMOE_SCORE_SOFTMAX, FMOE_ERR_INVALID,
               "score_topk: unknown score %d", score);
  const ScoreArgs a{n_tokens, n_expert, top_k, 1, 1, 1, score == FMOE_SCORE_SOFTMAX,
                    renormalize != 0, scale};
  if (const int rc = check_args(a, dtype)) return rc;
  if (n_tokens == 0) return FMOE_OK;
  FMOE_REQUIRE(dweight && logits && idx && dlogits, FMOE_ERR_INVALID, "score_topk: null pointer");
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FMOE_F32: return launch_bwd<float>(dweight, logits, idx, a, dlogits, s);
    case FMOE_F16: return launch_bwd<__half>(dweight, logits, idx, a, dlogits, s);
    default: return launch_bwd<__hip_bfloat16>(dweight, logits, idx, a, dlogits, s);
  }
}
