// Rows of values on their way into and out of quantised form: loads and stores of 8 values a lane,
// segment bounds from counts, rows that a kernel clears in passing.
#pragma once
#include <type_traits>

#include "common.h"

namespace fmoe {

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

// 8 values as they lie in memory, in whole registers.
template <typename T> struct Eight {
  uint32_t w[2 * sizeof(T)];

  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (std::is_same<T, float>::value) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __hip_bfloat16>::value) {
      return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    } else {
      return __half2float(__builtin_bit_cast(__half, (uint16_t)(w[i >> 1] >> (16 * (i & 1)))));
    }
  }
  __device__ __forceinline__ void widen(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (*this)[i];
  }

  // The values are runs of 16 bytes, N each, at k, k + gap (consecutive by default: values k .. k + 7).
  static constexpr int N = 16 / (int)sizeof(T);
  typedef uint32_t Pack __attribute__((ext_vector_type(4), aligned(2)));     // rows of any alignment

  // From p on, all of them there.  ONCE: nobody reads them again (the loads do not displace what the
  // caches hold: 131072 rows of 2048 summed up by eights, 119 us without, 102 with).
  template <bool ONCE = false> __device__ __forceinline__ void load(const T* p, int gap = N) {
#pragma unroll
    for (int q = 0; q < 8 / N; ++q) {
      const Pack* const from = reinterpret_cast<const Pack*>(p + q * gap);
      const Pack v = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * q + j] = v[j];
    }
  }
  // From k on, zeros from the row's end d on.
  template <bool ONCE = false>
  __device__ __forceinline__ void load(const T* row, int k, int d, int gap = N) {
    if (k + 7 / N * gap + N <= d) {
      load<ONCE>(row + k, gap);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * (int)sizeof(T); ++i) w[i] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = k + i / N * gap + i % N;
        if (at >= d) continue;
        if constexpr (sizeof(T) == 4) w[i] = __builtin_bit_cast(uint32_t, row[at]);
        else w[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, row[at]) << (16 * (i & 1));
      }
    }
  }
  // 8 values, rounded, likewise, nothing behind the row's end d.  ONCE: not to be read before much
  // else was written.
  template <bool ONCE = false>
  static __device__ __forceinline__ void store(T* row, int k, int d, const float (&v)[8], int gap = N) {
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = Elem<T>::from_acc(v[i]);
#pragma unroll
    for (int q = 0; q < 8 / N; ++q) {
      const int at = k + q * gap;
      if (at + N <= d) {
        Pack p;
        __builtin_memcpy(&p, o + q * N, 16);
        if constexpr (ONCE) __builtin_nontemporal_store(p, reinterpret_cast<Pack*>(row + at));
        else *reinterpret_cast<Pack*>(row + at) = p;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at + i < d) row[at + i] = o[q * N + i];
      }
    }
  }

  // The bits, as f32, of the largest magnitude (NaN > infinity > numbers) of these and of `bits`,
  // what earlier calls returned (0 at first); f32_bits() of the last one is the answer.
  __device__ __forceinline__ uint32_t widest(uint32_t bits) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) bits = max(bits, w[i] & 0x7fffffffu);
    } else {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = __builtin_bit_cast(u16x2, bits);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
      bits = __builtin_bit_cast(uint32_t, m);
    }
    return bits;
  }
  static __device__ __forceinline__ uint32_t f32_bits(uint32_t bits) {
    if constexpr (sizeof(T) == 4) return bits;
    const uint32_t m = max(bits & 0xffffu, bits >> 16);
    if constexpr (std::is_same<T, __hip_bfloat16>::value) return m << 16;
    else return __float_as_uint(__half2float(__builtin_bit_cast(__half, (uint16_t)m)));
  }
};

// Sum and maximum over the wave, the same in every lane (the moves of wave_inclusive_sum()).
#define FMOE_ROW_MOVES(STEP) \
  STEP(0x111, 0xf) /* row_shr:1 */ STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf) \
  STEP(0x142, 0xa) /* row_bcast:15 */ STEP(0x143, 0xc) /* row_bcast:31 */
__device__ __forceinline__ float wave_sum(float x) {
#define FMOE_ADD(CTRL, ROWS) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xf, false));
  FMOE_ROW_MOVES(FMOE_ADD)
#undef FMOE_ADD
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), kWave - 1));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t m) {
#define FMOE_MAX(CTRL, ROWS) \
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, ROWS, 0xf, false));
  FMOE_ROW_MOVES(FMOE_MAX)
#undef FMOE_MAX
  return (uint32_t)__builtin_amdgcn_readlane((int)m, kWave - 1);
}
#undef FMOE_ROW_MOVES

// Row counts of experts as segment bounds, for the call's first workgroup to leave behind.
struct SegmentsOut {
  const int64_t* count = nullptr;
  int n_expert = 0;
  int32_t* seg_off = nullptr;
};

// seg_off = exclusive prefix of the counts, by one wave.  Counts on the device nobody has looked
// at: negative ones count as zero, and what lies beyond the rows there are is cut off.
__device__ __forceinline__ void write_segments(const SegmentsOut& sg, int64_t n_rows, int lane) {
  if (sg.count == nullptr) {              // all rows are the only expert's
    if (lane < 2) sg.seg_off[lane] = lane == 0 ? 0 : (int32_t)n_rows;
    return;
  }
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

// The rows of a gradient that no expert owns, for a kernel in front of the gradient's product to
// clear in passing: rows *end .. n_rows - 1 of k values at p.
template <typename T> struct ClearedTail {
  const int32_t* end = nullptr;
  T* p = nullptr;
  int64_t n_rows = 0;

  __device__ __forceinline__ void clear(int k) const {
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)max(*end, 0) * k + (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
         i < n_rows * k; i += stride)
      p[i] = Elem<T>::from_acc(0.f);
  }
};

// The longest run (of at most 16 bytes) that every row holds a whole number of, at its alignment.
template <typename T> static int run_length(const void* p, int k) {
  int n = 16 / (int)sizeof(T);
  while (n > 1 && (k % n || (uintptr_t)p % (n * sizeof(T)))) n /= 2;
  return n;
}

}  // namespace fmoe
