// Rows of values on their way into and out of quantised form: loads and stores of 8 values a lane,
// segment bounds from counts, rows that a kernel clears in passing.
#pragma once
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
