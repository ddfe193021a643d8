// Rows in 8-bit integers with one scale each: codes q in -127 .. 127 and a float s, the values
// being q s.  A row of K features is 128 ceil(K / 128) bytes of codes, those behind the last
// feature zero: whole stages of the product's copies, so that no kernel has an edge along K.
//
// With a = max |x| over a row, s = a / 127 in f32 and q = the integer nearest to 127 x / a, ties to
// even, exactly.  A row of zeros has s = 0; one with an infinity or a NaN has s = NaN and q = 0, so
// that its values, and its products with anything, are NaN.
#pragma once
#include "common.h"

namespace fmoe {

constexpr int kI8Step = 128;

__host__ __device__ inline int64_t i8_row_bytes(int64_t k) {
  return (k + kI8Step - 1) / kI8Step * kI8Step;
}

}  // namespace fmoe
