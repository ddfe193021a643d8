// Rows in microscaled 4-bit floating point (MXFP4 of the OCP Microscaling Formats
// specification): blocks of 32 values along the features, every value an E2M1 code of 4 bits
// (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign), every block a power of two held as an E8M0 byte
// (exponent + 127; 255 is NaN).
//
// In memory a row of K features is 64 ceil(K / 128) bytes of codes, the even feature of a pair
// in the low half of its byte, and 16 ceil(K / 512) scale bytes: whole steps of the matrix
// instruction (128 features) and whole 16-byte packs, so that no kernel has an edge along K.
// Codes behind the last feature are zero, scale bytes of blocks up to the next multiple of
// 128 features are not 255; scale bytes further on are never used.
#pragma once
#include "common.h"

namespace fmoe {

constexpr int kMxBlock = 32;         // features that share a scale
constexpr int kMxStep = 128;         // features of one matrix instruction: 64 bytes of codes
constexpr int kMxGroup = 512;        // features whose scales fill a 16-byte pack
constexpr int kMxNan = 255;

__host__ __device__ inline int64_t mx_code_bytes(int64_t k) { return (k + kMxStep - 1) / kMxStep * 64; }
__host__ __device__ inline int64_t mx_scale_bytes(int64_t k) { return (k + kMxGroup - 1) / kMxGroup * 16; }

// 2^(byte - 127); byte 0 is the subnormal 2^-127, which the conversions below take as well.
__device__ __forceinline__ float mx_power(int byte) {
  return __uint_as_float(byte > 0 ? (uint32_t)byte << 23 : 0x00400000u);
}

// Scale byte of a block from the bits of its largest magnitude as f32: the exponent two below
// that magnitude's own (6 = 1.5 * 2^2 is the largest code; what lies between 6 and 8 times the
// scale saturates, as the specification has it), not below 2^-127.
__device__ __forceinline__ int mx_scale_byte(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return kMxNan;
  return max((int)(max_bits >> 23) - 2, 0);
}

// The 8 codes of v / 2^(byte - 127), v[0] in the lowest bits: nearest, ties to the even code,
// saturated at 6 (what the conversion instruction does; a NaN block's codes are zero).
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], int byte) {
  if (byte == kMxNan) return 0;
  const float p = mx_power(byte);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], p, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], p, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], p, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], p, 3);
  return r;
}

// The 8 values of a word of codes.
__device__ __forceinline__ void mx_values(uint32_t codes, int byte, float (&v)[8]) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const float p = mx_power(byte);
  f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, p, 0);
  f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, p, 1);
  f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, p, 2);
  f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, p, 3);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
  v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
  if (byte == kMxNan) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = NAN;
  }
}

__device__ __forceinline__ uint32_t magnitude_bits(float v) {
  return __float_as_uint(v) & 0x7fffffffu;
}

}  // namespace fmoe
