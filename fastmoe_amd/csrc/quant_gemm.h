// What the grouped products of quantised rows share (MXFP4: mx_gemm.hip, 8-bit integers:
// i8_gemm.hip): how a result leaves, and the tiles of many rows.
//
// Both formats feed the matrix cores 16 bytes a lane, 16 rows of 64 bytes an operand, in the same
// time, so that everything that moves bytes is the same for either; the formats differ in the
// matrix instruction, in the scales (a byte per block, copied beside the codes, against a float per
// row, applied to the sums) and in how many features 64 bytes are.
#pragma once
#include <type_traits>

#include "dma_desc.h"
#include "gemm_tiles.h"
#include "i8.h"
#include "mx.h"

namespace fmoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct QuantGemmArgs {
  const uint8_t *xc, *xs, *wc, *ws;      // (the scales of 8-bit rows are floats)
  const void* bias;            // [E, out] or null
  const int32_t* seg_off;
  void* y;                     // [n_rows, out], or null with yc
  uint8_t *yc, *ys;            // rows of `out` features
  int64_t n_rows;
  int in_feat, out_feat, n_expert, dtype;
};

// Feature, within its group of 32, of row m of fragment f.
__device__ __forceinline__ int mx_feature(int f, int m) { return 8 * (m >> 2) + 4 * f + (m & 3); }

__device__ __forceinline__ i32x4 mx_descriptor(const void* p, int64_t bytes) {
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(uint64_t)p);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint64_t)p >> 32) & 0xffff);   // stride 0
  r[2] = __builtin_amdgcn_readfirstlane(dma_num_records(bytes));
  r[3] = 0x00020000;
  return r;
}

__device__ __forceinline__ float mx_gelu(float x);     // (only the 4-bit product has it behind it)

// How a product leaves: y where rows are whole 16-byte packs, any other y, or MXFP4 again behind
// one of the activations.
enum MxMode { kMxPacked, kMxAny, kMxQuant, kMxQuantGelu, kMxQuantRelu };
constexpr bool mx_quantises(int mode) { return mode >= kMxQuant; }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_resource(const void* p, int64_t bytes) {
  const uint64_t u = (uint64_t)p;
  void* q = (void*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32) |
                    (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u));
  return __builtin_amdgcn_make_buffer_rsrc(
      q, 0, __builtin_amdgcn_readfirstlane(dma_num_records(bytes)), 0x00020000);
}

// The bias of expert e, as its rows are read: nothing behind the last feature, nothing at all
// without a bias.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_bias_rows(const QuantGemmArgs& a, int e) {
  const int64_t bytes = (int64_t)a.out_feat * (a.dtype == FMOE_F32 ? 4 : 2);
  return mx_resource((const char*)a.bias + e * bytes, a.bias ? bytes : 0);
}
// 8 values of the bias's 16-bit type.
__device__ __forceinline__ void mx_widen(const QuantGemmArgs& a, i32x4 u, float (&b)[8]) {
  if (a.dtype == FMOE_BF16) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b[i] = __uint_as_float(i & 1 ? (uint32_t)u[i >> 1] & 0xffff0000u : (uint32_t)u[i >> 1] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b[i] = __half2float(__builtin_bit_cast(__half, (uint16_t)((uint32_t)u[i >> 1] >> (16 * (i & 1)))));
  }
}
// The bias of 8 consecutive features from n0 on (zeros where there is none).
__device__ __forceinline__ void mx_load_bias(const QuantGemmArgs& a, __amdgpu_buffer_rsrc_t rows,
                                             int n0, float (&b)[8]) {
  // (one test for all, or every load is waited for by itself)
  if (a.bias == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.f;
  } else if (a.dtype == FMOE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, (n0 + i) * 4, 0, 0));
  } else {
    uint16_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      u[i] = __builtin_amdgcn_raw_buffer_load_b16(rows, (n0 + i) * 2, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b[i] = a.dtype == FMOE_BF16 ? __uint_as_float((uint32_t)u[i] << 16)
                                  : __half2float(__builtin_bit_cast(__half, u[i]));
  }
}

// What a tile writes: descriptors that end with its last valid row, so that rows past the end
// need no branch.
template <typename T, int MODE> struct MxOutput {
  static constexpr bool QUANT = mx_quantises(MODE);
  __amdgpu_buffer_rsrc_t y, yc, ys;
  T* y_row;                 // row 0 of the tile
  int n, rows;

  // rows x0 .. x0 + rows - 1 of the output
  __device__ __forceinline__ MxOutput(const QuantGemmArgs& a, int64_t x0, int rows_) {
    n = a.out_feat;
    rows = rows_;
    if (QUANT) {
      const int64_t cr = mx_code_bytes(n), sr = mx_scale_bytes(n);
      yc = mx_resource(a.yc + x0 * cr, rows * cr);
      ys = mx_resource(a.ys + x0 * sr, rows * sr);
    } else {
      y_row = (T*)a.y + x0 * n;
      y = mx_resource(y_row, (int64_t)rows * n * sizeof(T));
    }
  }

  static __device__ __forceinline__ void activate(float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (MODE == kMxQuantGelu) v[i] = mx_gelu(v[i]);
      if constexpr (MODE == kMxQuantRelu) v[i] = __builtin_elementwise_maximum(v[i], 0.f);   // (a NaN stays)
    }
  }

  // The word of codes and the scale byte of features n0 .. n0 + 7 (`whole`: none of the wave's is
  // behind the last).  All lanes of a wave come here together; lanes l, l ^ 16, l ^ 32 and l ^ 48
  // hold one block of 32 features.
  __device__ __forceinline__ uint32_t quantised(int n0, bool whole, float (&v)[8], int& byte) const {
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = n0 + i < n ? v[i] : 0.f;
    }
    float top = 0.f;                         // (this maximum keeps a NaN)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __builtin_elementwise_maximum(top, __builtin_fabsf(v[i]));
    uint32_t m = magnitude_bits(top);
    // (rows of 16 lanes, then halves of the wave, swap places: either result holds one of the two)
    const auto r16 = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(r16[0], r16[1]);
    const auto r32 = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    m = max(r32[0], r32[1]);
    byte = mx_scale_byte(m);
    return mx_codes(v, byte);
  }

  // Activation and output of features n0 .. n0 + 7 of the tile's row `row`, from the registers.
  __device__ __forceinline__ void store(int row, int n0, float (&v)[8]) const {
    activate(v);
    if constexpr (QUANT) {
      int byte;
      const uint32_t word = quantised(n0, false, v, byte);
      const int cr = (int)mx_code_bytes(n), sr = (int)mx_scale_bytes(n);
      const bool in = n0 < cr * 2;
      __builtin_amdgcn_raw_buffer_store_b32(word, yc, in ? row * cr + n0 / 2 : kDmaOutOfRange, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b8(
          (uint8_t)byte, ys, in && (n0 & 31) == 0 ? row * sr + n0 / kMxBlock : kDmaOutOfRange, 0, 0);
    } else {
      T o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = Elem<T>::from_acc(v[i]);
      const uint32_t at = ((uint32_t)row * n + n0) * (uint32_t)sizeof(T);
      if constexpr (MODE == kMxPacked) {
#pragma unroll
        for (int p = 0; p < (int)sizeof(T) / 2; ++p) {
          i32x4 w;
          __builtin_memcpy(&w, (const char*)o + p * 16, 16);
          __builtin_amdgcn_raw_buffer_store_b128(
              w, y, n0 + p * Pack16<T>::kN < n ? at + p * 16 : kDmaOutOfRange, 0, 0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t to = n0 + i < n ? at + i * (uint32_t)sizeof(T) : kDmaOutOfRange;
          if constexpr (sizeof(T) == 4)
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, o[i]), y, to, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, o[i]), y, to, 0, 0);
        }
      }
    }
  }

  // Stores of a wave for 16 rows of P groups of 32 features, `times` over, where their number is
  // known (and the counter takes it).
  template <int P, int ROW> static constexpr int stores(int times) {
    const int n = times * (QUANT ? 2 : P * 32 * (int)sizeof(T) / 64);
    return n < 63 ? n : 63;
  }

  // Activation and output of 16 rows from row `row0` of the tile on: lane (m, g) holds features
  // 8 g .. 8 g + 7 of each of P groups of 32, from feature `col` on, of row m.  They change places
  // in `stage` (16 rows of ROW bytes, the wave's own) so that a store covers whole pieces of rows.
  template <int P, int ROW>
  __device__ __forceinline__ void store_rows(char* stage, int lane, int row0, int col,
                                             float (&v)[P][8]) const {
    const int m = lane & 15, g = lane >> 4;
#pragma unroll
    for (int p = 0; p < P; ++p) activate(v[p]);
    if constexpr (QUANT) {
      static_assert(P == 2 || P == 4, "a wave's features are 64 or 128");
      const int cr = (int)mx_code_bytes(n), sr = (int)mx_scale_bytes(n);
      uint32_t bytes = 0;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        int byte;
        const uint32_t word = quantised(col + p * 32 + 8 * g, col + 32 * P <= n, v[p], byte);
        bytes |= (uint32_t)byte << (8 * p);
        *(uint32_t*)(stage + m * (P * 16) + ((p * 16 + g * 4) ^ ((m & 4) * 4))) = word;
      }
      // (columns end on 128 features, and the row's scales reach at least as far as its codes)
      const int r = lane / P, c = lane % P, n0 = col + c * 32;
      const bool in = r < 16 && n0 < cr * 2;
      const i32x4 w = *(const i32x4*)(stage + (r & 15) * (P * 16) + ((c * 16) ^ ((r & 4) * 4)));
      __builtin_amdgcn_raw_buffer_store_b128(w, yc, in ? (row0 + r) * cr + n0 / 2 : kDmaOutOfRange, 0, 0);
      const int to = g == 0 && col < cr * 2 ? (row0 + m) * sr + col / kMxBlock : (int)kDmaOutOfRange;
      if constexpr (P == 4) __builtin_amdgcn_raw_buffer_store_b32(bytes, ys, to, 0, 0);
      else __builtin_amdgcn_raw_buffer_store_b16((uint16_t)bytes, ys, to, 0, 0);
    } else {
      constexpr int kPass = ROW / (32 * (int)sizeof(T)) < P ? ROW / (32 * (int)sizeof(T)) : P;
      constexpr int kBytes = kPass * 32 * (int)sizeof(T);       // of a row, in a pass
      constexpr int kPacks = kBytes / 16, kN = 16 / (int)sizeof(T);
      static_assert(P % kPass == 0 && (kPacks == 8 || kPacks == 16), "whole passes");
#pragma unroll
      for (int q = 0; q < P; q += kPass) {
#pragma unroll
        for (int p = 0; p < kPass; ++p)
#pragma unroll
          for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
            T o[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) o[i] = Elem<T>::from_acc(v[q + p][h * kN + i]);
            i32x4 w;
            __builtin_memcpy(&w, o, 16);
            const int pack = (p * 4 + g) * ((int)sizeof(T) / 2) + h;
            *(i32x4*)(stage + m * kBytes + ((pack ^ m) & (kPacks - 1)) * 16) = w;
          }
        const int c = lane % kPacks, n0 = col + q * 32 + c * kN;
#pragma unroll
        for (int u = 0; u < kPacks / 4; ++u) {
          const int r = u * (64 / kPacks) + lane / kPacks, row = row0 + r;
          const i32x4 w = *(const i32x4*)(stage + r * kBytes + ((c ^ r) & (kPacks - 1)) * 16);
          if constexpr (MODE == kMxPacked) {
            __builtin_amdgcn_raw_buffer_store_b128(
                w, y, n0 < n ? ((uint32_t)row * n + n0) * (uint32_t)sizeof(T) : kDmaOutOfRange, 0, 2);
          } else if (row < rows) {
            T* to = y_row + (int64_t)row * n + n0;
            if (n0 + kN <= n) {
              __builtin_memcpy(to, &w, 16);
            } else {
              T o[kN];
              __builtin_memcpy(o, &w, 16);
#pragma unroll
              for (int i = 0; i < kN; ++i)
                if (n0 + i < n) to[i] = o[i];
            }
          }
        }
      }
    }
  }
};

// ------------------------------------------------------------------------- many rows
// Tiles of TN features x TM rows by 2 x 2 waves, operands through LDS.  A stage is 256 features
// of K of both operands, rows of 128 bytes, and there are two of them; scales come in groups of
// 512 features, 16 bytes a row, in two buffers of their own.  Everything is copied by
// buffer_load_dwordx4 ... lds (1 KiB an instruction, no staging registers): the 16-byte pack that
// lane l of a copy fetches is the one that belongs at byte 16 l of its KiB, pack p of LDS row r
// sitting in slot p ^ ((r >> 1) & 7), which serves the fragment reads (16 rows x 4 packs) without
// bank conflicts; LDS row 16 f + m holds the feature that fragment f wants in lane row m.
//
// A stage is two matrix steps of FW * TW instructions per wave.  While the first multiplies, the
// second's fragments are read, and a barrier behind those reads releases the stage's buffer: the
// copies of the stage after next follow, dealt out over the rest of both steps.  In the second
// step a wait and a barrier publish the next stage, whose first fragments are read in the shadow
// of the remaining instructions.  The next group's scales are read in between, when no fragments
// are.
//
// One workgroup of 256 x 256 fills a CU (all its registers, all its LDS; of the smaller tiles two
// do) and runs tile after tile in one
// pipeline: the last group of a tile copies the next tile's first two stages and scales and ends
// with its first fragments in registers, so that between two tiles there is nothing but the
// output.  The results leave through a corner of LDS that turns the lanes' 16 bytes of 16 rows
// into pieces of 256 bytes of a row (stored from the registers, 64 bytes of each of 16 rows at a
// time, they took 16 us a tile instead of 9).
//
// Measured: 32768 rows of 8 experts, 16384 -> 4096, 926 us, 4.75 PFLOP/s; 4096 -> 14336 917 us,
// 4.20.  A loop of these matrix instructions alone reaches 7.3 on random codes (9.7 on zeros: the
// card's power limit sets the clock).  Of the first shape's 1.68 M cycles at 1.9 GHz the matrix
// pipes are busy for 1.05; without copies it takes 1.45 M, without fragment reads as many as with
// them.  128 x 128 tiles on 15560 rows of 128 experts, 2048 -> 1408: 61 us, 257 MB at 4.2 TB/s.
typedef __attribute__((address_space(3))) char lds_char;

template <int I, int N, typename F> __device__ __forceinline__ void unroll(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unroll<I + 1, N>(f);
  }
}

// c += a * b in place, with byte BYTE of either scale word.  Written as assembly because the
// compiler, given the builtin, moves accumulators between registers in a loop that uses all of
// them; whoever reads c behind the last one waits out the matrix pipe (mx_mfma_done()).
template <int BYTE>
__device__ __forceinline__ void mx_mfma_at(i32x4 a, int sa, i32x4 b, int sb, f32x4& c) {
#define FMOE_MFMA(SEL)                                                                      \
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL " cbsz:4 blgp:4" \
               : "+a"(c) : "v"(a), "v"(b), "v"(sa), "v"(sb))
  if constexpr (BYTE == 0) FMOE_MFMA("op_sel_hi:[0,0,0]");
  if constexpr (BYTE == 1) FMOE_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  if constexpr (BYTE == 2) FMOE_MFMA("op_sel_hi:[1,1,0]");
  if constexpr (BYTE == 3) FMOE_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef FMOE_MFMA
}
// Likewise c += a * b in 8-bit integers: lane l holds 16 codes of row l % 16 in either operand, and
// which features these are is free as long as both agree.
__device__ __forceinline__ void i8_mfma_at(i32x4 a, i32x4 b, i32x4& c) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// An accumulator's value.  (Read like this, accumulators have no use in which they would have to
// be ordinary registers, so that they stay where the matrix instructions want them.)
__device__ __forceinline__ float mx_read(float c) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(c));
  return v;
}
__device__ __forceinline__ float mx_read(int c) {
  int v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(c));
  return (float)v;
}
// The 18 wait states between the last matrix instruction and a read of its result.
__device__ __forceinline__ void mx_mfma_done() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

template <bool INT8, int TN, int TM> struct QuantTile {
  static constexpr int kStageBytes = (TN + TM) * 128;
  static constexpr int kLoadsW = TN / 32, kLoadsX = TM / 32;       // copies of a wave per stage
  static constexpr int kLoads = kLoadsW + kLoadsX;
  static constexpr int kScaleLoads = INT8 ? 0 : ((TN + TM) / 64 + 3) / 4;   // and per group of scales
  static constexpr int kScaleBytes = kScaleLoads * 4096;
  static constexpr int kOutRow = TN <= 128 ? 128 : 256;            // bytes of a row on its way out
  static constexpr int kOutBytes = 4 * 16 * kOutRow;
  // (the floats of 8-bit rows, and the bias with them, in a place of their own: 2 KiB a wave)
  static constexpr int kFactorBytes = INT8 ? 4 * 2048 : 0;
  static constexpr int kLdsBytes = 2 * (kStageBytes + kScaleBytes) + kOutBytes + kFactorBytes;
  static constexpr int kGroups = kLdsBytes > 81920 ? 1 : 2;        // workgroups on a CU
  static_assert(TN % 128 == 0 && TM % 64 == 0 && TN <= 256 && TM <= 256, "even copies per wave");
};

// `v`, as a value that the compiler has to derive things from anew: what it could compute once
// for all tiles would be kept in scratch memory through the K loop, and reading it back waits for
// the copies under way.
__device__ __forceinline__ int mx_fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Where a tile lies.
struct MxPlace {
  int e, base, rows;      // expert, first feature, valid rows
  int64_t x0;             // first row
};

template <bool INT8, typename T, int TN, int TM, int MODE>
__device__ __forceinline__ void quant_tiles(const QuantGemmArgs& a) {
  using S = QuantTile<INT8, TN, TM>;
  constexpr int FW = TN / 32, TW = TM / 32;         // fragments of a wave
  constexpr int kMma = FW * TW;
  extern __shared__ __align__(16) char lds[];
  // (the first wave's corner, behind the bias; results on their way out may pass over it)
  int* const s_find = (int*)(lds + 2 * (S::kStageBytes + S::kScaleBytes) + 1024);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  RowTiles<TM, kOneHeight, 4> tiles;
  tiles.scan(a.seg_off, a.n_expert, s_find);
  const int n_pad = mx_quantises(MODE) ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const int n_cols = (n_pad + TN - 1) / TN;
  const int live = __builtin_amdgcn_readfirstlane(tiles.rows_f * n_cols);
  const int code_row = (int)(INT8 ? i8_row_bytes(a.in_feat) : mx_code_bytes(a.in_feat));
  const int scale_row = INT8 ? 4 : (int)mx_scale_bytes(a.in_feat);
  const int steps = __builtin_amdgcn_readfirstlane(INT8 ? code_row / 64
                                                        : (a.in_feat + kMxStep - 1) / kMxStep);
  const int stages = (steps + 1) / 2;

  // The offset a lane fetches from in each of its wave's copies, one stage (of the scales: one
  // group) back: a copy moves its own on.
  constexpr int kScaleLoads = S::kScaleLoads;
  uint32_t c_off[S::kLoads], s_off[INT8 ? 1 : kScaleLoads];
  i32x4 w_rsrc, x_rsrc, s_rsrc[INT8 ? 1 : kScaleLoads];
  auto pack_of = [](int lane, int p) { return (lane & 7) ^ ((4 * p + (lane >> 4)) & 7); };
  auto place = [&](int number) {
    int v, col;
    tile_order(number, tiles.rows_f, n_cols, v, col);
    const TileRows t = tiles.find(a.seg_off, v, false, s_find + 16);
    MxPlace at;
    at.e = t.e;
    at.base = col * TN;                             // (below out_feat: columns end on 128)
    at.x0 = (int64_t)t.row0 + t.m0;
    at.rows = min(TM, t.cnt - t.m0);
    return at;
  };
  auto aim = [&](const MxPlace& at) {
    const int lane = mx_fresh(threadIdx.x & 63), r8 = lane >> 3;
    const int64_t w0 = (int64_t)at.e * a.out_feat + at.base;
    const int w_rows = min(TN, a.out_feat - at.base);
    // every descriptor ends with its last valid row: rows past the end read as zeros
    w_rsrc = mx_descriptor(a.wc + w0 * code_row, (int64_t)w_rows * code_row);
    x_rsrc = mx_descriptor(a.xc + at.x0 * code_row, (int64_t)at.rows * code_row);
    // every wave has its share of either operand, so that nothing here depends on the wave but
    // numbers; rows of a weight fragment are features 8 (m / 4) + m % 4 of 32
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int kib = i < S::kLoadsW ? wave * S::kLoadsW + i : wave * S::kLoadsX + i - S::kLoadsW;
      const int row = i < S::kLoadsW ? wave * (TN / 4) + 32 * (i >> 2) + 16 * (i & 1) +
                                           4 * ((i >> 1) & 1) + 8 * (r8 >> 2) + (r8 & 3)
                                     : kib * 8 + r8;
      c_off[i] = (uint32_t)(row * code_row + pack_of(lane, kib & 1) * 16 - 128);
    }
    // the scales of 64 rows of one operand (past both: zeros)
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
      const int kib = wave * kScaleLoads + i;
      const bool w = kib < TN / 64;
      const i32x4 rw = mx_descriptor(a.ws + w0 * scale_row, (int64_t)w_rows * scale_row);
      const i32x4 rx = mx_descriptor(a.xs + at.x0 * scale_row, (int64_t)at.rows * scale_row);
      const int row = w ? kib * 64 + (lane & 32) + mx_feature((lane >> 4) & 1, lane & 15)
                        : (kib - TN / 64) * 64 + lane;
      s_rsrc[i] = w ? rw : rx;
      s_off[i] = (w || row < TM ? (uint32_t)(row * scale_row) : kDmaOutOfRange) - 16;
    }
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)lds;
  // A copy is two parts that stand behind different matrix instructions (together they would take
  // longer than one of them): where it goes, and the load.
  auto dma_to = [&](uint32_t dst) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, %1" : "={m0}"(m0) : "s"(__builtin_amdgcn_readfirstlane(dst)));
    return m0;
  };
  auto dma = [&](uint32_t m0, uint32_t offset, i32x4 rsrc) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds"
                 :: "v"(offset), "s"(rsrc), "{m0}"(m0) : "memory");
  };
  auto dma4 = [&](uint32_t dst, uint32_t offset, i32x4 rsrc) {      // a word per lane
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :: "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(offset), "s"(rsrc)
                 : "memory", "m0");
  };
  // Copies 0 .. kScaleLoads - 1 are the next group's scales, into buffer `buf`; those behind them
  // the next stage, into buffer `par`.
  auto aim_copy = [&](auto ic, auto par, int buf) {
    constexpr int i = decltype(ic)::value, c = i - kScaleLoads;
    const uint32_t stage_at = lds0 + decltype(par)::value * S::kStageBytes;
    if constexpr (c < 0) {
      s_off[i] += 16;
      return dma_to(lds0 + 2 * S::kStageBytes + buf * S::kScaleBytes +
                    (wave * kScaleLoads + i) * 1024);
    } else if constexpr (c < S::kLoadsW) {
      c_off[c] += 128;
      return dma_to(stage_at + (wave * S::kLoadsW + c) * 1024);
    } else {
      c_off[c] += 128;
      return dma_to(stage_at + TN * 128 + (wave * S::kLoadsX + c - S::kLoadsW) * 1024);
    }
  };
  auto copy = [&](auto ic, uint32_t m0) {
    constexpr int i = decltype(ic)::value, c = i - kScaleLoads;
    if constexpr (c < 0) dma(m0, s_off[i], s_rsrc[i]);
    else dma(m0, c_off[c], c < S::kLoadsW ? w_rsrc : x_rsrc);
  };
  auto copy_now = [&](auto ic, auto par, int buf) {
    const uint32_t m0 = aim_copy(ic, par, buf);
    asm volatile("s_nop 0");                           // between the write of m0 and the load
    copy(ic, m0);
  };
  constexpr int kFirst = kScaleLoads, kCopiesAll = kScaleLoads + S::kLoads;
  // Before the copies of stage `st`: past the end of K nothing is read any more, and of a last
  // stage of one step only the first four packs of a row.
  auto bound = [&](int st) {
    const bool past = st >= stages;
    if (!INT8 && st * 2 + 1 == steps) {              // (rows of 8-bit codes are whole stages)
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i)
        c_off[i] = pack_of(lane, i & 1) >= 4 ? kDmaOutOfRange : c_off[i];
    }
    w_rsrc[2] = past ? 0 : w_rsrc[2];
    x_rsrc[2] = past ? 0 : x_rsrc[2];
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) s_rsrc[i][2] = past ? 0 : s_rsrc[i][2];
  };
  // the bias comes by LDS where it is words throughout; it has x's type, which is y's
  constexpr int kBiasCopies = 2;                     // (16-bit types need only the first)
  constexpr int kFactorCopies = INT8 ? 4 : 0;        // the floats of 8-bit rows, likewise
  const bool wide = mx_quantises(MODE) ? a.dtype == FMOE_F32 : std::is_same<T, float>::value;
  const bool bias_by_lds = a.bias != nullptr &&
                           (wide || (a.out_feat % 2 == 0 && (uintptr_t)a.bias % 4 == 0));
  const int m = lane & 15, g = lane >> 4, wn = wave >> 1, wm = wave & 1;
  const int frag0 = m * 128 + (g ^ ((m >> 1) & 7)) * 16;      // step 0; step 1 has packs 4..7
  const char* const w_lds = lds + wn * (TN / 2) * 128;
  const char* const x_lds = lds + (TN + wm * (TM / 2)) * 128;
  i32x4 wf[2][FW], xf[2][TW];
  int wsc[FW], xsc[TW];            // per fragment, this lane's bytes of the group's 4 steps
  int wsn[FW], xsn[TW];            // the next group's
  // fragment j (features first) of step S of the stage in buffer `buf`
  auto read = [&](auto jc, auto step, auto buf) {
    constexpr int j = decltype(jc)::value, s = decltype(step)::value;
    const int at = decltype(buf)::value * S::kStageBytes + (s ? frag0 ^ 64 : frag0);
    if constexpr (j < FW) wf[s][j] = *(const i32x4*)(w_lds + at + j * 2048);
    else xf[s][j - FW] = *(const i32x4*)(x_lds + at + (j - FW) * 2048);
  };
  // byte g of each of a row's four words (the steps of a group)
  const uint32_t pick = (uint32_t)g | (uint32_t)(4 + g) << 8 | 0x0c0c0000u;
  const uint32_t last_mask = (steps & 3) ? (1u << (8 * (steps & 3))) - 1 : ~0u;
  // Scales are read kLag ahead of their use, so that nobody waits where they are read: call j
  // reads fragment j's and finishes fragment j - kLag's.
  constexpr int kLag = 4;
  i32x4 sraw[kLag];
  auto read_scale = [&](auto jc, int group, int buf) {
    constexpr int j = decltype(jc)::value;
    if constexpr (INT8) return;
    if constexpr (j >= kLag) {
      constexpr int d = j - kLag;
      const i32x4 b = sraw[d % kLag];
      const uint32_t lo = __builtin_amdgcn_perm((uint32_t)b[1], (uint32_t)b[0], pick);
      const uint32_t hi = __builtin_amdgcn_perm((uint32_t)b[3], (uint32_t)b[2], pick);
      // bytes behind the last step of K may hold anything, and 255 would make a NaN of a zero
      const int all = (int)(__builtin_amdgcn_perm(hi, lo, 0x05040100u) &
                            (group * 4 + 4 <= steps ? ~0u : last_mask));
      if constexpr (d < FW) wsn[d] = all;
      else xsn[d - FW] = all;
    }
    if constexpr (j < FW + TW) {
      const int row = j < FW ? wn * (TN / 2) + j * 16 : TN + wm * (TM / 2) + (j - FW) * 16;
      sraw[j % kLag] = *(const i32x4*)(lds + 2 * S::kStageBytes + buf * S::kScaleBytes +
                                       (row + m) * 16);
    }
  };
  // (In assembly so that they stay here: a matrix instruction reads what an ordinary one wrote two
  // wait states later at the earliest, and the compiler does not know that ours are such.)
  auto next_scales = [&] {
    if constexpr (INT8) return;
#pragma unroll
    for (int j = 0; j < FW; ++j) asm volatile("v_mov_b32 %0, %1" : "=v"(wsc[j]) : "v"(wsn[j]));
#pragma unroll
    for (int j = 0; j < TW; ++j) asm volatile("v_mov_b32 %0, %1" : "=v"(xsc[j]) : "v"(xsn[j]));
    asm volatile("s_nop 1");
  };
  using Acc = std::conditional_t<INT8, i32x4, f32x4>;
  Acc acc[TW][FW];
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;

  // Where things happen among the 2 * kMma instructions of a stage: the second step's fragments
  // are read behind the first ones, the buffer is released behind kRelease, the next stage is
  // published behind kPublish and its first fragments (and the next group's scales) are read.
  constexpr int kReads = FW + TW;
  constexpr int kWindow = kReads < kMma / 2 ? kReads : kMma / 2;
  constexpr int kRelease = kWindow + kMma / 8;
  constexpr int kPublish = kMma + kMma / 4;
  static_assert(kRelease < kMma && kPublish + kWindow < 2 * kMma, "room for the reads");
  // The stage in buffer `odd`; meanwhile the copies of stage `st` (of this tile or the next) into
  // the same buffer and, in an even stage, of its group's scales into `sbuf`.  `first`: of a tile
  // behind another one.
  constexpr int kSent = MODE == kMxAny ? 0
                            : MxOutput<T, MODE>::template stores<FW / 2, S::kOutRow>(TW);
  auto one_stage = [&](auto odd_c, int st, int sbuf, bool first) {
    constexpr int odd = decltype(odd_c)::value;
    using Odd = std::integral_constant<int, odd>;
    using Other = std::integral_constant<int, 1 - odd>;
    constexpr int kSkip = odd ? kFirst : 0, kCopies = kCopiesAll - kSkip;
    // of `count` things dealt over the instructions from .. from + len - 1, those out behind k
    constexpr auto dealt = [](int k, int from, int len, int count) {
      const int n = k < from ? 0 : (k - from + 1) * count / len;
      return n < count ? n : count;
    };
    // copies aimed up to instruction k, and issued: an instruction later where there is room
    constexpr int kFrom = kRelease + 1, kLen = 2 * kMma - kFrom - 1;
    constexpr bool kApart = 2 * kCopies <= kLen;
    constexpr auto aimed = [dealt](int k) { return dealt(k, kFrom, kLen, kCopies); };
    constexpr auto copied = [aimed](int k) { return aimed(kApart ? k - 1 : k); };
    uint32_t m0 = 0;
    auto issue = [&](auto kc) {
      constexpr int k = decltype(kc)::value;
      if constexpr (kApart) {
        unroll<kSkip + copied(k - 1), kSkip + copied(k)>([&](auto c) { copy(c, m0); });
        unroll<kSkip + aimed(k - 1), kSkip + aimed(k)>(
            [&](auto c) { m0 = aim_copy(c, Odd{}, sbuf); });
      } else {
        unroll<kSkip + copied(k - 1), kSkip + copied(k)>(
            [&](auto c) { copy_now(c, Odd{}, sbuf); });
      }
    };
    auto scale_reads = [&](auto kc) {
      constexpr int k = decltype(kc)::value, from = kRelease + 1, len = kPublish - kRelease;
      if constexpr (odd)
        unroll<dealt(k - 1, from, len, kReads + kLag), dealt(k, from, len, kReads + kLag)>(
            [&](auto j) { read_scale(j, st >> 1, sbuf); });
    };
    bound(st);
    unroll<0, kMma>([&](auto kc) {
      constexpr int k = decltype(kc)::value, i = k / FW, f = k % FW;
      if constexpr (INT8) i8_mfma_at(wf[0][f], xf[0][i], acc[i][f]);
      else mx_mfma_at<2 * odd>(wf[0][f], wsc[f], xf[0][i], xsc[i], acc[i][f]);
      unroll<dealt(k - 1, 0, kWindow, kReads), dealt(k, 0, kWindow, kReads)>(
          [&](auto j) { read(j, C1{}, Odd{}); });
      if constexpr (k == kRelease) {
        __builtin_amdgcn_s_waitcnt(0xc07f);           // lgkmcnt(0): my reads of this stage are done
        // the next group's scales have landed; behind them the last stage's copies were issued
        if constexpr (odd && !INT8) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
      }
      scale_reads(kc);
      issue(kc);
      __builtin_amdgcn_sched_barrier(0);
    });
    unroll<kMma, 2 * kMma>([&](auto kc) {
      constexpr int k = decltype(kc)::value, i = (k - kMma) / FW, f = (k - kMma) % FW;
      if constexpr (INT8) i8_mfma_at(wf[1][f], xf[1][i], acc[i][f]);
      else mx_mfma_at<2 * odd + 1>(wf[1][f], wsc[f], xf[1][i], xsc[i], acc[i][f]);
      if constexpr (k == kPublish) {
        // everything but this stage's own copies has landed; the last tile's results, the bias and
        // the factors, which lie between a tile's second stage and its third, may still be on their way
        constexpr int own = copied(kPublish - 1), most = 63;
        constexpr int behind = own + kSent + kFactorCopies;
        constexpr int sent = behind < most ? behind : most;
        constexpr int sent_bias = behind + kBiasCopies < most ? behind + kBiasCopies : most;
        static_assert(own < 64, "vmcnt is a 6-bit counter");
        if (!odd && first && bias_by_lds && kSent > 0)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(sent_bias) : "memory");
        else if (!odd && first) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(sent) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(own) : "memory");
        __builtin_amdgcn_s_barrier();
      }
      constexpr int r0 = kPublish + 1;
      unroll<dealt(k - 1, r0, kWindow, kReads), dealt(k, r0, kWindow, kReads)>(
          [&](auto j) { read(j, C0{}, Other{}); });
      scale_reads(kc);
      issue(kc);
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (odd) next_scales();
  };

  char* const stage = lds + 2 * (S::kStageBytes + S::kScaleBytes) + wave * (16 * S::kOutRow);
  char* const factors = INT8 ? lds + 2 * (S::kStageBytes + S::kScaleBytes) + S::kOutBytes + wave * 2048
                             : stage;
  // (the last group's missing steps, if any, multiply zeros)
  const int groups = (steps + 3) >> 2;
  int pid = blockIdx.x;
  int number = tile_number(pid, live);
  if (number >= live) return;
  MxPlace at = place(number), next = at;
  bool first = false;
  int sbuf = 0;                                       // buffer of the current group's scales
  aim(at);
  bound(0);
  unroll<0, kCopiesAll>([&](auto i) { copy_now(i, C0{}, 0); });
  bound(1);
  unroll<kFirst, kCopiesAll>([&](auto i) { copy_now(i, C1{}, 0); });
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoads) : "memory");
  __builtin_amdgcn_s_barrier();
  unroll<0, FW + TW>([&](auto j) { read(j, C0{}, C0{}); });
  unroll<0, FW + TW + kLag>([&](auto j) { read_scale(j, 0, 0); });
  next_scales();
  for (;;) {
    // the bias waits out the K loop, of 4-bit rows where the results will pass
    if (bias_by_lds) {
      const int64_t row = (int64_t)a.out_feat * (wide ? 4 : 2);
      const i32x4 rsrc = mx_descriptor((const char*)a.bias + at.e * row, row);
      const uint32_t dst = lds0 + (uint32_t)(factors - lds);
      const uint32_t off = (uint32_t)((at.base + wn * (TN / 2)) * (wide ? 4 : 2) + lane * 4);
      dma4(dst, off, rsrc);
      dma4(dst + 256, off + 256, rsrc);
    }
    // and the scales of 8-bit rows with it: the wave's features' at 512, its rows' at 1024 (128 of
    // either, which may be more than it has)
    if constexpr (INT8) {
      const uint32_t dst = lds0 + (uint32_t)(factors - lds);
      const i32x4 rw = mx_descriptor(a.ws + ((int64_t)at.e * a.out_feat + at.base) * 4,
                                     (int64_t)(a.out_feat - at.base) * 4);
      const i32x4 rx = mx_descriptor(a.xs + at.x0 * 4, (int64_t)at.rows * 4);
      const uint32_t w_off = (uint32_t)(wn * (TN / 2) + lane) * 4;
      const uint32_t x_off = (uint32_t)(wm * (TM / 2) + lane) * 4;
      dma4(dst + 512, w_off, rw);
      dma4(dst + 768, w_off + 256, rw);
      dma4(dst + 1024, x_off, rx);
      dma4(dst + 1280, x_off + 256, rx);
    }
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
      for (int f = 0; f < FW; ++f) acc[i][f] = Acc{};
    bool more = true;
    int q = 0;
    do {
      int st = 2 * q + 2;                             // the stages copied meanwhile
      if (q + 1 == groups) {
        st = 0;
        pid += gridDim.x;
        number = tile_number(pid, live);
        more = number < live;
        if (more) {
          next = place(number);
          aim(next);
        } else {
          bound(stages);                              // nothing any more
        }
      }
      one_stage(C0{}, st, sbuf ^ 1, first);
      one_stage(C1{}, st + 1, sbuf ^ 1, false);
      sbuf ^= 1;
      first = false;
    } while (++q < groups);
    mx_mfma_done();
    const int fresh = mx_fresh(lane);
    auto read_bias = [&](int p, float (&b)[8]) {
      if (bias_by_lds) {
        const char* const at_g = factors + (fresh >> 4) * (wide ? 32 : 16);
        if (wide) {
#pragma unroll
          for (int i = 0; i < 8; ++i) b[i] = *(const float*)(at_g + p * 128 + i * 4);
        } else {
          const i32x4 u = *(const i32x4*)(at_g + p * 64);
          mx_widen(a, u, b);
        }
      } else {
        mx_load_bias(a, mx_bias_rows(a, at.e), at.base + wn * (TN / 2) + p * 32 + 8 * (fresh >> 4), b);
      }
    };
    auto read_factors = [&](int p, float (&sw)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        sw[j] = *(const float*)(factors + 512 + (p * 32 + 8 * (fresh >> 4) + j) * 4);
    };
    // (held for all rows; but where rows are not whole packs and the tile is the largest, registers
    // do not suffice, and these are read for every 16 rows)
    constexpr bool kHold = !(INT8 && MODE == kMxAny && TN == 256);
    float b[FW / 2][8], sw[FW / 2][8];
    if constexpr (kHold) {
#pragma unroll
      for (int p = 0; p < FW / 2; ++p) {
        read_bias(p, b[p]);
        if constexpr (INT8) read_factors(p, sw[p]);
      }
    }
    const MxOutput<T, MODE> out(a, at.x0, at.rows);
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      float r[FW / 2][8], sx = 1.f;
      if constexpr (INT8) sx = *(const float*)(factors + 1024 + (i * 16 + (fresh & 15)) * 4);
#pragma unroll
      for (int p = 0; p < FW / 2; ++p) {
        if constexpr (!kHold) {
          read_bias(p, b[p]);
          read_factors(p, sw[p]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = mx_read(acc[i][2 * p + (j >> 2)][j & 3]);
          r[p][j] = INT8 ? fmaf(v * sx, sw[p][j], b[p][j]) : v + b[p][j];
        }
      }
      out.template store_rows<FW / 2, S::kOutRow>(stage, fresh, wm * (TM / 2) + i * 16,
                                                  at.base + wn * (TN / 2), r);
    }
    if (!more) break;
    at = next;
    first = true;
    // (the corner is read out before the next bias lands there)
    __builtin_amdgcn_s_waitcnt(0xc07f);
    // With more experts than lanes, place() writes to the first wave's corner from another one.  A
    // tile of one group calls it before the K loop's first barrier, so it waits here until the
    // first wave's results have left.
    if (groups == 1 && !tiles.by_lane) __syncthreads();
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing may land in LDS after the end
}

}  // namespace fmoe
