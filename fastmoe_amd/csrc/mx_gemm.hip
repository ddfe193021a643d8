// Grouped product of MXFP4 rows with MXFP4 expert weights on gfx950 (the format: mx.h):
//   y[r][n] = sum_k x[r][k] w_e[n][k] + b_e[n],   r in the rows of expert e,
// and, for the first of an expert's two layers, act(y) quantised again: y never reaches memory.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows of 128 codes by 16 rows of 128 codes and
// applies both operands' block scales itself, with f32 sums: lane l holds row l % 16, features
// 32 (l / 16) .. +31, i.e. one block, 16 bytes of codes and one scale byte.  The weights are the
// first operand (result rows = output features), so a lane ends up with 4 consecutive features
// of one token per fragment.  Which weight row a lane reads is free: fragment f of a group of 32
// features gives lane row m the feature 8 (m / 4) + 4 f + m % 4, so the two fragments of a group
// leave 8 CONSECUTIVE features of a token in a lane, and a block of 32 in four lanes: the output
// leaves in 16-byte packs, and the block maximum of the quantising epilogue takes two exchanges.
//
// Few rows are bound by the weights' bytes (17/32 of one per weight), many by the matrix cores;
// which of two kernels and three tile shapes runs: choose_kernel().
#include <algorithm>
#include <type_traits>

#include "dma_desc.h"
#include "gemm_tiles.h"
#include "mx.h"

namespace fmoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct MxGemmArgs {
  const uint8_t *xc, *xs, *wc, *ws;
  const void* bias;            // [E, out] or null
  const int32_t* seg_off;
  void* y;                     // [n_rows, out], or null with yc
  uint8_t *yc, *ys;            // rows of `out` features
  int64_t n_rows;
  int in_feat, out_feat, n_expert, dtype;
};

__device__ __forceinline__ f32x4 mx_mfma(i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
  const i32x8 a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 b8 = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  // 4 = E2M1 in either operand; the scale bytes are the lowest ones of sa and sb
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, sa, 0, sb);
}

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

// gelu(x) = x Phi(x) with Phi(x) = 1 / (1 + 2^z), z = -log2(Phi(x) / Phi(-x)) = x P(x^2) for
// |x| <= 6 and x P(36) outside: P of degree 12 in x^2 / 18 - 1, a reweighted least-squares fit on
// Chebyshev nodes.  Within 2e-7 + 3e-7 |gelu| of gelu everywhere (the fit, evaluated in f32 with an
// exact exponential and quotient: 1.42e-7 + 1e-7 |gelu|; the two instructions for these are good to
// 1.2e-7 each), so that hardly more codes than the sums' own rounding makes land on the other side
// of a boundary (degree 9, three instructions less, was off by 7e-7), and, for |x| <= 6, within
// 5e-6 of its value (3.7e-6 likewise), so that blocks whose values all lie in the negative tail
// keep their digits as well.  26 issue slots where erff takes about
// 60, with branches, and loses the tail: with one wave on a SIMD nothing hides them (a 256 x 256
// tile of 4096 features: 27 us of matrix instructions, 26 us of erff).
__device__ __forceinline__ float mx_gelu(float x) {
  const float t = fminf(fmaf(x * x, 1.f / 18.f, -1.f), 1.f);
  float p = 0.00220932276f;
  p = fmaf(p, t, -0.00235819351f);
  p = fmaf(p, t, -0.00623256993f);
  p = fmaf(p, t, 0.0106137199f);
  p = fmaf(p, t, -0.00437692506f);
  p = fmaf(p, t, 0.0022452944f);
  p = fmaf(p, t, -0.00346183078f);
  p = fmaf(p, t, -0.00412944285f);
  p = fmaf(p, t, 0.0250278097f);
  p = fmaf(p, t, -0.0735082775f);
  p = fmaf(p, t, 0.223777682f);
  p = fmaf(p, t, -1.27482498f);
  p = fmaf(p, t, -3.8811202f);
  // (2^z overflows to infinity far down, its inverse is 0 there)
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * p));
}

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
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_bias_rows(const MxGemmArgs& a, int e) {
  const int64_t bytes = (int64_t)a.out_feat * (a.dtype == FMOE_F32 ? 4 : 2);
  return mx_resource((const char*)a.bias + e * bytes, a.bias ? bytes : 0);
}
// 8 values of the bias's 16-bit type.
__device__ __forceinline__ void mx_widen(const MxGemmArgs& a, i32x4 u, float (&b)[8]) {
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
__device__ __forceinline__ void mx_load_bias(const MxGemmArgs& a, __amdgpu_buffer_rsrc_t rows,
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
  __device__ __forceinline__ MxOutput(const MxGemmArgs& a, int64_t x0, int rows_) {
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
      if (MODE == kMxQuantGelu) v[i] = mx_gelu(v[i]);
      if (MODE == kMxQuantRelu) v[i] = __builtin_elementwise_maximum(v[i], 0.f);   // (a NaN stays)
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

// ------------------------------------------------------------------------- few rows
// Weights straight from memory into registers, since nothing would read them twice: a workgroup's
// 4 waves take 16 rows of an expert, 32 features, and a quarter of K each, whose sums meet in LDS.
// K is split because there are few tiles otherwise: 128 rows of 16 experts, 4096 -> 1024, are 512
// workgroups and take 10 us (36 MB; 7 at the rate of a large copy) where 128 x 64 tiles take 13.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void mx_stream_kernel(MxGemmArgs a) {
  constexpr int kWaves = 4, kCols = 32;
  __shared__ int s_sum[2 * kWaves], s_out[4];
  __shared__ float part[(kWaves - 1) * 8 * kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowTiles<16, kOneHeight, kWaves> tiles;
  tiles.scan(a.seg_off, a.n_expert, s_sum);
  const int n_pad = mx_quantises(MODE) ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const int n_cols = (n_pad + kCols - 1) / kCols;
  if (tiles.rows_f == 0) return;
  const int col = blockIdx.x / tiles.rows_f, v = blockIdx.x - col * tiles.rows_f;
  if (col >= n_cols) return;
  const TileRows t = tiles.find(a.seg_off, v, false, s_out);

  const int m = lane & 15, g = lane >> 4, base = col * kCols;
  const int64_t code_row = mx_code_bytes(a.in_feat), scale_row = mx_scale_bytes(a.in_feat);
  // rows and features past the end repeat the last one; their results are not stored
  const uint8_t *wc[2], *ws[2];
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const int64_t n = (int64_t)t.e * a.out_feat + min(base + mx_feature(f, m), a.out_feat - 1);
    wc[f] = a.wc + n * code_row + g * 16;
    ws[f] = a.ws + n * scale_row;
  }
  const int64_t r = (int64_t)t.row0 + min(t.m0 + m, t.cnt - 1);
  const uint8_t *const xc = a.xc + r * code_row + g * 16, *const xs = a.xs + r * scale_row;
  const int steps = (a.in_feat + kMxStep - 1) / kMxStep, groups = (steps + 3) / 4;
  const int g1 = (wave + 1) * groups / kWaves;
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  for (int q = wave * groups / kWaves; q < g1; ++q) {
    const i32x4 xsv = *(const i32x4*)(xs + q * 16);
    i32x4 wsv[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) wsv[f] = *(const i32x4*)(ws[f] + q * 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (q * 4 + s >= steps) break;
      const int64_t off = (int64_t)(q * 4 + s) * 64;
      const i32x4 x = *(const i32x4*)(xc + off);
#pragma unroll
      for (int f = 0; f < 2; ++f)
        acc[f] = mx_mfma(*(const i32x4*)(wc[f] + off), (int)((uint32_t)wsv[f][s] >> (8 * g)), x,
                         (int)((uint32_t)xsv[s] >> (8 * g)), acc[f]);
    }
  }
  // the quarters meet in the first wave, always in the same order
  if (wave > 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[((wave - 1) * 8 + j) * kWave + lane] = acc[j >> 2][j & 3];
  }
  __syncthreads();
  if (wave > 0) return;
  float b[8], y[8];
  mx_load_bias(a, mx_bias_rows(a, t.e), base + 8 * g, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    y[j] = acc[j >> 2][j & 3];
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) y[j] += part[(w * 8 + j) * kWave + lane];
    y[j] += b[j];
  }
  const MxOutput<T, MODE> out(a, (int64_t)t.row0 + t.m0, min(16, t.cnt - t.m0));
  out.store(m, base + 8 * g, y);
}

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
// An accumulator's value.  (Read like this, accumulators have no use in which they would have to
// be ordinary registers, so that they stay where the matrix instructions want them.)
__device__ __forceinline__ float mx_read(float c) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(c));
  return v;
}
// The 18 wait states between the last matrix instruction and a read of its result.
__device__ __forceinline__ void mx_mfma_done() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

template <int TN, int TM> struct MxTile {
  static constexpr int kStageBytes = (TN + TM) * 128;
  static constexpr int kLoadsW = TN / 32, kLoadsX = TM / 32;       // copies of a wave per stage
  static constexpr int kLoads = kLoadsW + kLoadsX;
  static constexpr int kScaleLoads = ((TN + TM) / 64 + 3) / 4;     // and per group of scales
  static constexpr int kScaleBytes = kScaleLoads * 4096;
  static constexpr int kOutRow = TN <= 128 ? 128 : 256;            // bytes of a row on its way out
  static constexpr int kOutBytes = 4 * 16 * kOutRow;
  static constexpr int kLdsBytes = 2 * (kStageBytes + kScaleBytes) + kOutBytes;
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

template <typename T, int TN, int TM, int MODE>
__global__ __launch_bounds__(256, (MxTile<TN, TM>::kGroups)) void mx_tile_kernel(MxGemmArgs a) {
  using S = MxTile<TN, TM>;
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
  const int code_row = (int)mx_code_bytes(a.in_feat), scale_row = (int)mx_scale_bytes(a.in_feat);
  const int steps = __builtin_amdgcn_readfirstlane((a.in_feat + kMxStep - 1) / kMxStep);
  const int stages = (steps + 1) / 2;

  // The offset a lane fetches from in each of its wave's copies, one stage (of the scales: one
  // group) back: a copy moves its own on.
  uint32_t c_off[S::kLoads], s_off[S::kScaleLoads];
  i32x4 w_rsrc, x_rsrc, s_rsrc[S::kScaleLoads];
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
    for (int i = 0; i < S::kScaleLoads; ++i) {
      const int kib = wave * S::kScaleLoads + i;
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
    constexpr int i = decltype(ic)::value, c = i - S::kScaleLoads;
    const uint32_t stage_at = lds0 + decltype(par)::value * S::kStageBytes;
    if constexpr (c < 0) {
      s_off[i] += 16;
      return dma_to(lds0 + 2 * S::kStageBytes + buf * S::kScaleBytes +
                    (wave * S::kScaleLoads + i) * 1024);
    } else if constexpr (c < S::kLoadsW) {
      c_off[c] += 128;
      return dma_to(stage_at + (wave * S::kLoadsW + c) * 1024);
    } else {
      c_off[c] += 128;
      return dma_to(stage_at + TN * 128 + (wave * S::kLoadsX + c - S::kLoadsW) * 1024);
    }
  };
  auto copy = [&](auto ic, uint32_t m0) {
    constexpr int i = decltype(ic)::value, c = i - S::kScaleLoads;
    if constexpr (c < 0) dma(m0, s_off[i], s_rsrc[i]);
    else dma(m0, c_off[c], c < S::kLoadsW ? w_rsrc : x_rsrc);
  };
  auto copy_now = [&](auto ic, auto par, int buf) {
    const uint32_t m0 = aim_copy(ic, par, buf);
    asm volatile("s_nop 0");                           // between the write of m0 and the load
    copy(ic, m0);
  };
  constexpr int kFirst = S::kScaleLoads, kCopiesAll = S::kScaleLoads + S::kLoads;
  // Before the copies of stage `st`: past the end of K nothing is read any more, and of a last
  // stage of one step only the first four packs of a row.
  auto bound = [&](int st) {
    const bool past = st >= stages;
    if (st * 2 + 1 == steps) {
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i)
        c_off[i] = pack_of(lane, i & 1) >= 4 ? kDmaOutOfRange : c_off[i];
    }
    w_rsrc[2] = past ? 0 : w_rsrc[2];
    x_rsrc[2] = past ? 0 : x_rsrc[2];
#pragma unroll
    for (int i = 0; i < S::kScaleLoads; ++i) s_rsrc[i][2] = past ? 0 : s_rsrc[i][2];
  };
  // the bias comes by LDS where it is words throughout; it has x's type, which is y's
  constexpr int kBiasCopies = 2;                     // (16-bit types need only the first)
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
#pragma unroll
    for (int j = 0; j < FW; ++j) asm volatile("v_mov_b32 %0, %1" : "=v"(wsc[j]) : "v"(wsn[j]));
#pragma unroll
    for (int j = 0; j < TW; ++j) asm volatile("v_mov_b32 %0, %1" : "=v"(xsc[j]) : "v"(xsn[j]));
    asm volatile("s_nop 1");
  };
  f32x4 acc[TW][FW];
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
      mx_mfma_at<2 * odd>(wf[0][f], wsc[f], xf[0][i], xsc[i], acc[i][f]);
      unroll<dealt(k - 1, 0, kWindow, kReads), dealt(k, 0, kWindow, kReads)>(
          [&](auto j) { read(j, C1{}, Odd{}); });
      if constexpr (k == kRelease) {
        __builtin_amdgcn_s_waitcnt(0xc07f);           // lgkmcnt(0): my reads of this stage are done
        // the next group's scales have landed; behind them the last stage's copies were issued
        if constexpr (odd) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
      }
      scale_reads(kc);
      issue(kc);
      __builtin_amdgcn_sched_barrier(0);
    });
    unroll<kMma, 2 * kMma>([&](auto kc) {
      constexpr int k = decltype(kc)::value, i = (k - kMma) / FW, f = (k - kMma) % FW;
      mx_mfma_at<2 * odd + 1>(wf[1][f], wsc[f], xf[1][i], xsc[i], acc[i][f]);
      if constexpr (k == kPublish) {
        // everything but this stage's own copies has landed; the last tile's results and the bias,
        // which lie between a tile's second stage and its third, may still be on their way
        constexpr int own = copied(kPublish - 1), most = 63;
        constexpr int sent = own + kSent < most ? own + kSent : most;
        constexpr int sent_bias = own + kSent + kBiasCopies < most ? own + kSent + kBiasCopies : most;
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
    // the bias waits out the K loop where the results will pass
    if (bias_by_lds) {
      const int64_t row = (int64_t)a.out_feat * (wide ? 4 : 2);
      const i32x4 rsrc = mx_descriptor((const char*)a.bias + at.e * row, row);
      const uint32_t dst = lds0 + (uint32_t)(stage - lds);
      const uint32_t off = (uint32_t)((at.base + wn * (TN / 2)) * (wide ? 4 : 2) + lane * 4);
      dma4(dst, off, rsrc);
      dma4(dst + 256, off + 256, rsrc);
    }
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
      for (int f = 0; f < FW; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};
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
    float b[FW / 2][8];
    const int fresh = mx_fresh(lane);
    if (bias_by_lds) {
      const char* const at_g = stage + (fresh >> 4) * (wide ? 32 : 16);
#pragma unroll
      for (int p = 0; p < FW / 2; ++p) {
        if (wide) {
#pragma unroll
          for (int i = 0; i < 8; ++i) b[p][i] = *(const float*)(at_g + p * 128 + i * 4);
        } else {
          const i32x4 u = *(const i32x4*)(at_g + p * 64);
          mx_widen(a, u, b[p]);
        }
      }
    } else {
      const auto rows = mx_bias_rows(a, at.e);
#pragma unroll
      for (int p = 0; p < FW / 2; ++p)
        mx_load_bias(a, rows, at.base + wn * (TN / 2) + p * 32 + 8 * (fresh >> 4), b[p]);
    }
    const MxOutput<T, MODE> out(a, at.x0, at.rows);
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      float r[FW / 2][8];
#pragma unroll
      for (int p = 0; p < FW / 2; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) r[p][j] = mx_read(acc[i][2 * p + (j >> 2)][j & 3]) + b[p][j];
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

constexpr int kCus = 256;

// Which kernel: by the mean number of rows per expert, the features and the number of tiles this
// makes.  Measured with three sets of operands in turn (us; GELU and quantisation behind the
// products marked q), with even loads and, behind the slash, with half of all rows on one expert;
// two runs differ by up to 10 % below 100 us:
//   rows  experts  in -> out        stream     128x64   128x128  256x256
//    128   16    4096 -> 1024      11 / 13    12 / 12   14 / 14   27 / 27
//     64   16    1024 -> 4096      12 / 12    10 / 10   11 / 11   16 / 15
//    128    8    4096 -> 14336 q   68 / 85    54 / 51   60 / 62   91 / 90
//   4096   32    4096 -> 1024     114 / 118   18 / 26   18 / 25   29 / 29
//  15560  128    2048 -> 1408 q   338 / 280   78 / 75   62 / 78  102 / 130
//  30000   16    2048 -> 2048     727 / 725  110 / 109  80 / 79   74 / 74
//  32768    8    4096 -> 14336              1649 / 1661 1222 / 1231 917 / 959
//  16384    4    4096 -> 11008 q             696 / 706  510 / 526  495 / 515
//  32768    8    4096 -> 14336 q            1806 / 1825 1326 / 1384 1235 / 1272
// The mean stands for both: what it picks is within 5 % of the best under these uneven loads too.
// Few rows and few tiles: the kernel that splits K.  The largest tiles move the least through L2
// and win where K is long and there are rounds enough of them; smaller ones share a CU by two, so
// that one's beginning and end (with GELU, half its time) are the other's middle.
enum MxKernel { kStream, kTile128x64, kTile128x128, kTile256x256 };
static MxKernel choose_kernel(const MxGemmArgs& a) {
  const double live = (double)std::min<int64_t>(a.n_expert, a.n_rows);
  const double mean = (double)a.n_rows / a.n_expert;
  // (an expert's last tile is half empty on average)
  auto tiles = [&](int tn, int tm) {
    return std::max((double)a.n_rows / tm + live / 2, live) * ceil_div(a.out_feat, tn);
  };
  if (mean <= 16 && tiles(128, 64) <= kCus / 2) return kStream;
  if (mean < 56) return kTile128x64;
  const bool quant = a.yc != nullptr;
  if (mean >= 192 && a.in_feat >= (quant ? 4096 : 2048) && tiles(256, 256) >= (quant ? 4000 : 600))
    return kTile256x256;
  return kTile128x128;
}

template <typename T, int MODE>
static int launch(const MxGemmArgs& a, hipStream_t s) {
  const int n_pad = mx_quantises(MODE) ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
#define FMOE_TILE(TN, TM)                                                                        \
  do {                                                                                           \
    const int64_t rows = a.n_rows / TM + std::min<int64_t>(a.n_expert, a.n_rows);                \
    FMOE_REQUIRE(rows * ceil_div(n_pad, TN) <= INT32_MAX, FMOE_ERR_UNSUPPORTED,                  \
                 "mx_linear: too many tiles");                                                   \
    FMOE_SET_DYNAMIC_LDS_ONCE((mx_tile_kernel<T, TN, TM, MODE>), (MxTile<TN, TM>::kLdsBytes));   \
    hipLaunchKernelGGL((mx_tile_kernel<T, TN, TM, MODE>), dim3(kCus * MxTile<TN, TM>::kGroups),  \
                       dim3(256), (MxTile<TN, TM>::kLdsBytes), s, a);                            \
  } while (0)
  switch (choose_kernel(a)) {
    case kStream: {
      const int64_t rows = a.n_rows / 16 + std::min<int64_t>(a.n_expert, a.n_rows);
      hipLaunchKernelGGL((mx_stream_kernel<T, MODE>), dim3((unsigned)(rows * ceil_div(n_pad, 32))),
                         dim3(256), 0, s, a);      // (few tiles, or this kernel is not chosen)
      break;
    }
    case kTile128x64: FMOE_TILE(128, 64); break;
    case kTile128x128: FMOE_TILE(128, 128); break;
    case kTile256x256: FMOE_TILE(256, 256); break;
  }
#undef FMOE_TILE
  FMOE_LAUNCH_CHECK("mx_linear");
  return FMOE_OK;
}

template <typename T> static int launch_y(const MxGemmArgs& a, hipStream_t s) {
  constexpr int kN = Pack16<T>::kN;
  return a.out_feat % kN == 0 && (uintptr_t)a.y % 16 == 0 ? launch<T, kMxPacked>(a, s)
                                                          : launch<T, kMxAny>(a, s);
}

}  // namespace fmoe

extern "C" int fmoe_mx_linear_fwd(const void* x_codes, const void* x_scales, const void* w_codes,
                                  const void* w_scales, const void* bias, const int32_t* seg_off,
                                  int act, void* y, void* y_codes, void* y_scales, int64_t n_rows,
                                  int64_t in_feat, int64_t out_feat, int64_t n_expert, int dtype,
                                  void* stream) {
  using namespace fmoe;
  FMOE_REQUIRE(n_rows >= 0 && n_rows < INT32_MAX && n_expert >= 1 && n_expert < INT32_MAX &&
                   in_feat >= 1 && out_feat >= 1 && in_feat <= FMOE_MX_MAX_FEATURES &&
                   out_feat <= FMOE_MX_MAX_FEATURES,
               FMOE_ERR_INVALID, "mx_linear: bad sizes");
  FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_F16 || dtype == FMOE_BF16, FMOE_ERR_UNSUPPORTED,
               "mx_linear: unsupported dtype %d", dtype);
  FMOE_REQUIRE(act == FMOE_ACT_NONE || act == FMOE_ACT_GELU || act == FMOE_ACT_RELU,
               FMOE_ERR_INVALID, "mx_linear: unknown activation %d", act);
  FMOE_REQUIRE(act == FMOE_ACT_NONE || y == nullptr, FMOE_ERR_INVALID,
               "mx_linear: an activation only in front of y_codes");
  if (n_rows == 0) return FMOE_OK;
  FMOE_REQUIRE(x_codes && x_scales && w_codes && w_scales && seg_off, FMOE_ERR_INVALID,
               "mx_linear: null pointer");
  FMOE_REQUIRE((y != nullptr) != (y_codes != nullptr) && (y_codes != nullptr) == (y_scales != nullptr),
               FMOE_ERR_INVALID, "mx_linear: either y, or y_codes and y_scales");
  FMOE_REQUIRE(((uintptr_t)x_codes | (uintptr_t)x_scales | (uintptr_t)w_codes |
                (uintptr_t)w_scales | (uintptr_t)y_codes | (uintptr_t)y_scales) % 16 == 0,
               FMOE_ERR_INVALID, "mx_linear: codes and scales must be 16-byte aligned");
  const MxGemmArgs a{(const uint8_t*)x_codes, (const uint8_t*)x_scales, (const uint8_t*)w_codes,
                     (const uint8_t*)w_scales, bias, seg_off, y, (uint8_t*)y_codes,
                     (uint8_t*)y_scales, n_rows, (int)in_feat, (int)out_feat, (int)n_expert, dtype};
  hipStream_t s = (hipStream_t)stream;
  if (y_codes)      // (the element type then is that of the bias alone, which is read as it comes)
    return act == FMOE_ACT_GELU   ? launch<float, kMxQuantGelu>(a, s)
           : act == FMOE_ACT_RELU ? launch<float, kMxQuantRelu>(a, s)
                                  : launch<float, kMxQuant>(a, s);
  switch (dtype) {
    case FMOE_F32: return launch_y<float>(a, s);
    case FMOE_F16: return launch_y<__half>(a, s);
    default: return launch_y<__hip_bfloat16>(a, s);
  }
}
