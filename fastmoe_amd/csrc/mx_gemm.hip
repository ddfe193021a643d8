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
// is stored in 16-byte packs straight from the registers, and the block maximum of the quantising
// epilogue takes two exchanges.
#include <algorithm>
#include <type_traits>

#include "act_math.h"
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
  int in_feat, out_feat, n_expert, act, dtype;
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

// What a tile writes: descriptors that end with its last valid row, so that rows past the end
// need no branch, and the bias of its expert.
template <typename T, bool QUANT> struct MxOutput {
  __amdgpu_buffer_rsrc_t y, yc, ys, bias;
  int n, size, bias_dtype, act;
  bool packed, has_bias;

  // rows x0 .. x0 + rows - 1 of the output, of expert e
  __device__ __forceinline__ MxOutput(const MxGemmArgs& a, int e, int64_t x0, int rows) {
    n = a.out_feat;
    act = a.act;
    bias_dtype = a.dtype;
    has_bias = a.bias != nullptr;
    const int bsize = a.dtype == FMOE_F32 ? 4 : 2;
    bias = resource((const char*)a.bias + (int64_t)e * n * bsize, (int64_t)n * bsize);
    if (QUANT) {
      const int64_t cr = mx_code_bytes(n), sr = mx_scale_bytes(n);
      yc = resource(a.yc + x0 * cr, rows * cr);
      ys = resource(a.ys + x0 * sr, rows * sr);
    } else {
      y = resource((T*)a.y + x0 * n, (int64_t)rows * n * sizeof(T));
      packed = n % 8 == 0 && (uintptr_t)a.y % 16 == 0;
    }
  }
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, int64_t bytes) {
    const uint64_t u = (uint64_t)p;
    void* q = (void*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32) |
                      (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u));
    return __builtin_amdgcn_make_buffer_rsrc(
        q, 0, __builtin_amdgcn_readfirstlane(dma_num_records(bytes)), 0x00020000);
  }

  // The bias of features n0 .. n0 + 7 (zero behind the last one, and without a bias).
  __device__ __forceinline__ void load_bias(int n0, float (&b)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.f;
    if (!has_bias) return;
    if (bias_dtype == FMOE_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        b[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(bias, (n0 + i) * 4, 0, 0));
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t u = __builtin_amdgcn_raw_buffer_load_b16(bias, (n0 + i) * 2, 0, 0);
      b[i] = bias_dtype == FMOE_BF16 ? __uint_as_float((uint32_t)u << 16)
                                     : __half2float(__builtin_bit_cast(__half, u));
    }
  }

  // Activation and output of features n0 .. n0 + 7 of the tile's row `row`.  All lanes of a wave
  // come here together; lanes l, l ^ 16, l ^ 32 and l ^ 48 hold one block of 32 features.
  __device__ __forceinline__ void store(int row, int n0, float (&v)[8]) const {
    if (act == FMOE_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = gelu_direct(v[i]);
    } else if (act == FMOE_ACT_RELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];   // (a NaN stays)
    }
    if constexpr (!QUANT) {
      const uint32_t at = ((uint32_t)row * n + n0) * (uint32_t)sizeof(T);
      T o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = Elem<T>::from_acc(v[i]);
      if (packed) {
        const uint32_t to = n0 < n ? at : kDmaOutOfRange;
#pragma unroll
        for (int p = 0; p < (int)sizeof(T) / 2; ++p) {
          i32x4 w;
          __builtin_memcpy(&w, (const char*)o + p * 16, 16);
          __builtin_amdgcn_raw_buffer_store_b128(w, y, to, p * 16, 0);
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
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = n0 + i < n ? v[i] : 0.f;
        m = max(m, magnitude_bits(v[i]));
      }
      m = max(m, (uint32_t)__shfl_xor((int)m, 16, kWave));
      m = max(m, (uint32_t)__shfl_xor((int)m, 32, kWave));
      const int byte = mx_scale_byte(m);
      const int cr = (int)mx_code_bytes(n), sr = (int)mx_scale_bytes(n);
      const bool in = n0 < cr * 2;
      __builtin_amdgcn_raw_buffer_store_b32(mx_codes(v, byte), yc,
                                            in ? row * cr + n0 / 2 : kDmaOutOfRange, 0, 0);
      // (the row's scales reach at least as far as its codes)
      const bool first = in && (n0 & 31) == 0;
      __builtin_amdgcn_raw_buffer_store_b8((uint8_t)byte, ys,
                                           first ? row * sr + n0 / kMxBlock : kDmaOutOfRange, 0, 0);
    }
  }
};

// ------------------------------------------------------------------------- few rows
// Weights straight from memory into registers: a workgroup's 4 waves take 16 NT rows of an expert and
// 32 features each (KS == 1), or the same 32 features and a quarter of K each (KS == 4).
template <typename T, int NT, int KS, bool QUANT>
__global__ __launch_bounds__(256) void mx_stream_kernel(MxGemmArgs a) {
  constexpr int kWaves = 4, kCols = 32 * (kWaves / KS);
  __shared__ int s_sum[2 * kWaves], s_out[4];
  __shared__ float part[KS > 1 ? (KS - 1) * NT * 8 * kWave : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowTiles<16 * NT, kOneHeight, kWaves> tiles;
  tiles.scan(a.seg_off, a.n_expert, s_sum);
  const int n_pad = QUANT ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const int n_cols = (n_pad + kCols - 1) / kCols;
  if (tiles.rows_f == 0) return;
  const int col = blockIdx.x / tiles.rows_f, v = blockIdx.x - col * tiles.rows_f;
  if (col >= n_cols) return;
  const TileRows t = tiles.find(a.seg_off, v, false, s_out);

  const int m = lane & 15, g = lane >> 4;
  const int base = col * kCols + (KS == 1 ? wave * 32 : 0);
  const int64_t code_row = mx_code_bytes(a.in_feat), scale_row = mx_scale_bytes(a.in_feat);
  // rows and features past the end repeat the last one; their results are not stored
  const uint8_t *wc[2], *ws[2], *xc[NT], *xs[NT];
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const int64_t n = (int64_t)t.e * a.out_feat + min(base + mx_feature(f, m), a.out_feat - 1);
    wc[f] = a.wc + n * code_row + g * 16;
    ws[f] = a.ws + n * scale_row;
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int64_t r = t.row0 + min(t.m0 + i * 16 + m, t.cnt - 1);
    xc[i] = a.xc + r * code_row + g * 16;
    xs[i] = a.xs + r * scale_row;
  }
  const int steps = (a.in_feat + kMxStep - 1) / kMxStep, groups = (steps + 3) / 4;
  const int g0 = KS == 1 ? 0 : wave * groups / KS, g1 = KS == 1 ? groups : (wave + 1) * groups / KS;
  f32x4 acc[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int q = g0; q < g1; ++q) {
    i32x4 wsv[2], xsv[NT];
#pragma unroll
    for (int f = 0; f < 2; ++f) wsv[f] = *(const i32x4*)(ws[f] + q * 16);
#pragma unroll
    for (int i = 0; i < NT; ++i) xsv[i] = *(const i32x4*)(xs[i] + q * 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (q * 4 + s >= steps) break;
      const int64_t off = (int64_t)(q * 4 + s) * 64;
      i32x4 w[2], x[NT];
#pragma unroll
      for (int f = 0; f < 2; ++f) w[f] = *(const i32x4*)(wc[f] + off);
#pragma unroll
      for (int i = 0; i < NT; ++i) x[i] = *(const i32x4*)(xc[i] + off);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int f = 0; f < 2; ++f)
          acc[i][f] = mx_mfma(w[f], (int)((uint32_t)wsv[f][s] >> (8 * g)), x[i],
                              (int)((uint32_t)xsv[i][s] >> (8 * g)), acc[i][f]);
    }
  }
  if (KS > 1) {
    // the quarters meet in the first wave, always in the same order
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          part[(((wave - 1) * NT + i) * 8 + j) * kWave + lane] = acc[i][j >> 2][j & 3];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w2 = 0; w2 < KS - 1; ++w2)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[i][j >> 2][j & 3] += part[((w2 * NT + i) * 8 + j) * kWave + lane];
  }
  const MxOutput<T, QUANT> out(a, t.e, (int64_t)t.row0 + t.m0, min(16 * NT, t.cnt - t.m0));
  float bias[8];
  out.load_bias(base + 8 * g, bias);
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = acc[i][j >> 2][j & 3] + bias[j];
    out.store(i * 16 + m, base + 8 * g, r);
  }
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
// copies of the stage after next follow, dealt out over the rest of both steps.  In the middle of
// the second step a wait and a barrier publish the next stage, whose first fragments are read in
// the shadow of the remaining instructions.
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
// The 18 wait states between the last matrix instruction and a read of its result.
__device__ __forceinline__ void mx_mfma_done() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

template <int TN, int TM> struct MxTile {
  static constexpr int kRows = TN + TM;
  static constexpr int kStageBytes = kRows * 128;
  static constexpr int kLoadsW = TN / 32, kLoadsX = TM / 32;       // copies of a wave per stage
  static constexpr int kLoads = kLoadsW + kLoadsX;
  static constexpr int kScaleLoads = 2;                            // and per group of scales
  static constexpr int kScaleBytes = 8192;                         // 4 KiB for either operand
  static constexpr int kLdsBytes = 2 * (kStageBytes + kScaleBytes);
  static constexpr int kGroups = kLdsBytes > 81920 ? 1 : 2;        // workgroups on a CU
  static_assert(TN % 64 == 0 && TM % 64 == 0 && TN <= 256 && TM <= 256, "even copies per wave");
};

template <typename T, int TN, int TM, bool QUANT>
__global__ __launch_bounds__(256, (MxTile<TN, TM>::kGroups)) void mx_tile_kernel(MxGemmArgs a) {
  using S = MxTile<TN, TM>;
  constexpr int FW = TN / 32, TW = TM / 32;         // fragments of a wave
  constexpr int kMma = FW * TW;
  extern __shared__ __align__(16) char lds[];
  __shared__ int s_sum[8], s_out[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  RowTiles<TM, kOneHeight, 4> tiles;
  tiles.scan(a.seg_off, a.n_expert, s_sum);
  const int n_pad = QUANT ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const int n_cols = (n_pad + TN - 1) / TN, live = tiles.rows_f * n_cols;
  const int number = tile_number(blockIdx.x, live);
  if (number >= live) return;
  int v, col;
  tile_order(number, tiles.rows_f, n_cols, v, col);
  const TileRows t = tiles.find(a.seg_off, v, false, s_out);

  const int code_row = (int)mx_code_bytes(a.in_feat), scale_row = (int)mx_scale_bytes(a.in_feat);
  const int base = col * TN;                        // (below out_feat: columns end on 128)
  const int steps = __builtin_amdgcn_readfirstlane((a.in_feat + kMxStep - 1) / kMxStep);
  const int stages = (steps + 1) / 2;
  const int64_t w0 = (int64_t)t.e * a.out_feat + base, x0 = (int64_t)t.row0 + t.m0;
  const int w_rows = min(TN, a.out_feat - base), x_rows = min(TM, t.cnt - t.m0);
  // every descriptor ends with its last valid row: rows past the end read as zeros
  const i32x4 w_rsrc = mx_descriptor(a.wc + w0 * code_row, (int64_t)w_rows * code_row);
  const i32x4 x_rsrc = mx_descriptor(a.xc + x0 * code_row, (int64_t)x_rows * code_row);
  const i32x4 ws_rsrc = mx_descriptor(a.ws + w0 * scale_row, (int64_t)w_rows * scale_row);
  const i32x4 xs_rsrc = mx_descriptor(a.xs + x0 * scale_row, (int64_t)x_rows * scale_row);
  // A lane's part of the offset of a copy, by the parity of the KiB (8 rows of a fragment's 16):
  // its row within the 8 and its pack.  Rows of a fragment are features 8 (m / 4) + m % 4 of 32.
  uint32_t w_lane[2], x_lane[2];
  const int r8 = lane >> 3;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int pack = (lane & 7) ^ ((4 * p + (r8 >> 1)) & 7);
    w_lane[p] = (uint32_t)((8 * (r8 >> 2) + (r8 & 3)) * code_row + pack * 16);
    x_lane[p] = (uint32_t)(r8 * code_row + pack * 16);
  }
  uint32_t ws_lane = (uint32_t)(((lane & 32) + mx_feature((lane >> 4) & 1, lane & 15)) * scale_row);
  uint32_t xs_lane = (uint32_t)(lane * scale_row);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)lds;
  auto dma = [&](uint32_t dst, uint32_t offset, i32x4 rsrc) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(offset), "s"(rsrc)
                 : "memory", "m0");
  };
  // Copy i of stage `st` into the buffer of its parity: every wave has its share of either
  // operand, so that nothing here depends on the wave but numbers.
  auto copy = [&](auto ic, int st) {
    constexpr int i = decltype(ic)::value;
    const uint32_t buf = lds0 + (st & 1) * S::kStageBytes;
    if constexpr (i < S::kLoadsW) {
      constexpr int in4 = 16 * (i & 1) + 4 * ((i >> 1) & 1);
      const int kib = wave * S::kLoadsW + i;
      const int row = S::kLoadsW % 4 ? 32 * (kib >> 2) + 16 * (kib & 1) + 4 * ((kib >> 1) & 1)
                                     : wave * (TN / 4) + 32 * (i >> 2) + in4;
      dma(buf + kib * 1024, w_lane[i & 1] + (uint32_t)(row * code_row + st * 128), w_rsrc);
    } else {
      const int kib = wave * S::kLoadsX + i - S::kLoadsW;
      dma(buf + TN * 128 + kib * 1024,
          x_lane[(i - S::kLoadsW) & 1] + (uint32_t)(kib * 8 * code_row + st * 128), x_rsrc);
    }
  };
  // The scales of 64 rows of either operand (past the tile: zeros).
  auto copy_scales = [&](int i, int group) {
    const uint32_t dst = lds0 + 2 * S::kStageBytes + (group & 1) * S::kScaleBytes + i * 4096 + wave * 1024;
    const uint32_t off = (uint32_t)(wave * 64 * scale_row + group * 16);
    if (i == 0) dma(dst, ws_lane + off, ws_rsrc);
    else dma(dst, xs_lane + off, xs_rsrc);
  };
  // Before the copies of stage `st`: past the end of K nothing is read any more, and of a last
  // stage of one step only the first four packs of a row.
  auto bound = [&](int st) {
    const bool past = st >= stages, half = st * 2 + 1 >= steps;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int pack = (lane & 7) ^ ((4 * p + (r8 >> 1)) & 7);
      const bool off = past | (half & (pack >= 4));
      w_lane[p] = off ? kDmaOutOfRange : w_lane[p];
      x_lane[p] = off ? kDmaOutOfRange : x_lane[p];
    }
    ws_lane = past ? kDmaOutOfRange : ws_lane;
    xs_lane = past ? kDmaOutOfRange : xs_lane;
  };

  const int m = lane & 15, g = lane >> 4, wn = wave >> 1, wm = wave & 1;
  const int frag0 = m * 128 + (g ^ ((m >> 1) & 7)) * 16;      // step 0; step 1 has packs 4..7
  const char* const w_lds = lds + wn * (TN / 2) * 128;
  const char* const x_lds = lds + (TN + wm * (TM / 2)) * 128;
  i32x4 wf[2][FW], xf[2][TW];
  int wsc[FW], xsc[TW];            // per fragment, this lane's bytes of the group's 4 steps
  int wsn[FW], xsn[TW];            // the next group's
  // fragment j (features first) of step S of the stage in buffer `buf`
  auto read = [&](auto jc, auto step, int buf) {
    constexpr int j = decltype(jc)::value, s = decltype(step)::value;
    const int at = buf * S::kStageBytes + (s ? frag0 ^ 64 : frag0);
    if constexpr (j < FW) wf[s][j] = *(const i32x4*)(w_lds + at + j * 2048);
    else xf[s][j - FW] = *(const i32x4*)(x_lds + at + (j - FW) * 2048);
  };
  // byte g of each of a row's four words (the steps of a group)
  const uint32_t pick = (uint32_t)g | (uint32_t)(4 + g) << 8 | 0x0c0c0000u;
  const uint32_t last_mask = (steps & 3) ? (1u << (8 * (steps & 3))) - 1 : ~0u;
  auto read_scale = [&](auto jc, int group) {
    constexpr int j = decltype(jc)::value;
    const int row = j < FW ? wn * (TN / 2) + j * 16 : 256 + wm * (TM / 2) + (j - FW) * 16;
    const i32x4 b = *(const i32x4*)(lds + 2 * S::kStageBytes + (group & 1) * S::kScaleBytes +
                                    (row + m) * 16);
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t)b[1], (uint32_t)b[0], pick);
    const uint32_t hi = __builtin_amdgcn_perm((uint32_t)b[3], (uint32_t)b[2], pick);
    // bytes behind the last step of K may hold anything, and 255 would make a NaN of a zero
    const int all = (int)(__builtin_amdgcn_perm(hi, lo, 0x05040100u) &
                          (group * 4 + 4 <= steps ? ~0u : last_mask));
    if constexpr (j < FW) wsn[j] = all;
    else xsn[j - FW] = all;
  };
  f32x4 acc[TW][FW];
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int f = 0; f < FW; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};

  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
  auto next_scales = [&] {
#pragma unroll
    for (int j = 0; j < FW; ++j) wsc[j] = wsn[j];
#pragma unroll
    for (int j = 0; j < TW; ++j) xsc[j] = xsn[j];
  };
  bound(0);
#pragma unroll
  for (int i = 0; i < S::kScaleLoads; ++i) copy_scales(i, 0);
  unroll<0, S::kLoads>([&](auto i) { copy(i, 0); });
  bound(1);
  unroll<0, S::kLoads>([&](auto i) { copy(i, 1); });
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoads) : "memory");
  __builtin_amdgcn_s_barrier();
  unroll<0, FW + TW>([&](auto j) { read(j, C0{}, 0); });
  unroll<0, FW + TW>([&](auto j) { read_scale(j, 0); });
  next_scales();

  // Where things happen among the 2 * kMma instructions of a stage: the second step's fragments
  // are read behind the first ones, the buffer is released behind kRelease, the next stage is
  // published behind kPublish and its first fragments (and the next group's scales) are read.
  constexpr int kReads = FW + TW;
  constexpr int kWindow = kReads < kMma / 2 ? kReads : kMma / 2;
  constexpr int kRelease = kWindow + kMma / 8;
  constexpr int kPublish = kMma + kMma / 4;
  static_assert(kRelease < kMma && kPublish + kWindow + kWindow / 2 < 2 * kMma, "room for the reads");
  auto one_stage = [&](auto odd_c, int st) {
    constexpr int odd = decltype(odd_c)::value;
    constexpr int kCopies = S::kLoads + (odd ? 0 : S::kScaleLoads);
    // of `count` things dealt over the instructions from .. from + len - 1, those out behind k
    constexpr auto dealt = [](int k, int from, int len, int count) {
      const int n = k < from ? 0 : (k - from + 1) * count / len;
      return n < count ? n : count;
    };
    constexpr auto copied = [dealt](int k) {
      return dealt(k, kRelease + 1, 2 * kMma - kRelease - 1, kCopies);
    };
    auto issue = [&](auto kc) {
      constexpr int k = decltype(kc)::value;
      unroll<copied(k - 1), copied(k)>([&](auto c) {
        constexpr int i = decltype(c)::value;
        if constexpr (i < S::kLoads) copy(c, st + 2);
        else copy_scales(i - S::kLoads, (st + 2) >> 1);
      });
    };
    bound(st + 2);
    unroll<0, kMma>([&](auto kc) {
      constexpr int k = decltype(kc)::value, i = k / FW, f = k % FW;
      mx_mfma_at<2 * odd>(wf[0][f], wsc[f], xf[0][i], xsc[i], acc[i][f]);
      unroll<dealt(k - 1, 0, kWindow, kReads), dealt(k, 0, kWindow, kReads)>(
          [&](auto j) { read(j, C1{}, st & 1); });
      if constexpr (k == kRelease) {
        __builtin_amdgcn_s_waitcnt(0xc07f);           // lgkmcnt(0): my reads of this stage are done
        __builtin_amdgcn_s_barrier();
      }
      issue(kc);
      __builtin_amdgcn_sched_barrier(0);
    });
    unroll<kMma, 2 * kMma>([&](auto kc) {
      constexpr int k = decltype(kc)::value, i = (k - kMma) / FW, f = (k - kMma) % FW;
      mx_mfma_at<2 * odd + 1>(wf[1][f], wsc[f], xf[1][i], xsc[i], acc[i][f]);
      if constexpr (k == kPublish) {
        static_assert(copied(kPublish - 1) < 64, "vmcnt is a 6-bit counter");
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(copied(kPublish - 1)) : "memory");
        __builtin_amdgcn_s_barrier();
      }
      constexpr int r0 = kPublish + 1, r1 = r0 + kWindow / 2;
      unroll<dealt(k - 1, r0, kWindow, kReads), dealt(k, r0, kWindow, kReads)>(
          [&](auto j) { read(j, C0{}, (st + 1) & 1); });
      if constexpr (odd)
        unroll<dealt(k - 1, r1, kWindow, kReads), dealt(k, r1, kWindow, kReads)>(
            [&](auto j) { read_scale(j, (st + 1) >> 1); });
      issue(kc);
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (odd) next_scales();
  };
  // (the last group's missing steps, if any, multiply zeros)
  const int groups = (steps + 3) >> 2;
  for (int q = 0; q < groups; ++q) {
    one_stage(C0{}, 2 * q);
    one_stage(C1{}, 2 * q + 1);
  }
  mx_mfma_done();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing may land in LDS after the end

  const MxOutput<T, QUANT> out(a, t.e, x0, x_rows);
#pragma unroll
  for (int p = 0; p < FW / 2; ++p) {
    const int n0 = base + wn * (TN / 2) + p * 32 + 8 * g;
    float bias[8];
    out.load_bias(n0, bias);
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      float r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = acc[i][2 * p + (j >> 2)][j & 3] + bias[j];
      out.store(wm * (TM / 2) + i * 16 + m, n0, r);
    }
  }
}

template <typename T, bool QUANT>
static int launch(const MxGemmArgs& a, hipStream_t s) {
  const int n_pad = QUANT ? (int)mx_code_bytes(a.out_feat) * 2 : a.out_feat;
  const double mean = (double)a.n_rows / a.n_expert;
#define FMOE_CALL(NT, KS)                                                                        \
  do {                                                                                           \
    const int64_t rows = a.n_rows / (16 * NT) + std::min<int64_t>(a.n_expert, a.n_rows);         \
    const int64_t blocks = rows * ceil_div(n_pad, 32 * (4 / KS));                                \
    FMOE_REQUIRE(blocks <= INT32_MAX, FMOE_ERR_UNSUPPORTED, "mx_linear: too many tiles");        \
    hipLaunchKernelGGL((mx_stream_kernel<T, NT, KS, QUANT>), dim3((unsigned)blocks), dim3(256), 0, \
                       s, a);                                                                    \
  } while (0)
#define FMOE_TILE(TN, TM)                                                                        \
  do {                                                                                           \
    const int64_t rows = a.n_rows / TM + std::min<int64_t>(a.n_expert, a.n_rows);                \
    const int64_t blocks = (rows * ceil_div(n_pad, TN) + 255) / 256 * 256;                       \
    FMOE_REQUIRE(blocks <= INT32_MAX, FMOE_ERR_UNSUPPORTED, "mx_linear: too many tiles");        \
    FMOE_SET_DYNAMIC_LDS_ONCE((mx_tile_kernel<T, TN, TM, QUANT>), (MxTile<TN, TM>::kLdsBytes));  \
    hipLaunchKernelGGL((mx_tile_kernel<T, TN, TM, QUANT>), dim3((unsigned)blocks), dim3(256),    \
                       (MxTile<TN, TM>::kLdsBytes), s, a);                                       \
  } while (0)
  if (mean >= 128) FMOE_TILE(256, 256);
  else if (mean <= 16) FMOE_CALL(1, 4);
  else FMOE_CALL(4, 1);
#undef FMOE_CALL
#undef FMOE_TILE
  FMOE_LAUNCH_CHECK("mx_linear");
  return FMOE_OK;
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
                     (uint8_t*)y_scales, n_rows, (int)in_feat, (int)out_feat, (int)n_expert, act, dtype};
  hipStream_t s = (hipStream_t)stream;
  const bool q = y_codes != nullptr;
  switch (dtype) {
    case FMOE_F32: return q ? launch<float, true>(a, s) : launch<float, false>(a, s);
    case FMOE_F16: return q ? launch<__half, true>(a, s) : launch<__half, false>(a, s);
    default: return q ? launch<__hip_bfloat16, true>(a, s) : launch<__hip_bfloat16, false>(a, s);
  }
}
