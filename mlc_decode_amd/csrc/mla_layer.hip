// mla_layer.hip -- what stands between the attentions of consecutive layers in a decode step (gfx950): the residual's
// addition and the root-mean-square norm, to 16-bit rows or to 8-bit rows with scales, and projections of few rows by
// 4-bit weights.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string>
#include <type_traits>

#include "mla_decode_amd.h"
#include "mla_elem.h"
#include "mla_serving.h"

namespace mla_layer {

using mla_srv::Bf16;
using mla_srv::F16;
using mla_srv::F32;
using mla_srv::i32x2;
using mla_srv::i32x4;
using mla_srv::pack;
using mla_srv::unpack;

// ---------------------------------------------------------------------------------------
// root-mean-square norm
// ---------------------------------------------------------------------------------------
// h = x + r,  y = h / sqrt(mean(h^2) + eps) * w.  A row is read once and stays in the registers of its workgroup, as fp32;
// its squares are summed in fp32, by lane, wave and workgroup.  The norm is of h as it was added, in 32 bits; what is
// returned of h is rounded once, and so is y.  As 8 bits y is e4m3 codes with a power of two per 32 dims, the smallest
// that brings them to 448 at most, of y in 32 bits (one rounding); 4 lanes share a block of 32 where a lane holds 8.
//
// A piece is 16 bytes of x (8 values, 4 of fp32), or one value where rows, strides or dims do not fall on such pieces;
// thread t of a row holds pieces t, t + threads, ...  P of them.
// Bound by memory for many rows, by latency for few (row, sum, barrier): 1 x 7168 with the residual 2.9 us, 256 rows 4.1,
// 1024 rows 11.0 (5.3 TB/s), 8192 rows 96 (4.9; to 16 bits without a residual 42.7, 5.5), 65536 x 512 39 us, 65536 x 128 12.8 (in
// the last-level cache: 6.9 and 5.2).
struct NormParams {
  const uint8_t* x;
  const uint8_t* residual;  // may be NULL
  const uint8_t* weight;
  uint8_t* out;             // rows, or codes
  uint8_t* scale;           // of codes: [tokens, dim / 32] contiguous; NULL: rows
  uint8_t* residual_out;    // may be NULL
  int64_t x_st, r_st, o_st, ro_st;  // bytes
  int32_t tokens, dim;
  float eps, inv_dim;
  int32_t w_f32;  // weights in fp32, else as x
};

// The smallest k with amax <= 448 * 2^k, from the bits of amax (finite); 0 of zeros, at least -126.
__device__ __forceinline__ int block_exp8(uint32_t bits) {
  const float a = __uint_as_float(bits);
  const int e = __builtin_amdgcn_frexp_expf(a);  // a = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
  const int k = __builtin_amdgcn_frexp_mantf(a) <= 0.875f ? e - 9 : e - 8;
  return bits == 0 ? 0 : k < -126 ? -126 : k;
}

// What a thread holds of a row: P pieces of V values.
template <class E, int V>
__device__ __forceinline__ void load_piece(const uint8_t* src, int at, float* x) {
  if constexpr (V == 1)
    x[0] = E::value(*(const typename E::bits*)(src + (int64_t)at * E::kBytes));
  else
    unpack<E>(*(const i32x4*)(src + 16 * (int64_t)at), x);
}
template <class E, int V>
__device__ __forceinline__ void store_piece(uint8_t* dst, int at, const float* x) {
  if constexpr (V == 1)
    *(typename E::bits*)(dst + (int64_t)at * E::kBytes) = E::of(x[0]);
  else
    *(i32x4*)(dst + 16 * (int64_t)at) = pack<E>(x);
}
template <class E, int V>
__device__ __forceinline__ void load_weight(const NormParams& p, int at, float* w) {
  if (p.w_f32) {  // uniform
    if constexpr (V == 8) {
      load_piece<F32, 4>(p.weight, 2 * at, w);
      load_piece<F32, 4>(p.weight, 2 * at + 1, w + 4);
    } else {
      load_piece<F32, V>(p.weight, at, w);
    }
  } else {
    load_piece<E, V>(p.weight, at, w);
  }
}
// V values of y as codes; 32 / V consecutive lanes hold a block.
template <int V>
__device__ __forceinline__ void store_codes(const NormParams& p, int64_t row, int at, bool in, const float* y) {
  uint32_t top = 0;  // |y| as bits: ordered like the values, with infinities and NaNs at the end
  if (in)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t a = __float_as_uint(y[j]) & 0x7FFFFFFFu;
      top = top > a ? top : a;
    }
#pragma unroll
  for (int m = 1; m < 32 / V; m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)top, m);
    top = top > o ? top : o;
  }
  if (!in) return;
  const bool bad = top >= 0x7F800000u;
  const int k = bad ? 0 : block_exp8(top);
  const float down = __uint_as_float((uint32_t)(127 - k) << 23);  // 2^-k, k in -126 .. 120: exact products
  uint8_t* dst = p.out + row * p.o_st + (int64_t)at * V;
  if constexpr (V == 1) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * down, 0.f, 0, false);
    *dst = bad ? 0x7F : (uint8_t)w;
  } else {
    int w[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      w[j] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j] * down, y[4 * j + 1] * down, 0, false);
      w[j] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2] * down, y[4 * j + 3] * down, w[j], true);
      w[j] = bad ? 0x7F7F7F7F : w[j];
    }
    if constexpr (V == 8)
      *(i32x2*)dst = i32x2{w[0], w[1]};
    else
      *(int*)dst = w[0];
  }
  const int dim = at * V;
  if (dim % 32 == 0) p.scale[row * (p.dim / 32) + dim / 32] = bad ? 255 : (uint8_t)(k + 127);
}

// One row by T threads; 256 / T rows a workgroup where T < 256, 64 / T rows a wave where T < 64.
template <class E, int V, int T, int P>
__global__ __launch_bounds__(T < 256 ? 256 : T) void mla_rms_norm_kernel(NormParams p) {
  constexpr int kRows = T < 256 ? 256 / T : 1;
  constexpr int kWaves = T > 64 ? T / 64 : 1;
  __shared__ float sum_sh[kRows][kWaves];
  const int sub = T < 64 ? (int)threadIdx.x / T : kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : 0;
  const int t = kRows > 1 ? threadIdx.x % T : threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * kRows + sub;
  const bool on = row < p.tokens;  // uniform over a row's threads
  const int pieces = p.dim / V;
  const uint8_t* x = p.x + row * p.x_st;
  const uint8_t* r = p.residual + row * p.r_st;
  float h[P][V], w[P][V];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int at = t + i * T;
#pragma unroll
    for (int j = 0; j < V; ++j) h[i][j] = 0.f;
    if (on && at < pieces) load_piece<E, V>(x, at, h[i]);
  }
  if (p.residual != nullptr) {  // uniform
    float a[P][V];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int at = t + i * T;
#pragma unroll
      for (int j = 0; j < V; ++j) a[i][j] = 0.f;
      if (on && at < pieces) load_piece<E, V>(r, at, a[i]);
    }
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) h[i][j] += a[i][j];
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int at = t + i * T;
    if (at < pieces) load_weight<E, V>(p, at, w[i]);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) sum += h[i][j] * h[i][j];
#pragma unroll
  for (int d = T < 64 ? T / 2 : 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if constexpr (kWaves > 1) {
    if ((t & 63) == 0) sum_sh[sub][t >> 6] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum += sum_sh[sub][i];
  }
  if (!on) return;  // a row's threads together
  const float f = 1.f / sqrtf(sum * p.inv_dim + p.eps);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int at = t + i * T;
    const bool in = at < pieces;
    if (in && p.residual_out != nullptr) store_piece<E, V>(p.residual_out + row * p.ro_st, at, h[i]);
    float y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = h[i][j] * f * w[i][j];
    if (p.scale != nullptr)  // uniform
      store_codes<V>(p, row, at, in, y);
    else if (in)
      store_piece<E, V>(p.out + row * p.o_st, at, y);
  }
}

// Rows longer than a workgroup's registers hold: read a second time for the output.
template <class E, int V>
__global__ __launch_bounds__(1024) void mla_rms_norm_long_kernel(NormParams p) {
  __shared__ float sum_sh[16];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int pieces = p.dim / V;
  const uint8_t* x = p.x + row * p.x_st;
  const uint8_t* r = p.residual + row * p.r_st;
  auto load = [&](int at, float* h) __attribute__((always_inline)) {
    load_piece<E, V>(x, at, h);
    if (p.residual != nullptr) {  // uniform
      float a[V];
      load_piece<E, V>(r, at, a);
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] += a[j];
    }
  };
  float sum = 0.f;
  for (int at = t; at < pieces; at += 1024) {
    float h[V];
    load(at, h);
#pragma unroll
    for (int j = 0; j < V; ++j) sum += h[j] * h[j];
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((t & 63) == 0) sum_sh[t >> 6] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += sum_sh[i];
  const float f = 1.f / sqrtf(sum * p.inv_dim + p.eps);
  for (int base = 0; base < pieces; base += 1024) {  // uniform: whole waves share the blocks of codes
    const int at = base + t;
    const bool in = at < pieces;
    float h[V], w[V], y[V];
    if (in) {
      load(at, h);
      load_weight<E, V>(p, at, w);
      if (p.residual_out != nullptr) store_piece<E, V>(p.residual_out + row * p.ro_st, at, h);
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = h[j] * f * w[j];
    }
    if (p.scale != nullptr)  // uniform
      store_codes<V>(p, row, at, in, y);
    else if (in)
      store_piece<E, V>(p.out + row * p.o_st, at, y);
  }
}

template <class E, int V, int T, int P>
static void launch_norm_as(const NormParams& p, hipStream_t st) {
  constexpr int kRows = T < 256 ? 256 / T : 1;
  hipLaunchKernelGGL((mla_rms_norm_kernel<E, V, T, P>), dim3((p.tokens + kRows - 1) / kRows), dim3(T < 256 ? 256 : T), 0, st, p);
}
template <class E, int V>
static void launch_norm(const NormParams& p, int cus, hipStream_t st) {
  const int pieces = p.dim / V;
  // Short rows share a wave; us for a wave a row and so (bf16): 65536 x 64 14.2, 4.2    x 128 14.6, 6.3    x 256 18.1, 13.0
  if (pieces <= 8) return launch_norm_as<E, V, 8, 1>(p, st);
  if (pieces <= 16) return launch_norm_as<E, V, 16, 1>(p, st);
  if (pieces <= 32) return launch_norm_as<E, V, 32, 1>(p, st);
  if (pieces <= 64) return launch_norm_as<E, V, 64, 1>(p, st);
  if (pieces <= 128) return launch_norm_as<E, V, 64, 2>(p, st);
  if (pieces <= 256) return launch_norm_as<E, V, 256, 1>(p, st);
  if (pieces <= 512) return launch_norm_as<E, V, 256, 2>(p, st);
  // Few rows take threads, many rows workgroups that fit a CU in numbers; us for 1024 and 256 threads a row of 7168 with the
  // residual: 1 row 2.9, 4.2    128 3.5, 4.9    256 4.2, 5.5    512 5.8, 7.0    768 9.0, 9.0    1024 11.8, 11.0
  if (pieces <= 1024) {
    if (p.tokens <= 2 * cus) return launch_norm_as<E, V, 1024, 1>(p, st);
    return launch_norm_as<E, V, 256, 4>(p, st);
  }
  if (pieces <= 2048) return launch_norm_as<E, V, 1024, 2>(p, st);
  if (pieces <= 4096) return launch_norm_as<E, V, 1024, 4>(p, st);
  if constexpr (V == 1) {
    if (pieces <= 8192) return launch_norm_as<E, V, 1024, 8>(p, st);
  }
  hipLaunchKernelGGL((mla_rms_norm_long_kernel<E, V>), dim3(p.tokens), dim3(1024), 0, st, p);
}
template <class E>
static void launch_norm_type(const NormParams& p, bool vec, int cus, hipStream_t st) {
  if (vec)
    launch_norm<E, 16 / E::kBytes>(p, cus, st);
  else
    launch_norm<E, 1>(p, cus, st);
}

// ---------------------------------------------------------------------------------------
// projections by 4-bit weights
// ---------------------------------------------------------------------------------------
// y[t, n] = sum_k x[t, k] w[n, k], w[n, k] = e2m1(code) * 2^(s[n, k / 32] - 127), for few rows t: the weights are read
// once, 17 bits for 32 of them, and that is what bounds it.  They are laid out as the operand of the matrix unit: of
// 16 outputs x 128 inputs (a chunk), lane (g, i) holds inputs 32 g .. +31 of output i, 16 bytes; the scale bytes alike.
//   8 codes become 8 bf16 (exact) or fp16, four 16x16x32 MFMAs a chunk.  fp16 has no room for a scale's range: a row's
//     scales are taken relative to its largest, 2^11, and the output is multiplied back; what lies 2^-35 below the
//     largest of its row is lost there.
//   8-bit rows become bf16 rows on their way into LDS: e4m3 has 4 significant bits, so every value inside bf16's range is
//     exact.  The block-scaled 16x16x128 MFMA would take both sides' codes and scales as they are, but it adds its products
//     in groups of eight within about 13 bits below the largest: 448 * 6 less itself beside six products of 2^-8 gives 0.
//     Faster it is: 8 x 24576 x 1536 4.6 us against 6.0, 64 x 7168 x 16384 20.4 against 25.8.
// A lane of a result holds outputs 4 g .. +3 of row i.  Everything is summed in fp32.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((__vector_size__(8 * sizeof(__bf16))));
typedef _Float16 f16x8 __attribute__((__vector_size__(8 * sizeof(_Float16))));

enum { kRowsBf16 = 0, kRowsF16 = 1, kRowsFp8 = 2 };

struct LinearParams {
  const uint8_t* x;        // rows
  const uint8_t* x_scale;  // of 8-bit rows
  int64_t x_st, xs_st;     // bytes
  const uint8_t* codes;    // [tiles][chunks][64][16]
  const uint8_t* scale;    // [tiles][chunks][64]
  const uint8_t* top;      // [16 tiles] the largest scale byte of an output's weights
  uint8_t* y;
  int64_t y_st;            // bytes
  float* part;             // [splits][tokens][16 tiles] partial sums
  int32_t tokens, n, k, tiles, chunks, per_split;  // per_split: chunks of a split
  int32_t y_f16, y_vec;    // y_vec: rows of y take 8-byte stores
};

constexpr int kTileX = 16 * 256;  // 16 rows of a chunk in LDS, 16-bit values

// A piece of 16 bytes of a row's chunk in LDS (p of 16): its place in the 16 rows' chunk.  Blocks of 256 bytes hold what one
// lane group of an operand reads, MFMA p % 4, lane group p / 4 (inputs 32 g + 8 j), the rows' order in them turned by the
// piece, so that a write's pieces of a few rows and a lane group's read of 16 rows each go over all banks.  (Lane groups meet
// in some: conflicts are 25 to 39% of LDS's busy cycles with 16-bit rows, 47% with 8-bit ones.)
__device__ __forceinline__ int piece_place(int p, int row) { return (p & 3) * 1024 + (p >> 2) * 256 + ((row ^ p) << 4); }
// The operand of MFMA j for lane (g, i).
__device__ __forceinline__ i32x4 read_piece(const uint8_t* tile, int j, int g, int i) {
  return *(const i32x4*)(tile + piece_place(4 * g + j, i));
}

// Registers of the first LOADS * kEach rows of a 16-row chunk, by one wave, 16 bytes a lane and load.  Rows past the last are
// the last again: they are columns of the product that nothing reads.
template <int XT, int LOADS>
struct RowsChunk {
  i32x4 v[LOADS];
  int sc[XT == kRowsFp8 ? LOADS : 1];  // 8-bit rows: the scale byte of v's 16 codes
};
template <int XT>
constexpr int kPieces = XT == kRowsFp8 ? 8 : 16;  // of 16 bytes, of a row's chunk in memory
template <int XT>
constexpr int kEach = 64 / kPieces<XT>;  // rows of a load
template <int XT, int LOADS>
__device__ __forceinline__ void load_rows(const LinearParams& p, int first, int chunk, int lane, RowsChunk<XT, LOADS>& c) {
  const int piece = lane % kPieces<XT>;
  const int most = p.k / (XT == kRowsFp8 ? 16 : 8) - 1;  // the last piece of a row
  int at = chunk * kPieces<XT> + piece;
  at = at < most ? at : most;
  const uint8_t* src = p.x + 16 * (int64_t)at;
#pragma unroll
  for (int q = 0; q < LOADS; ++q) {
    int row = first + kEach<XT> * q + lane / kPieces<XT>;
    row = row < p.tokens ? row : p.tokens - 1;
    c.v[q] = *(const i32x4*)(src + row * p.x_st);
    if constexpr (XT == kRowsFp8) c.sc[q] = p.x_scale[row * p.xs_st + at / 2];
  }
}
// To LDS.  Pieces past the row's end are zeros (their weights are, but an infinity times 0 is a NaN).
template <int XT, int LOADS>
__device__ __forceinline__ void put_rows(const LinearParams& p, uint8_t* tile, int chunk, int lane, RowsChunk<XT, LOADS>& c) {
  const int piece = lane % kPieces<XT>;
  const bool past = chunk * 128 + piece * (XT == kRowsFp8 ? 16 : 8) >= p.k;
  if (chunk * 128 + 128 > p.k)  // uniform
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      if (past) c.v[q] = i32x4{0, 0, 0, 0};
      if (XT == kRowsFp8 && past) c.sc[q] = 127;
    }
#pragma unroll
  for (int q = 0; q < LOADS; ++q) {
    const int row = kEach<XT> * q + lane / kPieces<XT>;
    if constexpr (XT == kRowsFp8) {
      const float sc = __uint_as_float((uint32_t)c.sc[q] << 23);  // the conversion takes its exponent alone
      const int nan = c.sc[q] == 255 ? 0x7F7F7F7F : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int a = c.v[q][2 * h] | nan, b = c.v[q][2 * h + 1] | nan;
        *(i32x4*)(tile + piece_place(2 * piece + h, row)) =
            i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, false)),
                  __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, true)),
                  __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, false)),
                  __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, true))};
      }
    } else {
      *(i32x4*)(tile + piece_place(piece, row)) = c.v[q];
    }
  }
}

struct WeightChunk {
  i32x4 codes;
  int sc;
};
__device__ __forceinline__ void load_weights(const LinearParams& p, int64_t tile, int chunk, int lane, WeightChunk& w) {
  const int64_t at = (tile * p.chunks + chunk) * 64 + lane;
  w.codes = *(const i32x4*)(p.codes + at * 16);
  w.sc = p.scale[at];
}
// The weights of one chunk as operands.
struct Operand {
  i32x4 a[4];
};
template <int XT>
__device__ __forceinline__ void widen(const WeightChunk& w, int up, Operand& o) {
  if constexpr (XT != kRowsF16) {
    const float sc = __uint_as_float((uint32_t)w.sc << 23);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = w.codes[j];
      o.a[j] = i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3))};
    }
  } else {
    // up = 138 - the row's largest byte: that one becomes 2^11; 255 stays (a NaN).  Inputs past the end, zeros of a scale
    // that has no part in that largest, stay zeros.
    const int to = w.sc + up < 254 ? w.sc + up : 254;
    const int e = w.sc == 255 ? 255 : to > 1 ? to : 1;
    const float sc = __uint_as_float((uint32_t)e << 23);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = w.codes[j];
      o.a[j] = i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 0)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 1)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 2)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 3))};
    }
  }
}
// acc[t] += the weights of tile t times 16 rows of a chunk, each operand of the rows read once.
template <int XT, int NT>
__device__ __forceinline__ void multiply(const Operand (&w)[NT], const uint8_t* tile, int g, int i, f32x4 (&acc)[NT]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const i32x4 b = read_piece(tile, j, g, i);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (XT == kRowsF16)
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w[t].a[j]), __builtin_bit_cast(f16x8, b), acc[t], 0, 0, 0);
      else
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[t].a[j]), __builtin_bit_cast(bf16x8, b), acc[t], 0, 0, 0);
    }
  }
}

// Four outputs n .. n + 3 of a row.
__device__ __forceinline__ void store_outputs(const LinearParams& p, int row, int n, f32x4 v) {
  if (row >= p.tokens || n >= p.n) return;
  uint16_t* dst = (uint16_t*)(p.y + row * p.y_st) + n;
  float x[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
  const i32x4 w = p.y_f16 ? pack<F16>(x) : pack<Bf16>(x);
  if (p.y_vec && n + 4 <= p.n) {
    *(i32x2*)dst = i32x2{w[0], w[1]};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.n) dst[j] = (uint16_t)((uint32_t)w[j >> 1] >> (16 * (j & 1)));
  }
}
// fp16 rows: back from the scales that the products were made with.
template <int XT>
__device__ __forceinline__ f32x4 scale_back(const LinearParams& p, int n, f32x4 v) {
  if constexpr (XT == kRowsF16)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __builtin_ldexpf(v[j], (int)p.top[n + j] - 138);
  return v;
}

// 16 rows (the first LOADS * kEach of them).  A wave takes 16 outputs and every WK-th chunk, its rows through LDS of its own (no
// barrier in the loop), weights and rows kDepth chunks ahead; the waves of a tile add up through LDS, in order.
// us where the weights are in the last-level cache (the same ones again and again), and where they come from memory (others
// in turns, as a model's layers are): 1 x 7168 x 16384 12.1, 14.5 (4.3 TB/s: bound by the weights)    16 x 7168 x 16384 17.6,
// 25.1 (2.5)    8 x 24576 x 1536 (8-bit rows) 5.7, 8.0 (2.5)    1 x 576 x 7168 3.8, 5.3, a load's latency over and over.
// Where rows are several, the waves wait for LDS and loads in turn: of the CU's cycles LDS is busy 38 to 47%, the matrix
// units 9 to 18%.
template <int XT, int LOADS, int WK>
__global__ __launch_bounds__(64 * WK) void mla_linear_few_kernel(LinearParams p) {
  constexpr int kDepth = LOADS == 4 && WK >= 8 ? 2 : 4;  // 128 registers: two workgroups of 8 waves a CU
  __shared__ __attribute__((aligned(16))) uint8_t x_sh[WK][2][kTileX];
  __shared__ f32x4 sum_sh[WK][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, i = lane & 15;
  const int64_t tile = blockIdx.x;
  const int first = 16 * blockIdx.y;
  WeightChunk w[kDepth];
  RowsChunk<XT, LOADS> x[kDepth];
  auto fetch = [&](int c, int s) __attribute__((always_inline)) {
    if (c < p.chunks) {  // uniform
      load_weights(p, tile, c, lane, w[s]);
      load_rows<XT, LOADS>(p, first, c, lane, x[s]);
    }
  };
#pragma unroll
  for (int s = 0; s < kDepth; ++s) fetch(wave + s * WK, s);
  const int up = XT == kRowsF16 ? 138 - (int)p.top[tile * 16 + i] : 0;
  f32x4 acc[2][1] = {{{0.f, 0.f, 0.f, 0.f}}, {{0.f, 0.f, 0.f, 0.f}}};
  for (int c0 = wave; c0 < p.chunks; c0 += kDepth * WK) {
#pragma unroll
    for (int s = 0; s < kDepth; ++s) {
      const int c = c0 + s * WK;
      if (c < p.chunks) {  // uniform
        uint8_t* xt = x_sh[wave][s & 1];
        Operand o[1];
        put_rows<XT, LOADS>(p, xt, c, lane, x[s]);
        widen<XT>(w[s], up, o[0]);
        fetch(c + kDepth * WK, s);
        __builtin_amdgcn_wave_barrier();  // the wave's own rows: LDS runs its accesses in order
        multiply<XT, 1>(o, xt, g, i, acc[s & 1]);
      }
    }
  }
  f32x4 sum = acc[0][0] + acc[1][0];
  sum_sh[wave][lane] = sum;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int k = 1; k < WK; ++k) sum += sum_sh[k][lane];
  const int n = (int)tile * 16 + 4 * g;
  store_outputs(p, first + i, n, scale_back<XT>(p, n, sum));
}

// More rows: a workgroup takes 128 outputs for 16 RT rows and a split of the chunks.  Its two halves take the steps of two
// chunks in turns, each with its own rows in LDS, a wave 32 outputs, the next step's on the way meanwhile; the halves
// add up through LDS.  64 x 7168 x 16384 (bf16, 62 MB of weights) 25 us with the splits' sums, 27 where the weights come from
// memory; in a trace, which runs one kernel after the other, 24 and 4 of sums.  Of the CU's cycles the matrix units are busy
// 37% and LDS 47% (two fifths of that bank conflicts); the waves wait 35% of theirs and queue to issue 38%: no unit is
// full, and two waves a SIMD do not cover each other.  Two workgroups of one half each and twice the splits: 27.9 us in all
// against 27.2, 16384 x 2048 15.0 against 12.7; one workgroup of 256 outputs 27.8, that with twice as much on the way 30.8.
template <int XT, int RT>
__global__ __launch_bounds__(512, 1) void mla_linear_rows_kernel(LinearParams p) {
  constexpr int kStep = 2, NT = 2;
  constexpr int kParts = kStep * RT;           // 16-row chunks of a step
  constexpr int kMine = (kParts + 3) / 4;      // of a wave
  __shared__ __attribute__((aligned(16))) uint8_t rows_sh[2][2][kParts][kTileX];
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3), lane = threadIdx.x & 63;
  auto& x_sh = rows_sh[half];
  const int g = lane >> 4, i = lane & 15;
  const int first = blockIdx.z * 16 * RT;
  const int c_begin = blockIdx.y * p.per_split;
  const int c_end = c_begin + p.per_split < p.chunks ? c_begin + p.per_split : p.chunks;
  int64_t tile[NT];
  int up[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t at = (int64_t)blockIdx.x * 8 + 2 * wave + t;
    tile[t] = at < p.tiles ? at : p.tiles - 1;  // past the end: the last one again, not stored
    up[t] = XT == kRowsF16 ? 138 - (int)p.top[tile[t] * 16 + i] : 0;
  }
  constexpr int kLoads = 16 / kEach<XT>;
  RowsChunk<XT, kLoads> x[kMine];
  WeightChunk w[2][kStep][NT];
  auto fetch_rows = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int part = 4 * m + wave, chunk = c + part / RT;  // uniform
      if (kParts % 4 == 0 || part < kParts) load_rows<XT, kLoads>(p, first + 16 * (part % RT), chunk < c_end ? chunk : c_end - 1, lane, x[m]);
    }
  };
  auto fetch_weights = [&](int c, WeightChunk (&v)[kStep][NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < kStep; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t) load_weights(p, tile[t], c + s < c_end ? c + s : c_end - 1, lane, v[s][t]);
  };
  f32x4 acc[RT][NT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int c_first = c_begin + half * kStep;  // steps in turns
  fetch_rows(c_first);
  fetch_weights(c_first, w[0]);
  auto step = [&](int c, int b, WeightChunk (&now)[kStep][NT], WeightChunk (&next)[kStep][NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int part = 4 * m + wave;
      if (kParts % 4 == 0 || part < kParts) put_rows<XT, kLoads>(p, x_sh[b][part], c + part / RT, lane, x[m]);
    }
    if (c + 2 * kStep < c_end) {  // uniform
      fetch_rows(c + 2 * kStep);
      fetch_weights(c + 2 * kStep, next);
    }
    __syncthreads();  // a buffer is written again two steps on, behind the next step's barrier
#pragma unroll
    for (int s = 0; s < kStep; ++s) {
      if (c + s >= c_end) break;  // uniform
      Operand o[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) widen<XT>(now[s][t], up[t], o[t]);
#pragma unroll
      for (int r = 0; r < RT; ++r)
        multiply<XT, NT>(o, x_sh[b][s * RT + r], g, i, acc[r]);
    }
  };
  for (int c = c_first; c - half * kStep < c_end; c += 4 * kStep) {  // as often for both halves
    step(c, 0, w[0], w[1]);
    if (c - half * kStep + 2 * kStep < c_end) step(c + 2 * kStep, 1, w[1], w[0]);  // uniform
  }
  // the halves' sums, in order
  f32x4* sum_sh = (f32x4*)&rows_sh[0][0][0][0];
  __syncthreads();
  if (half == 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t) sum_sh[((wave * RT + r) * NT + t) * 64 + lane] = acc[r][t];
  }
  __syncthreads();
  if (half == 1) return;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] += sum_sh[((wave * RT + r) * NT + t) * 64 + lane];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if ((int64_t)blockIdx.x * 8 + 2 * wave + t >= p.tiles) continue;
    const int n = (int)tile[t] * 16 + 4 * g;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = first + 16 * r + i;
      const f32x4 v = scale_back<XT>(p, n, acc[r][t]);
      if (p.part != nullptr) {  // uniform
        if (row < p.tokens) *(f32x4*)(p.part + ((int64_t)blockIdx.y * p.tokens + row) * (16 * (int64_t)p.tiles) + n) = v;
      } else {
        store_outputs(p, row, n, v);
      }
    }
  }
}

// The splits' sums, in order.
__global__ __launch_bounds__(256) void mla_linear_sum_kernel(LinearParams p, int splits) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int quads = 4 * p.tiles;
  const int row = (int)(at / quads), n = (int)(at % quads) * 4;
  if (row >= p.tokens) return;
  const int64_t stride = (int64_t)p.tokens * 16 * p.tiles;
  const float* src = p.part + (int64_t)row * 16 * p.tiles + n;
  f32x4 acc = *(const f32x4*)src;
  for (int s = 1; s < splits; ++s) acc += *(const f32x4*)(src + s * stride);
  store_outputs(p, row, n, acc);
}

// Whether every 16 rows go by themselves: up to 16 rows, and more where the work is small, where a launch for the splits'
// sums costs more than reading the weights from L2 for each 16.  us by themselves, and together (bf16, rows x n x k):
//   17 x 576 x 7168 5.3, 9.6    64 x 2048 x 2048 4.4, 10.8    100 x 512 x 16384 10.3, 15.8    32 x 4096 x 4096 6.6, 10.3
//   64 x 4096 x 4096 11.9, 14.4    32 x 8192 x 4096 11.6, 11.5    32 x 7168 x 7168 16.7, 12.5    20 x 16384 x 2048 11.1, 8.3
//   32 x 12288 x 512 4.5, 4.1    64 x 8192 x 1024 7.0, 7.5
static bool linear_few(int64_t tokens, int64_t tiles, int64_t chunks, int cus) {
  const int64_t all = (tokens + 15) / 16 * tiles;
  return tokens <= 16 || (all <= 4 * (int64_t)cus && all * chunks <= 128 * (int64_t)cus);
}

// Splits of the chunks where rows go together: as many workgroups as CUs, but twelve chunks each at least, below which the
// splits' sums cost more than the CUs give.  us for 1, 2, 3, 4, 6 splits (bf16, rows x n x k; a workgroup is 128 outputs):
//   64 x 7168 x 16384 63.4, 38.2, 30.7, 27.2, 34.2    64 x 7168 x 7168 30.7, 21.1, 18.5, 17.0, 23.2    256 x 4096 x 4096 19.8,
//   19.2, 24.4    64 x 16384 x 2048 12.7, 14.9    64 x 8192 x 1024 7.3, 9.3    64 x 24576 x 1536 11.8, 20.0
static int linear_splits(int64_t tokens, int64_t tiles, int64_t chunks, int cus) {
  if (linear_few(tokens, tiles, chunks, cus)) return 1;
  const int rt = tokens <= 32 ? 2 : 4;
  const int64_t groups = (tiles + 7) / 8 * ((tokens + 16 * rt - 1) / (16 * rt));
  const int64_t s = cus / groups < chunks / 12 ? cus / groups : chunks / 12;
  return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

// Waves that share a tile of 16 outputs; us for 4, 8, 16 of them (one bf16 row unless said):
//   n x k  576 x 7168 5.0, 4.0, 4.0    2048 x 16384 13.2, 8.2, 6.7    4096 x 2048 3.0, 2.9, 3.1    8192 x 8192 9.3, 8.6, 10.1
//   7168 x 16384 15.0, 12.3, 14.6 (16 rows 18.9, 17.8, 19.2)    12288 x 4096 (8 rows) 8.2, 8.3, 10.3    24576 x 1536 6.8, 7.6, 11.5
//   32768 x 7168 25.9, 27.9, 33.2
template <int XT, int LOADS>
static void launch_few(const LinearParams& p, int cus, hipStream_t st) {
  const dim3 grid(p.tiles, (p.tokens + 15) / 16);
  const int64_t all = (int64_t)p.tiles * grid.y;
  if (2 * all > 5 * (int64_t)cus)
    hipLaunchKernelGGL((mla_linear_few_kernel<XT, LOADS, 4>), grid, dim3(256), 0, st, p);
  else if (2 * all <= cus && p.chunks >= 96)
    hipLaunchKernelGGL((mla_linear_few_kernel<XT, LOADS, 16>), grid, dim3(1024), 0, st, p);
  else
    hipLaunchKernelGGL((mla_linear_few_kernel<XT, LOADS, 8>), grid, dim3(512), 0, st, p);
}

template <int XT>
static void launch_linear(LinearParams p, int splits, int cus, hipStream_t st) {
  if (linear_few(p.tokens, p.tiles, p.chunks, cus)) {
    constexpr int kFew = kEach<XT>;  // rows of one load
    if (p.tokens <= kFew) return launch_few<XT, 1>(p, cus, st);
    if (p.tokens <= 2 * kFew || 2 * kFew == 16) return launch_few<XT, 2>(p, cus, st);
    if constexpr (4 * kFew <= 16) return launch_few<XT, 4>(p, cus, st);
  }
  // whole steps of two chunks for both halves, so that the last split is the short one
  p.per_split = ((p.chunks + splits - 1) / splits + 3) / 4 * 4;
  splits = (p.chunks + p.per_split - 1) / p.per_split;
  if (splits == 1) p.part = nullptr;
  const int rt = p.tokens <= 32 ? 2 : 4;
  const dim3 grid((p.tiles + 7) / 8, splits, (p.tokens + 16 * rt - 1) / (16 * rt));
  if (rt == 2)
    hipLaunchKernelGGL((mla_linear_rows_kernel<XT, 2>), grid, dim3(512), 0, st, p);
  else
    hipLaunchKernelGGL((mla_linear_rows_kernel<XT, 4>), grid, dim3(512), 0, st, p);
  if (splits > 1) {
    const int64_t quads = (int64_t)p.tokens * 4 * p.tiles;
    hipLaunchKernelGGL(mla_linear_sum_kernel, dim3((uint32_t)((quads + 255) / 256)), dim3(256), 0, st, p, splits);
  }
}

static bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
static int refuse(const char* what, int code = MLA_ERR_INVALID) { return mla_srv::set_error(code, what); }
static int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mla_srv::set_error(MLA_ERR_HIP, std::string(what) + " launch failed: " + hipGetErrorString(e));
  return MLA_OK;
}

}  // namespace mla_layer

using namespace mla_layer;

extern "C" {

int mla_rms_norm(const mla_rms_norm_args* a, void* stream) {
  if (!a) return refuse("args is NULL");
  if (a->dtype != MLA_DTYPE_BF16 && a->dtype != MLA_DTYPE_F16 && a->dtype != MLA_DTYPE_F32)
    return refuse("dtype must be MLA_DTYPE_BF16, MLA_DTYPE_F16 or MLA_DTYPE_F32");
  if (a->weight_dtype != a->dtype && a->weight_dtype != MLA_DTYPE_F32) return refuse("weight_dtype must be dtype or MLA_DTYPE_F32");
  if (a->tokens < 0 || a->dim < 1 || a->reserved != 0) return refuse("tokens must be >= 0, dim >= 1, reserved 0");
  if (!(a->eps >= 0.f) || !isfinite(a->eps)) return refuse("eps must be finite and >= 0");
  if (a->scale && a->dim % 32) return refuse("8-bit rows take a dim that is a multiple of 32");
  if (a->tokens >= (1 << 24) || a->dim > (1 << 24)) return refuse("tokens must be below 2^24, dim at most 2^24", MLA_ERR_UNSUPPORTED);
  if (a->tokens == 0) return MLA_OK;
  if (!a->x || !a->weight || !a->out) return refuse("a required pointer is NULL");
  if (a->residual_out && !a->residual) return refuse("residual_out is the sum with a residual: it needs one");
  const int es = a->dtype == MLA_DTYPE_F32 ? 4 : 2, ws = a->weight_dtype == MLA_DTYPE_F32 ? 4 : 2;
  if (!aligned(a->x, es) || !aligned(a->residual, es) || !aligned(a->residual_out, es) || !aligned(a->weight, ws) ||
      (!a->scale && !aligned(a->out, es)))
    return refuse("pointers must be aligned to their elements");
  if (a->scale && (!aligned(a->out, 8) || a->out_stride % 8)) return refuse("8-bit rows must be 8-byte aligned, their stride a multiple of 8");
  if (a->x_stride < 0 || a->residual_stride < 0 || a->out_stride < 0 || a->residual_out_stride < 0) return refuse("strides must be non-negative");
  NormParams k{};
  k.x = (const uint8_t*)a->x;
  k.residual = (const uint8_t*)a->residual;
  k.weight = (const uint8_t*)a->weight;
  k.out = (uint8_t*)a->out;
  k.scale = a->scale;
  k.residual_out = (uint8_t*)a->residual_out;
  k.x_st = a->x_stride * es;
  k.r_st = a->residual_stride * es;
  k.o_st = a->out_stride * (a->scale ? 1 : es);
  k.ro_st = a->residual_out_stride * es;
  k.tokens = a->tokens;
  k.dim = a->dim;
  k.eps = a->eps;
  k.inv_dim = 1.f / (float)a->dim;
  k.w_f32 = a->weight_dtype == MLA_DTYPE_F32;
  const bool vec = aligned(a->x, 16) && aligned(a->weight, 16) && k.x_st % 16 == 0 && a->dim % (16 / es) == 0 &&
                   (!a->residual || (aligned(a->residual, 16) && k.r_st % 16 == 0)) &&
                   (!a->residual_out || (aligned(a->residual_out, 16) && k.ro_st % 16 == 0)) &&
                   (a->scale || (aligned(a->out, 16) && k.o_st % 16 == 0));
  const int cus = mla_srv::cu_count();
  const hipStream_t st = (hipStream_t)stream;
  constexpr int32_t kMost = 1 << 21;  // rows of a launch: it holds less than 2^32 threads, a row up to 1024
  for (int32_t left = a->tokens; left > 0; left -= kMost) {
    k.tokens = left < kMost ? left : kMost;
    if (a->dtype == MLA_DTYPE_BF16) launch_norm_type<Bf16>(k, vec, cus, st);
    else if (a->dtype == MLA_DTYPE_F16) launch_norm_type<F16>(k, vec, cus, st);
    else launch_norm_type<F32>(k, vec, cus, st);
    k.x += kMost * k.x_st;
    if (k.residual) k.residual += kMost * k.r_st;
    k.out += kMost * k.o_st;
    if (k.residual_out) k.residual_out += kMost * k.ro_st;
    if (k.scale) k.scale += (int64_t)kMost * (k.dim / 32);
  }
  return launched("rms norm");
}

static bool linear_shape(int32_t tokens, int32_t n, int32_t k) {
  return tokens >= 0 && tokens <= (1 << 20) && n >= 1 && n <= (1 << 22) && k >= 32 && k <= (1 << 22) && k % 32 == 0;
}

int64_t mla_linear_workspace_bytes(int32_t tokens, int32_t n, int32_t k) {
  if (!linear_shape(tokens, n, k)) return 0;
  const int64_t tiles = (n + 15) / 16, chunks = (k + 127) / 128;
  const int splits = linear_splits(tokens, tiles, chunks, mla_srv::cu_count());
  return splits > 1 ? (int64_t)splits * tokens * tiles * 64 : 0;
}

int mla_linear_fp4(const mla_linear_args* a, void* stream) {
  if (!a) return refuse("args is NULL");
  if (!linear_shape(a->tokens, a->n, a->k))
    return refuse("tokens must be in [0, 2^20], n in [1, 2^22], k a multiple of 32 in [32, 2^22]");
  if (a->y_dtype != MLA_DTYPE_BF16 && a->y_dtype != MLA_DTYPE_F16) return refuse("y_dtype must be MLA_DTYPE_BF16 or MLA_DTYPE_F16");
  if (a->reserved != 0) return refuse("reserved must be 0");
  if (!a->x_scale && a->x_dtype != MLA_DTYPE_BF16 && a->x_dtype != MLA_DTYPE_F16)
    return refuse("x_dtype must be MLA_DTYPE_BF16 or MLA_DTYPE_F16 (or 8-bit rows with x_scale)");
  if (a->tokens == 0) return MLA_OK;
  if (!a->x || !a->codes || !a->scale || !a->top || !a->y) return refuse("a required pointer is NULL");
  if (!aligned(a->x, 16) || !aligned(a->codes, 16) || !aligned(a->y, 2)) return refuse("x and codes must be 16-byte aligned");
  const int es = a->x_scale ? 1 : 2;
  if (a->x_stride < 0 || a->x_stride * es % 16 || a->x_scale_stride < 0 || a->y_stride < 0)
    return refuse("strides must be non-negative, x's a multiple of 16 bytes");
  LinearParams k{};
  k.x = (const uint8_t*)a->x;
  k.x_scale = a->x_scale;
  k.x_st = a->x_stride * es;
  k.xs_st = a->x_scale_stride;
  k.codes = (const uint8_t*)a->codes;
  k.scale = a->scale;
  k.top = a->top;
  k.y = (uint8_t*)a->y;
  k.y_st = a->y_stride * 2;
  k.tokens = a->tokens;
  k.n = a->n;
  k.k = a->k;
  k.tiles = (a->n + 15) / 16;
  k.chunks = (a->k + 127) / 128;
  k.y_f16 = a->y_dtype == MLA_DTYPE_F16;
  k.y_vec = aligned(a->y, 8) && k.y_st % 8 == 0;
  const int cus = mla_srv::cu_count();
  const int splits = linear_splits(k.tokens, k.tiles, k.chunks, cus);
  if (splits > 1) {
    if (!a->workspace || a->workspace_bytes < mla_linear_workspace_bytes(a->tokens, a->n, a->k))
      return refuse("workspace missing or smaller than mla_linear_workspace_bytes()", MLA_ERR_WORKSPACE);
    if (!aligned(a->workspace, 16)) return refuse("workspace must be 16-byte aligned", MLA_ERR_WORKSPACE);
    k.part = (float*)a->workspace;
  }
  const hipStream_t st = (hipStream_t)stream;
  if (a->x_scale) launch_linear<kRowsFp8>(k, splits, cus, st);
  else if (a->x_dtype == MLA_DTYPE_F16) launch_linear<kRowsF16>(k, splits, cus, st);
  else launch_linear<kRowsBf16>(k, splits, cus, st);
  return launched("linear");
}

}  // extern "C"
