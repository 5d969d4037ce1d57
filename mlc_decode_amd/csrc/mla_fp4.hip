// mla_fp4.hip -- split-KV MLA decode over the 4-bit latent cache (gfx950).
//
// A cached token is 512 latent dims as e2m1 codes (two a byte, the even dim in the low half), one
// scale byte s per 32 dims (value = e2m1(code) * 2^(s - 127); 255: the block is NaN) and 64 rope dims
// in bf16: 400 bytes.  Math, schedule, splits and partials are those of mla_decode.hip:
//   S = sm_scale * [q_nope|q_rope] . [latent|rope]^T,  O = softmax(S) . latent,  lse = log sum exp S.
//
// Three forms, by query rows and pages (see launch_decode): 16 and 64 rows in workgroups of four waves, two to a CU
// (one's matrix work covers the other's loads and barriers), and 128 rows in one of eight.  A workgroup owns one
// schedule part for its rows and walks it in stages of T tokens.
//  1. 64 and 128 rows: a lane holds 32 dims of one token as codes: that is the A operand of the block-scaled
//     16x16x128 MFMA as it stands, the scale byte its scale.  Nothing is converted for the QK product, whose tokens
//     every wave scores.  The queries are split once per segment into two e4m3 parts, q = hi + lo: a bf16 has eight
//     significant bits, each part holds four (see split_query for what is left).  The rope dims take the bf16 MFMA.
//     16 rows: a wave scores the tokens that it converts for V (2.), so QK takes those bf16 words: the same MFMA
//     clocks, exact products, and a score's relative error is 6e-8 instead of 1e-6.
//  2. The V operand needs tokens along k, and its scales vary along k, which the block-scaled MFMA does not
//     take: each wave converts its tokens' codes to bf16 (exact: two significant bits and a power of two)
//     and writes them to LDS, where transposed reads form V^T.
//  3. S^T tiles (token, row) are held by the wave that owns a row tile's token tiles; P^T goes through LDS in
//     operand order, rounded to bf16 (the PV operand's type; the sum that divides the output is of the rounded
//     weights, so that the rounding cancels in it), to all waves, each of which accumulates its share of the
//     512 output dims in fp32.
// What bounds them (one token a sequence unless said): 16 rows, 128 ragged sequences, 213 MB: 44.5 us in the main
// kernel, 4.8 TB/s, a large copy's rate, 52 with the merge.  64 rows: two barriers a stage with nothing between the
// products but the softmax: 64 x 64 heads x 4096 tokens 57 us where bytes and operations take 28, the matrix
// pipes busy 32% of the time.  128 rows: issue and waits (see mla_fp4_wide_kernel): 64 x 4096 tokens x 128 heads
// 78 us with the merge, 32 x 16384 x 2 x 128 235 us, 1.24 PFLOP/s of bf16 products.
// The running row maximum moves only when a score passes it by more than 2^kSlack (P then stays far from
// overflow in bf16 and fp32), so the output is rescaled rarely and exactly.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>

#include "mla_decode_amd.h"
#include "mla_fp4.h"
#include "mla_sched.h"

namespace mla4 {

using mla::kPageTokens;
using mla::kSchedWords;
using mla::pages_of;

constexpr int kDV = 512;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kSlack = 8.f;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((__vector_size__(4 * sizeof(short))));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((__vector_size__(8 * sizeof(__bf16))));
#define LDS_AS __attribute__((address_space(3)))

// LDS hand-off between the waves: own LDS accesses done, then the barrier.  Loads from HBM stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One wave's copy from HBM into LDS, 16 (or 4) bytes a lane: lane l's bytes land at lds + 16 l (4 l).  Inline asm,
// so that the compiler, which takes the builtin for an LDS store, does not wait for every copy in flight before
// it reads LDS; copies_landed() is the wait.  M0 is written without a save: nothing else here reads it; the copy
// needs one wait state after the write (s_nop 0), which the compiler would add for the builtin only.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16(const void* lane_addr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(lane_addr), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copy16(uint64_t base, uint32_t lane_off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copy4(uint64_t base, uint32_t lane_off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(lane_off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copy4(const void* lane_addr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(lane_addr), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void copies_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ float xor16(float v, bool sum) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
  return sum ? a + b : fmaxf(a, b);
}
__device__ __forceinline__ float xor32(float v, bool sum) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
  return sum ? a + b : fmaxf(a, b);
}
// The lane id.  FRESH: formed where it is called and not before, so that addresses derived from it are recomputed
// where they are used.  Hoisted out of the stage loop they take some forty registers that the 64-row form
// does not have, and a spilled address is reloaded behind every copy in flight (vmcnt is in order): 64 x 128
// heads x 4096 tokens 177 us with those reloads, 112 without.  The 16-row form has the registers (128 ragged
// sequences: 64.5 us with FRESH, 60 without).
template <bool FRESH>
__device__ __forceinline__ int lane_id() {
  if constexpr (!FRESH) return threadIdx.x & 63;
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}
// The maximum without fmaxf's canonicalising of each operand (scores are no signalling NaNs; a quiet one is passed over).
// Its operands come from ordinary vector instructions, or from MFMAs through settled(): the compiler does not see
// what asm reads, and keeps the wait states after an MFMA for its own instructions only.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// The results of the scaled MFMAs that were issued last, 12 wait states on.
__device__ __forceinline__ void settled(f32x4 (&s)[2]) { asm volatile("s_nop 7\n\ts_nop 3" : "+v"(s[0]), "+v"(s[1])); }
// over the four lane groups that hold one row
__device__ __forceinline__ float row_max(float v) { return xor32(xor16(v, false), false); }
__device__ __forceinline__ float row_sum(float v) { return xor32(xor16(v, true), true); }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}
__device__ __forceinline__ float sum2_bf16(uint32_t w, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{(__bf16)1.f, (__bf16)1.f}, acc, false);
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ f32x4 mfma_bf16(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// 16 tokens x 16 rows x 128 dims: A e2m1 (lane (g, i): dims 32g .. 32g+31 of token i), B e4m3 (lane (g, i):
// dims 16g .. +15 and 64 + 16g .. +15 of row i); the scale of dims 32g .. 32g+31 is byte CA (CB) of lane
// group g's word.
template <int CA, int CB>
__device__ __forceinline__ f32x4 mfma_scaled(i32x4 a, i32x8 b, f32x4 c, int scale_a, int scale_b) {
  const i32x8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b, c, 4, 0, CA, scale_a, CB, scale_b);
}
// chunk C of a score tile, the codes' scales in the low byte
__device__ __forceinline__ f32x4 score(int c, i32x4 k, const i32x8 (&q)[4], f32x4 acc, int scale_k, int scale_q) {
  return c == 0   ? mfma_scaled<0, 0>(k, q[0], acc, scale_k, scale_q)
         : c == 1 ? mfma_scaled<0, 1>(k, q[1], acc, scale_k, scale_q)
         : c == 2 ? mfma_scaled<0, 2>(k, q[2], acc, scale_k, scale_q)
                  : mfma_scaled<0, 3>(k, q[3], acc, scale_k, scale_q);
}

// the same with the scales of the four chunks in one word
__device__ __forceinline__ f32x4 score_packed(int c, i32x4 k, const i32x8 (&q)[4], f32x4 acc, int scale_k, int scale_q) {
  return c == 0   ? mfma_scaled<0, 0>(k, q[0], acc, scale_k, scale_q)
         : c == 1 ? mfma_scaled<1, 1>(k, q[1], acc, scale_k, scale_q)
         : c == 2 ? mfma_scaled<2, 2>(k, q[2], acc, scale_k, scale_q)
                  : mfma_scaled<3, 3>(k, q[3], acc, scale_k, scale_q);
}

// V in LDS: token t of a tile of 16 is a row of 1 KiB; its 16-byte chunk k sits at slot k ^ swz(t) of the
// 256-byte window it is in.  The conversions' 16-byte writes go eight lanes (tokens, one chunk) at a time over
// 128 bytes, so swz's low three bits tell eight tokens apart; the transposed reads go 32 lanes (eight tokens, 32
// bytes) at a time over 256, so its high three bits do too.  (A swizzle for the reads alone wrote at half rate.)
__device__ __forceinline__ int swz(int t) { return ((t & 3) << 1) | ((t >> 2) & 1) * 9; }

// Eight codes (one dword) to bf16 times 2^(byte - 127), the byte given as the exponent of a float.
__device__ __forceinline__ i32x4 widen8(int w, float scale) {
  return i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}

// One row's queries of a lane for one 128-dim chunk (v: four times eight bf16, the B operand's k = 16g .. +15 and
// 64 + 16g .. +15) as two e4m3 parts.  Per block of 32 dims, hi = q / 2^k rounded to e4m3 with the block's
// amax in [2, 4) * 2^k: e4m3 then steps by 2^-9 at least, and a product with a code (up to twelve halves)
// needs at most 13 bits.  The MFMA adds groups of eight products in a window of about that width below the
// largest (measured; between groups it adds as fp32), so hi's products lose nothing there, which a scale
// that uses all of e4m3's range does not give (relative error of S, normal data: 4.6e-6 at amax 240, 1.1e-6
// here).  lo = (q - hi) / 2^(k - 10) holds four more bits: values of the block's top seven binades are
// exact, smaller ones off by at most 2^-15 of the amax a.  So beside an outlier a thousand times as large a value is
// held to 2^-5, less than bf16's 2^-8; in a logit that is 2^-15 a |k_d|, where the outlier's own rounding to bf16 has
// put up to 2^-8 a |k|.  Queries of 512 dims with such an outlier in every block stay within the decodes' bar of 1e-3 (lse)
// and 1e-2 (outputs).
struct QuerySplit {
  i32x8 hi, lo;
  int scale;  // this lane group's scale byte of hi
};
__device__ __forceinline__ QuerySplit split_query(const i32x4 (&v)[4], int g, int li) {
  QuerySplit r;
  int byte[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // 32-dim block: h == 0: g / 2, h == 1: 2 + g / 2; half of it in lane group g ^ 1
    float x[16];
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int w = v[2 * h + (j >> 2)][j & 3];
      x[2 * j] = __uint_as_float((uint32_t)w << 16);
      x[2 * j + 1] = __uint_as_float((uint32_t)w & 0xFFFF0000u);
      amax = fmaxf(amax, fmaxf(fabsf(x[2 * j]), fabsf(x[2 * j + 1])));
    }
    amax = xor16(amax, false);
    int e = (int)(__float_as_uint(amax) >> 23) - 1;  // biased exponent of 2^k; an infinite amax gives 254
    e = e < 11 ? 11 : e;                              // lo's scale stays a normal power of two
    byte[h] = e;
    const float up = __uint_as_float((uint32_t)e << 23), down = __uint_as_float((uint32_t)(e - 10) << 23);
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // four values a dword
      i16x2 hi = {0, 0}, lo = {0, 0};
      hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[4 * j], x[4 * j + 1], up, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[4 * j + 2], x[4 * j + 3], up, true);
      const int hw = __builtin_bit_cast(int, hi);
      const f32x2 b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, up, false);
      const f32x2 b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, up, true);
      lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[4 * j] - b0[0], x[4 * j + 1] - b0[1], down, false);
      lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[4 * j + 2] - b1[0], x[4 * j + 3] - b1[1], down, true);
      r.hi[4 * h + j] = hw;
      r.lo[4 * h + j] = __builtin_bit_cast(int, lo);
    }
  }
  // lane group g gives block g's byte: blocks 0, 1 are the groups' 0, 2 first halves, 2, 3 their second ones
  const int src = li + 32 * (g & 1);
  const int first = __shfl(byte[0], src), second = __shfl(byte[1], src);
  r.scale = g < 2 ? first : second;
  return r;
}

// RT row tiles of 16 rows.  RT == 1: stages of 64 tokens, wave w takes token tile w from its loads, in registers,
// to its scores.  RT == 4: stages of 32 tokens, copied into one of two LDS buffers in fragment order (the
// copies of a stage are in flight during the one before), from which every wave scores; wave w converts half
// of the dims of token tile w % 2 and scores row tile w against both token tiles.
template <int RT>
struct Shape {
  static constexpr int T = RT == 1 ? 64 : 32;
  static constexpr int kTokTiles = T / 16;
  static constexpr int kTiles = RT * kTokTiles / 4;  // score tiles per wave
  static constexpr int kShare = 4 / RT;              // waves that share a row tile
};

// RT == 1: a stage's loads of one lane.
struct Stage {
  i32x4 code[4];
  i32x4 rope[2];
  i32x4 scale;
};

// RT == 4: a stage in LDS: per token tile four 1 KiB code fragments and two of rope, then the tokens' scale bytes.
constexpr int kRawTile = 6 * 1024;
constexpr int kRawScale = 2 * kRawTile;
constexpr int kRawStage = kRawScale + 512;

// The kernel's DecodeParams argument, read where it is used: as ordinary arguments they are all loaded at the start and
// kept, which is more scalar registers than there are, and the spilled ones live in vector registers.
typedef const DecodeParams __attribute__((address_space(4))) ArgParams;
constexpr int kArgOffset = 16;  // behind sched, row_blocks and num_parts
__device__ __forceinline__ ArgParams& params_here() {
  auto a = (const char __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(ArgParams*)(a + kArgOffset);
}

// Workgroups go to the eight XCDs in turn: the row blocks of a part, which read the same pages, take
// consecutive turns on one XCD and find them in its L2.
__device__ __forceinline__ void place_workgroup(int row_blocks, int num_parts, int& part, int& rb) {
  part = blockIdx.x;
  rb = 0;
  if (row_blocks > 1) {
    if ((num_parts & 7) == 0) {
      const int turn = blockIdx.x >> 3;
      rb = turn % row_blocks;
      part = (turn / row_blocks) * 8 + (blockIdx.x & 7);
    } else {
      rb = blockIdx.x % row_blocks;
      part = blockIdx.x / row_blocks;
    }
  }
}

// The tokens [tok0, tok1) of sequence b that a part takes from `page` on, L the sequence's length.
struct Segment {
  int L, tok0, tok1;
};
template <bool SPARSE>
__device__ __forceinline__ Segment segment_of(ArgParams& p, int b, int page, int end_b, int end_page) {
  int L = SPARSE ? p.topk : p.seqlens[b];
  L = L > 0 ? L : 0;
  if (!SPARSE && L > (int64_t)p.bt_width * kPageTokens) {  // uniform: cut to the table
    L = p.bt_width * kPageTokens;
    if (p.status != nullptr) *p.status = 1;
  }
  const int np = pages_of(L);
  int stop = b == end_b ? end_page : np;
  stop = stop < np ? stop : np;
  return Segment{L, page * kPageTokens, stop * kPageTokens < L ? stop * kPageTokens : L};
}

// The page id in column `at` of sequence b's table row, clamped into the pool: a scalar load.
template <bool SPARSE>
__device__ __forceinline__ int page_at(ArgParams& p, int b, int at) {
  if constexpr (SPARSE) return 0;
  const int last = p.bt_width - 1;
  const auto table = (const int32_t __attribute__((address_space(4)))*)p.block_table;
  const int v = table[(int64_t)b * p.bt_stride + (at < last ? at : last)];
  return v < 0 ? 0 : (v >= p.num_blocks ? p.num_blocks - 1 : v);
}

// Where token t of a segment is: row t % 64 of page pg, or the pool token that the segment's index list idx[0 .. n)
// names (an index that names none, and a t past the list, read a token that is masked later).
struct Row {
  const uint8_t* codes;
  const uint8_t* scale;
  const uint8_t* rope;
};
template <bool SPARSE>
__device__ __forceinline__ Row row_at(ArgParams& p, int t, int64_t pg, const int32_t* idx, int n) {
  int row = t & 63;
  if constexpr (SPARSE) {
    const int id = idx[t < n ? t : n - 1];
    const int64_t at = id >= 0 && id < p.pool_tokens ? id : 0;
    pg = at >> 6;
    row = (int)(at & 63);
  }
  return Row{p.codes + pg * p.c_sp + (uint32_t)(row * (int)p.c_st), p.scale + pg * p.s_sp + (uint32_t)(row * (int)p.s_st),
             (const uint8_t*)(p.rope + pg * p.r_sp + (uint32_t)(row * (int)p.r_st))};
}
// The segment's index list into LDS; whether any of it names no key (holes: a word a wave).  Every wave passes here.
__device__ __forceinline__ bool load_indices(ArgParams& p, int b, int tok0, int n, int threads, int32_t* idx, int* holes) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  bool none = false;
  for (int i = threadIdx.x; i < n; i += threads) {
    const int id = p.indices[(int64_t)b * p.idx_stride + tok0 + i];
    idx[i] = id;
    none |= id < 0 || id >= p.pool_tokens;
  }
  holes[wave] = __builtin_amdgcn_ballot_w64(none) != 0;
  lds_barrier();
  int any = 0;
  for (int w = 0; w < threads / 64; ++w) any |= holes[w];
  return __builtin_amdgcn_readfirstlane(any) != 0;
}
// Whether token t of a segment of n names no key (t < n, sparse), or is past the segment.
template <bool SPARSE>
__device__ __forceinline__ bool no_key(ArgParams& p, int t, const int32_t* idx, int n) {
  if constexpr (SPARSE) {
    const int id = idx[t < n ? t : n - 1];
    return t >= n || id < 0 || id >= p.pool_tokens;
  }
  return t >= n;
}

// The power of two that brings a chunk of a split's partial with this largest value into [2^14, 2^15).
__device__ __forceinline__ int part_exp(float amax) {
  const int e = 15 - __builtin_amdgcn_frexp_expf(amax);
  return e < 127 ? e : 127;
}
// Dims 16d + 4g .. + 3 (a) and 16(d + 1) + 4g .. + 3 (b) of a row, held by lane groups g, to dst: odd and even groups
// exchange, so that a lane stores 16 bytes and the row's four lanes a whole 64.
__device__ __forceinline__ void store_dims(uint16_t* dst, int d, int g, i32x2 a, i32x2 b) {
  const auto x = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), y = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  typedef i32x4 __attribute__((aligned(8))) unaligned_t;
  *(unaligned_t*)(dst + 16 * (d + (g & 1)) + 8 * (g >> 1)) = i32x4{(int)x[0], (int)y[0], (int)x[1], (int)y[1]};
}
// A row's lse from its reference m (log2) and the sum x of its weights; a row without a key has x = 0.  A NaN row (a NaN
// block, or a NaN in its query) reports lse -inf beside its NaN output, as the 16-bit and fp8 decodes do; its
// partials carry the NaN, which the merge turns into the same.
__device__ __forceinline__ void write_lse(ArgParams& p, int b, int row, int g, int64_t slot, bool single, float m, float x) {
  if (row >= p.rows || g != 0) return;
  const float lse2 = x == 0.f ? -INFINITY : m + __log2f(x);
  if (single) {
    const int sq = row / p.heads, h = row - sq * p.heads;
    if (p.lse != nullptr) p.lse[((int64_t)b * p.heads + h) * p.s_q + sq] = x > 0.f ? lse2 * kLn2 : -INFINITY;
  } else {
    p.ws_lse[slot * p.rows + row] = lse2;
  }
}

// The queries of a lane's row (rows past the last load the last, and are never written).
struct Query {
  i32x8 hi[4], lo[4];
  i32x4 rope[2];
  int scale_hi, scale_lo;  // a byte a chunk
  int lim;                 // the row sees tokens below it
};
__device__ __forceinline__ int clamp_row(ArgParams& p, int row) { return row < p.rows ? row : p.rows - 1; }
__device__ __forceinline__ const uint16_t* nope_of(ArgParams& p, int b, int tok, int h) {
  return p.q_nope + ((int64_t)b * p.q_sb + (int64_t)tok * p.q_ss + (int64_t)h * p.q_sh);
}
__device__ __forceinline__ const uint16_t* rope_of(ArgParams& p, int b, int tok, int h) {
  return p.q_rope + ((int64_t)b * p.qr_sb + (int64_t)tok * p.qr_ss + (int64_t)h * p.qr_sh);
}
__device__ __forceinline__ int limit_of(ArgParams& p, int L, int tok) { return L - (p.causal ? p.s_q - 1 - tok : 0); }
// Chunk c is dims 128c .. 128c + 127, or with SPREAD 32c .. 32c + 31 of each 128: lane group g of the codes then holds
// block 4g + c, whose scale byte is byte c of the token's dword g.
template <bool SPREAD>
__device__ __forceinline__ Query load_query(ArgParams& p, int b, int row, int L, int lane) {
  Query q;
  const int g = lane >> 4, li = lane & 15;
  row = clamp_row(p, row);
  const int tok = row / p.heads, h = row - tok * p.heads;
  const uint16_t* qn = nope_of(p, b, tok, h);
  const uint16_t* qp = rope_of(p, b, tok, h);
  q.scale_hi = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint16_t* src = qn + (SPREAD ? 128 * (g >> 1) + 32 * c + 16 * (g & 1) : 128 * c + 16 * g);
    constexpr int kHalf = SPREAD ? 256 : 64;
    const i32x4 v[4] = {*(const i32x4*)src, *(const i32x4*)(src + 8), *(const i32x4*)(src + kHalf), *(const i32x4*)(src + kHalf + 8)};
    const QuerySplit r = split_query(v, g, li);
    q.hi[c] = r.hi;
    q.lo[c] = r.lo;
    q.scale_hi |= r.scale << (8 * c);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) q.rope[j] = *(const i32x4*)(qp + 32 * j + 8 * g);
  q.scale_lo = q.scale_hi - 0x0A0A0A0A;  // every byte is 11 at least
  q.lim = limit_of(p, L, tok);
  return q;
}

// The same in bf16, for the form whose waves score the tokens that they convert: dims 128c + 32g + 8i .. + 7 are those
// of a token's word i of chunk c in lane group g.  All four waves need the same queries: each loads chunk `wave` and
// they exchange them through 16 KiB of LDS (a segment starts 2.6 us earlier than with all of it loaded by each).
struct Query16 {
  i32x4 nope[4];
  i32x4 rope[2];
  int tok;
};
__device__ __forceinline__ Query16 load_query16(ArgParams& p, int b, int row, int lane, int wave) {
  Query16 q;
  const int g = lane >> 4;
  row = clamp_row(p, row);
  q.tok = row / p.heads;
  const int h = row - q.tok * p.heads;
  const uint16_t* qn = nope_of(p, b, q.tok, h);
  const uint16_t* qp = rope_of(p, b, q.tok, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) q.nope[i] = *(const i32x4*)(qn + 128 * wave + 32 * g + 8 * i);
#pragma unroll
  for (int j = 0; j < 2; ++j) q.rope[j] = *(const i32x4*)(qp + 32 * j + 8 * g);
  __builtin_amdgcn_sched_barrier(0);
  return q;
}

template <int RT, bool SPARSE>
__global__ __launch_bounds__(256, 2) void mla_fp4_kernel(const int32_t* __restrict__ sched, int row_blocks,
                                                                       int num_parts, DecodeParams) {
  static_assert(alignof(DecodeParams) == 8 && kArgOffset % 8 == 0, "the struct's place among the arguments");
  using Sh = Shape<RT>;
  constexpr int T = Sh::T;
  constexpr bool kRaw = RT > 1;
  __shared__ __attribute__((aligned(1024))) uint8_t v_sh[T * 1024];
  __shared__ __attribute__((aligned(16))) uint8_t p_sh[RT * T * 32];  // [row tile][32 tokens][lane][16 bytes]
  __shared__ __attribute__((aligned(16))) uint8_t raw_sh[kRaw ? 2 * kRawStage : 16];
  __shared__ __attribute__((aligned(16))) uint8_t qr_sh[kRaw ? 4 * 2048 : 16];  // the waves' rope queries, in operand order
  __shared__ float max_sh[4][16];
  __shared__ float alpha_sh[RT][16];
  __shared__ __attribute__((aligned(4))) uint8_t moved_sh[4];  // row tile's reference moved in this stage
  __shared__ float sum_sh[4][2][16];
  __shared__ int lim_sh[4][16];
  __shared__ int32_t idx_sh[SPARSE ? MLA_SPARSE_MAX_TOPK : 1];
  __shared__ int holes_sh[4];

  int part, rb;
  place_workgroup(row_blocks, num_parts, part, rb);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rt_own = wave % RT;                               // the row tile this wave scores
  const int tt_load = RT == 1 ? wave : (wave & 1);            // the token tile it loads
  const int tt_own = (wave / RT) * Sh::kTiles;                // the first token tile it scores
  const int c_load = RT == 1 ? 0 : 2 * (wave >> 1);           // the first 128-dim chunk it loads
  const int row0 = rb * 16 * RT;

  uint8_t LDS_AS* const v_lds = (uint8_t LDS_AS*)v_sh;
  uint8_t LDS_AS* const p_lds = (uint8_t LDS_AS*)p_sh;
  uint8_t LDS_AS* const raw_lds = (uint8_t LDS_AS*)raw_sh;

  const int32_t* rec = sched + (int64_t)part * kSchedWords;
  int b = rec[0], page = rec[1], split = rec[4];
  const int end_b = rec[2], end_page = rec[3];

  const int batch = params_here().batch;
#pragma unroll 1
  for (; b < batch; ++b, page = 0, split = 0) {
    if (!(b < end_b || (b == end_b && page < end_page))) break;
    ArgParams& p = params_here();
    auto page_of = [&](int k) __attribute__((always_inline)) { return page_at<SPARSE>(p, b, page + k * T / kPageTokens); };
    const int ql_lane = lane_id<(RT > 1)>();
    const int q_row = row0 + 16 * rt_own + (ql_lane & 15);
    Query q;
    Query16 q16;
    i32x4 qn[4][4];  // RT == 1: the rows' nope queries
    // Before the segment's length and page are known: the waits of the three overlap.
    if constexpr (!kRaw) q16 = load_query16(p, b, q_row, ql_lane, wave);
    const int pg_first = page_of(0);
    const Segment seg = segment_of<SPARSE>(p, b, page, end_b, end_page);
    const int L = seg.L, tok0 = seg.tok0, tok1 = seg.tok1;
    const int nst = tok1 > tok0 ? (tok1 - tok0 + T - 1) / T : 0;

    bool holes = false;
    if constexpr (SPARSE) holes = load_indices(p, b, tok0, tok1 - tok0, 256, idx_sh, holes_sh);

    auto row_of = [&](int t, int pg) __attribute__((always_inline)) { return row_at<SPARSE>(p, t, pg, idx_sh, tok1 - tok0); };
    auto load_stage = [&](int k, int pg, Stage& s) __attribute__((always_inline)) {  // RT == 1
      const int lane = lane_id<(RT > 1)>(), g = lane >> 4, li = lane & 15;
      const Row r = row_of(k * T + 16 * tt_load + li, pg);
#pragma unroll
      for (int c = 0; c < 4; ++c) s.code[c] = *(const i32x4*)(r.codes + 64 * c + 16 * g);
      s.scale = *(const i32x4*)r.scale;
#pragma unroll
      for (int j = 0; j < 2; ++j) s.rope[j] = *(const i32x4*)(r.rope + 64 * j + 16 * g);
    };
    auto copy_stage = [&](int k, int pg) __attribute__((always_inline)) {  // RT > 1
      const int lane = lane_id<(RT > 1)>(), g = lane >> 4, li = lane & 15;
      const Row r = row_of(k * T + 16 * tt_load + li, pg);
      const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)raw_lds + (k & 1) * kRawStage);
      const uint32_t tile = base + tt_load * kRawTile;
#pragma unroll
      for (int c = 0; c < 2; ++c) copy16(r.codes + 64 * (c_load + c) + 16 * g, tile + 1024 * (c_load + c));
      copy16(r.rope + 64 * (wave >> 1) + 16 * g, tile + 1024 * (4 + (wave >> 1)));
      if (wave < 2) {  // uniform: a dword of scales a lane, four lanes a token
        const Row w = row_of(k * T + 16 * wave + (lane >> 2), pg);
        copy4(w.scale + 4 * (lane & 3), base + kRawScale + 256 * wave);
      }
    };

    Stage nxt;
    int pg_next = 0;
    if (nst > 0) {
      if constexpr (kRaw)
        copy_stage(0, pg_first);
      else
        load_stage(0, pg_first, nxt);
      pg_next = page_of(nst > 1 ? 1 : 0);
    }

    if constexpr (kRaw) {
      q = load_query<false>(p, b, q_row, L, ql_lane);
#pragma unroll
      for (int j = 0; j < 2; ++j) *(i32x4 LDS_AS*)((uint8_t LDS_AS*)qr_sh + (wave * 2 + j) * 1024 + ql_lane * 16) = q.rope[j];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) *(i32x4 LDS_AS*)(v_lds + (4 * wave + i) * 1024 + ql_lane * 16) = q16.nope[i];
      lds_barrier();
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) qn[c][i] = *(const i32x4 LDS_AS*)(v_lds + (4 * c + i) * 1024 + ql_lane * 16);
      lds_barrier();  // read before the stages' V takes the place
      // used here once: the wait for them is not left to the stage loop
      asm volatile("" : "+v"(q16.rope[0]), "+v"(q16.rope[1]));
      q.lim = limit_of(p, L, q16.tok);
    }
    lim_sh[wave][ql_lane & 15] = q.lim;
    const int lim_min = L - (p.causal ? p.s_q - 1 : 0);     // every row sees those below it

    f32x4 o[8][RT];
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < RT; ++r) o[d][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_ref = -INFINITY, l_rnd = 0.f, l_exact = 0.f;
    const float scale_log2 = p.scale_log2;

#pragma unroll 1
    for (int k = 0; k < nst; ++k) {
      Stage cur;
      const uint8_t LDS_AS* const raw = raw_lds + (k & 1) * kRawStage;
      if constexpr (kRaw) {
        copies_landed();
        lds_barrier();  // the stage is in LDS; V, P and the other buffer are free
        if (k + 1 < nst) copy_stage(k + 1, pg_next);
      } else {
        cur = nxt;
        if (k + 1 < nst) load_stage(k + 1, pg_next, nxt);
      }
      pg_next = page_of(k + 2 < nst ? k + 2 : nst - 1);
      const int tok_k = tok0 + k * T;
      const int lane = lane_id<(RT > 1)>(), g = lane >> 4, li = lane & 15;
      // ---- 1. the wave's tokens to bf16 in LDS.  Tokens that do not exist become zeros: their weight is
      // zero, and what their rows hold must not make 0 * NaN of it.  So do the NaN blocks of tokens that some
      // rows do not see: the score of a row that sees one is NaN, and with it all of its outputs.
      const bool cut = holes || tok_k + T > tok1 || tok_k + T > lim_min;  // uniform
      const bool gone = cut && no_key<SPARSE>(p, tok_k + 16 * tt_load + li - tok0, idx_sh, tok1 - tok0);
      i32x4 code;  // chunk c of the token (c_load + c of its 128-dim chunks)
      float scale = 0.f;
      bool bad = false;  // one of the lane's blocks is NaN (RT == 1: QK takes the zeros too, and its score is set)
      auto code_in = [&](int c) __attribute__((always_inline)) {
        uint32_t w;
        if constexpr (kRaw) {
          code = *(const i32x4 LDS_AS*)(raw + tt_load * kRawTile + (c_load + c) * 1024 + lane * 16);
          w = *(const uint32_t LDS_AS*)(raw + kRawScale + (tt_load * 16 + li) * 16 + 4 * (c_load + c));
        } else {
          code = cur.code[c];
          w = (uint32_t)cur.scale[c];
        }
        scale = __uint_as_float(((w >> (8 * g)) & 0xFF) << 23);  // byte 255 is infinity
        if (cut) {  // uniform
          const bool nan = scale == INFINITY, none = gone || nan;
          bad |= nan;
          scale = none ? 1.f : scale;
#pragma unroll
          for (int j = 0; j < 4; ++j) code[j] = none ? 0 : code[j];
        }
      };
      // word i of a chunk: 8 dims of token li of tile tt_load, chunk 4g + i of a 256-byte window
      const int v_at = tt_load * 16384 + li * 1024 + (((4 * g) ^ swz(li)) << 4);
      auto widen_word = [&](int c, int i) __attribute__((always_inline)) {
        *(i32x4 LDS_AS*)(v_lds + 256 * (c_load + c) + (v_at ^ (16 * i))) = widen8(code[i], scale);
      };
      // ---- 2. scores of the wave's tiles
      f32x4 s[Sh::kTiles];
      if constexpr (kRaw) {
        // Two rope steps, then four of 128 dims; a step's fragments are read during the step before, and the
        // conversions of the wave's own tokens fill the gaps between the MFMAs.
        i32x4 kf[2][Sh::kTiles], qf[2];
        uint32_t ks[2][Sh::kTiles];  // the token's four scale bytes of the step's chunk
        const uint8_t LDS_AS* const tile = raw + tt_own * kRawTile + lane * 16;
        auto read_step = [&](int st) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < Sh::kTiles; ++i)
          {
            kf[st & 1][i] = *(const i32x4 LDS_AS*)(tile + i * kRawTile + 1024 * (st < 2 ? 4 + st : st - 2));
            if (st >= 2) ks[st & 1][i] = *(const uint32_t LDS_AS*)(raw + kRawScale + ((tt_own + i) * 16 + li) * 16 + 4 * (st - 2));
          }
        };
#pragma unroll
        for (int j = 0; j < 2; ++j) qf[j] = *(const i32x4 LDS_AS*)((const uint8_t LDS_AS*)qr_sh + (wave * 2 + j) * 1024 + lane * 16);
        read_step(0);
#pragma unroll
        for (int i = 0; i < Sh::kTiles; ++i) {
          s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int st = 0; st < 6; ++st) {
          if (st < 5) read_step(st + 1);
          if (st == 1) code_in(0);
          if (st < 2) {
#pragma unroll
            for (int i = 0; i < Sh::kTiles; ++i) s[i] = mfma_bf16(kf[st & 1][i], qf[st], s[i]);
          } else {
            int sc[Sh::kTiles];
#pragma unroll
            for (int i = 0; i < Sh::kTiles; ++i) sc[i] = (int)(ks[st & 1][i] >> (8 * g));  // the low byte counts
#pragma unroll
            for (int i = 0; i < Sh::kTiles; ++i) s[i] = score(st - 2, kf[st & 1][i], q.hi, s[i], sc[i], q.scale_hi);
#pragma unroll
            for (int i = 0; i < Sh::kTiles; ++i) s[i] = score(st - 2, kf[st & 1][i], q.lo, s[i], sc[i], q.scale_lo);
            widen_word((st - 2) >> 1, 2 * (st & 1));
            widen_word((st - 2) >> 1, 2 * (st & 1) + 1);
            if (st == 3) code_in(1);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < Sh::kTiles; ++i) s[i] *= scale_log2;
      } else {
        // The words that go to LDS for V are the QK operand too.
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, l = a;
        a = mfma_bf16(cur.rope[0], q16.rope[0], a);
        l = mfma_bf16(cur.rope[1], q16.rope[1], l);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          code_in(c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const i32x4 w = widen8(code[i], scale);
            *(i32x4 LDS_AS*)(v_lds + 256 * c + (v_at ^ (16 * i))) = w;
            if (i & 1)
              l = mfma_bf16(w, qn[c][i], l);
            else
              a = mfma_bf16(w, qn[c][i], a);
          }
        }
        s[0] = (a + l) * scale_log2;
      }
      if (cut) {  // uniform
        const int lim = lim_sh[wave][li];
        uint32_t nan_tokens = 0;  // of the tile, a bit each: lane (g, li) has token li's blocks of lane group g
        if constexpr (!kRaw) {
          const uint64_t m = __builtin_amdgcn_ballot_w64(bad);
          nan_tokens = (uint32_t)(m | m >> 16 | m >> 32 | m >> 48);
        }
#pragma unroll
        for (int i = 0; i < Sh::kTiles; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = tok_k + 16 * (tt_own + i) + 4 * g + j;
            const bool see = t < lim && !no_key<SPARSE>(p, t - tok0, idx_sh, tok1 - tok0);
            if constexpr (!kRaw) s[i][j] = (nan_tokens >> (4 * g + j)) & 1 ? NAN : s[i][j];
            s[i][j] = see ? s[i][j] : -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < Sh::kTiles; ++i) top = fmaxf(top, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
      top = row_max(top);
      if constexpr (Sh::kShare > 1) {
        max_sh[wave][li] = top;
        lds_barrier();
#pragma unroll
        for (int w = 0; w < Sh::kShare; ++w) top = fmaxf(top, max_sh[w * RT + rt_own][li]);
      }
      // ---- 3. weights.  The waves of a row tile see the same maxima and move the reference alike.
      const float m_old = m_ref;
      m_ref = top > m_ref + kSlack ? top : m_ref;
      const bool moved = __builtin_amdgcn_ballot_w64(m_ref != m_old) != 0;
      const float base = m_ref == -INFINITY ? 0.f : m_ref;
      float alpha = 1.f;
      if (moved) {  // uniform
        alpha = __builtin_amdgcn_exp2f((m_old == m_ref ? base : m_old) - base);
        l_rnd *= alpha;
        l_exact *= alpha;
      }
      if (wave < RT) {
        if (moved) alpha_sh[rt_own][li] = alpha;
        moved_sh[rt_own] = moved;
      }
#pragma unroll
      for (int i = 0; i < Sh::kTiles; ++i) {
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          e[j] = __builtin_amdgcn_exp2f(s[i][j] - base);
          l_exact += e[j];
        }
        const i32x2 w = {(int)pack_bf16(e[0], e[1]), (int)pack_bf16(e[2], e[3])};
        l_rnd = sum2_bf16((uint32_t)w[1], sum2_bf16((uint32_t)w[0], l_rnd));
        const int tt = tt_own + i;
        *(i32x2 LDS_AS*)(p_lds + ((rt_own * (T / 32) + (tt >> 1)) * 64 + lane) * 16 + 8 * (tt & 1)) = w;
      }
      lds_barrier();
      // ---- 4. output dims 128 * wave .. + 127 of all rows
      // V^T reads: token 4g + li/4, dims 128 * wave + 16d + 4 * (li % 4): the window's chunk 2d + (li/2) % 2
      const int ln = lane_id<(RT > 1)>(), rv = 4 * (ln >> 4) + ((ln & 15) >> 2);
      const int v_read = rv * 1024 + wave * 256 + ((((ln >> 1) & 1) ^ swz(rv)) << 4) + ((ln & 1) << 3);
      auto read_v = [&](int ks, int d) __attribute__((always_inline)) {
        const uint8_t LDS_AS* src = v_lds + (v_read ^ (32 * d)) + ks * 32768;
        const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)src));
        const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)(src + 16384)));
        return i32x4{lo[0], lo[1], hi[0], hi[1]};
      };
      const uint32_t moves = *(const uint32_t LDS_AS*)(const uint8_t LDS_AS*)moved_sh;  // a byte a row tile
      i32x4 pb[T / 32][RT], va[3];
#pragma unroll
      for (int ks = 0; ks < T / 32; ++ks)
#pragma unroll
        for (int r = 0; r < RT; ++r) pb[ks][r] = *(const i32x4 LDS_AS*)(p_lds + ((r * (T / 32) + ks) * 64 + ln) * 16);
      va[0] = read_v(0, 0);
      va[1] = read_v(0, 1);
      const uint32_t any = __builtin_amdgcn_readfirstlane(moves);
      if (any & (0xFFFFFFFFu >> (32 - 8 * RT))) {  // uniform, rare
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          if ((any >> (8 * r)) & 0xFF) {  // uniform
            const float al = alpha_sh[r][ln & 15];
#pragma unroll
            for (int d = 0; d < 8; ++d) o[d][r] *= al;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < T / 4; ++n) {  // (ks, d) = (n / 8, n % 8), two V^T fragments ahead
        if (n + 2 < T / 4) va[(n + 2) % 3] = read_v((n + 2) / 8, (n + 2) % 8);
#pragma unroll
        for (int r = 0; r < RT; ++r) o[n % 8][r] = mfma_bf16(va[n % 3], pb[n / 8][r], o[n % 8][r]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (!kRaw) lds_barrier();  // V, P and the words of this stage are free
    }
    if constexpr (kRaw) lds_barrier();  // the raw buffers are free for the next segment

    // ---- the rows' sums from the waves that scored them
    const int lane = lane_id<(RT > 1)>(), g = lane >> 4, li = lane & 15;
    ArgParams& e = params_here();
    const int slot0 = e.splits[b];
    const bool single = e.splits[b + 1] - slot0 == 1;
    l_rnd = row_sum(l_rnd);
    l_exact = row_sum(l_exact);
    sum_sh[wave][0][li] = l_rnd;
    sum_sh[wave][1][li] = l_exact;
    lds_barrier();
    const int64_t slot = (int64_t)slot0 + split;
    if (wave < RT) {  // lse of row tile `wave`
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < Sh::kShare; ++w) x += sum_sh[w * RT + rt_own][1][li];
      write_lse(e, b, row0 + 16 * rt_own + li, g, slot, single, m_ref, x);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < Sh::kShare; ++w) l += sum_sh[w * RT + r][0][li];
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int row = row0 + 16 * r + li;
      if (single) {
        if (row < e.rows) {
          const int sq = row / e.heads, h = row - sq * e.heads;
          uint16_t* dst = e.out + ((int64_t)b * e.o_sb + (int64_t)sq * e.o_ss + (int64_t)h * e.o_sh) + 128 * wave;
#pragma unroll
          for (int d = 0; d < 8; d += 2) {
            const f32x4 v = o[d][r] * inv, w = o[d + 1][r] * inv;
            store_dims(dst, d, g, i32x2{(int)pack_bf16(v[0], v[1]), (int)pack_bf16(v[2], v[3])},
                       i32x2{(int)pack_bf16(w[0], w[1]), (int)pack_bf16(w[2], w[3])});
          }
        }
      } else {  // scaled fp16, as every split's partial (the wave's 128 dims are one chunk)
        float am = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) am = fmaxf(am, fabsf(o[d][r][j]));
        am = row_max(am * inv);
        const int ex = part_exp(am);
        if (row < e.rows) {
          uint16_t* dst = e.ws_o + (slot * e.rows + row) * kDV + 128 * wave;
#pragma unroll
          for (int d = 0; d < 8; d += 2) {
            const f32x4 v = (o[d][r] * inv) * exp2i(ex), w = (o[d + 1][r] * inv) * exp2i(ex);
            store_dims(dst, d, g, i32x2{(int)pack_f16(v[0], v[1]), (int)pack_f16(v[2], v[3])},
                       i32x2{(int)pack_f16(w[0], w[1]), (int)pack_f16(w[2], w[3])});
          }
          if (g == 0) e.ws_scale[(slot * e.rows + row) * 4 + wave] = exp2i(-ex);
        }
      }
    }
    lds_barrier();  // the sums are read before the next segment's
  }
}

// 128 query rows: eight waves of one workgroup per CU, wave w scoring row tile w against both token tiles of a
// 32-token stage and accumulating output dims 64w .. 64w + 63 of all rows.  One barrier a stage: while a
// wave scores stage k and converts its share of V, P^T and V of stage k - 1 lie in the other half of two
// buffers, and their product is interleaved with the softmax of stage k.  V is converted once for 128 rows.
// (Two 64-row workgroups a CU: 64 x 128 heads x 4096 tokens 97 us, 32 x 2 x 128 x 16384 303; the first form of this
// kernel, which formed every address anew, 88 and 263, with the addresses kept 82 and 240, and with rows stored as 16
// bytes a lane 80 and 235.)
// What bounds it is issue and waits: of the waves' cycles (64 x 4096 tokens x 128 heads) 36% wait to issue and 32% at
// counters and barriers, which two waves a SIMD cannot cover for each other; the matrix pipes are busy 46% of the
// time, LDS 34%, a fifth of that in bank conflicts.  A SIMD's MFMA time and the vector instructions beyond
// two per MFMA add up (measured: two waves of one bf16 MFMA and 2, 4, 8 additions a step take 18.5, 26, 37 cycles a
// step), so the loop keeps its lane addresses, takes buffer halves as constants (two stages a turn) and page
// addresses as scalars.
//
// A stage in LDS (kRawStage bytes): per token tile the codes as [lane group g][token][16-byte piece c ^ (token / 2 % 4)]
// of the 64 bytes that hold blocks 4g .. 4g + 3 (the copies read whole 64 bytes, and the fragment reads of one c
// spread over the banks), two rope fragments, then the tokens' scale bytes.
template <bool SPARSE>
__global__ __launch_bounds__(512, 2) void mla_fp4_wide_kernel(const int32_t* __restrict__ sched, int row_blocks, int num_parts,
                                                              DecodeParams) {
  constexpr int T = 32, RT = 8, W = 8;
  __shared__ __attribute__((aligned(1024))) uint8_t v_sh[2][T * 1024];
  __shared__ __attribute__((aligned(16))) uint8_t p_sh[2][RT * 1024];  // [row tile][lane][16 bytes]
  __shared__ __attribute__((aligned(16))) uint8_t raw_sh[2][kRawStage];
  __shared__ __attribute__((aligned(16))) uint8_t qr_sh[W * 2048];  // the waves' rope queries, in operand order
  __shared__ float alpha_sh[2][RT][16];
  __shared__ int moved_sh[2][RT];  // stage in which the row tile's reference last moved, by its parity
  __shared__ int any_sh[2];        // and any row tile's
  __shared__ float sum_sh[RT][16];
  __shared__ float amax_sh[W][RT][16];
  __shared__ int lim_sh[W][16];
  __shared__ int32_t idx_sh[SPARSE ? MLA_SPARSE_MAX_TOPK : 1];
  __shared__ int holes_sh[W];

  int part, rb;
  place_workgroup(row_blocks, num_parts, part, rb);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tt_load = wave & 1, g_load = wave >> 1;  // the token tile and lane group's 128 dims it copies
  const int row0 = rb * 16 * RT;
  const auto lds_at = [](const void* a) { return (uint32_t)(uintptr_t)(const uint8_t LDS_AS*)a; };
  const auto at_lds = [](uint32_t a) { return (uint8_t LDS_AS*)a; };
  const uint32_t raw_base = __builtin_amdgcn_readfirstlane(lds_at(raw_sh));

  // lane addresses in LDS that live through the kernel
  const int lane0 = threadIdx.x & 63, g0 = lane0 >> 4, li0 = lane0 & 15;
  const uint32_t frag_at = lds_at(raw_sh) + g0 * 1024 + li0 * 64 + (((li0 >> 1) & 3) << 4);  // chunk 0; chunk c: ^ 16c
  const uint32_t word_at = lds_at(raw_sh) + kRawScale + li0 * 16 + 4 * g0;
  // V writes: token li of tile wave / 4, dims 128g + 32 (wave % 4) .. + 31: the chunk of this wave's conversion
  const int tt_conv = wave >> 2, c_conv = wave & 3;
  const uint32_t vw_base = lds_at(v_sh) + tt_conv * 16384;
  const auto v_write = [&](int lane) {
    return vw_base + (lane & 15) * 1024 + (lane >> 4) * 256 + (((4 * c_conv) ^ swz(lane & 15)) << 4);
  };
  const uint32_t vw_kept = v_write(lane0);
  // V^T reads: token 4g + li/4, dims 64 * wave + 16d + 4 * (li % 4)
  const int rv = 4 * g0 + (li0 >> 2);
  const uint32_t vr_at = lds_at(v_sh) + rv * 1024 + (wave >> 1) * 256 + (((8 * (wave & 1) + ((li0 >> 1) & 1)) ^ swz(rv)) << 4) + ((li0 & 1) << 3);

  const int32_t* rec = sched + (int64_t)part * kSchedWords;
  int b = rec[0], page = rec[1], split = rec[4];
  const int end_b = rec[2], end_page = rec[3];
  const int batch = params_here().batch;
#pragma unroll 1
  for (; b < batch; ++b, page = 0, split = 0) {
    if (!(b < end_b || (b == end_b && page < end_page))) break;
    ArgParams& p = params_here();
    const Segment seg = segment_of<SPARSE>(p, b, page, end_b, end_page);
    const int tok0 = seg.tok0, tok1 = seg.tok1;
    const int nst = tok1 > tok0 ? (tok1 - tok0 + T - 1) / T : 0;
    if (threadIdx.x < 2) any_sh[threadIdx.x] = -1;
    if (threadIdx.x < 2 * RT) moved_sh[0][threadIdx.x] = -1;
    bool holes = false;
    if constexpr (SPARSE) holes = load_indices(p, b, tok0, tok1 - tok0, 64 * W, idx_sh, holes_sh);
    // What the copies of every stage need, held in scalar registers: read from the arguments in the loop, each stage
    // waited for scalar loads.  A wave's second copy is of rope (waves 0 .. 3) or of scales (4, 5).
    uint64_t codes = (uint64_t)p.codes, second = wave < 4 ? (uint64_t)p.rope : (uint64_t)p.scale;
    int64_t c_sp = p.c_sp, second_sp = wave < 4 ? 2 * p.r_sp : p.s_sp;
    int c_st = (int)p.c_st, second_st = wave < 4 ? 2 * (int)p.r_st : (int)p.s_st;
    uint64_t table = SPARSE ? 0 : (uint64_t)(p.block_table + (int64_t)b * p.bt_stride);
    int last_col = p.bt_width - 1, last_page = p.num_blocks - 1;
    asm volatile("" : "+s"(codes), "+s"(second), "+s"(c_sp), "+s"(second_sp), "+s"(c_st), "+s"(second_st), "+s"(table), "+s"(last_col), "+s"(last_page));
    // Lane i holds the id of the segment's page `held` + i, clamped into the pool.
    int held = 0, ids = 0;
    auto hold_ids = [&](int first) __attribute__((always_inline)) {
      if constexpr (!SPARSE) {
        held = first;
        const int at = page + first + lane_id<true>();
        const int v = ((const int32_t*)table)[at < last_col ? at : last_col];
        ids = v < 0 ? 0 : (v < last_page ? v : last_page);
      }
    };
    auto page_of = [&](int k) __attribute__((always_inline)) {
      if constexpr (SPARSE) return 0;
      const int at = k * T / kPageTokens;
      if (at - held >= 64) hold_ids(at);  // uniform
      return __builtin_amdgcn_readlane(ids, at - held);
    };
    // each wave a KiB of codes, waves 0 .. 3 a rope fragment, 4 and 5 a tile's scale bytes
    auto copy_stage = [&](int k, int pg) __attribute__((always_inline)) {
      const int lane = lane_id<true>();
      const uint32_t base = raw_base + (k & 1) * kRawStage, tile = base + tt_load * kRawTile;
      // codes: four lanes a token, its 16-byte piece (lane % 4) ^ (token / 2 % 4)
      const int t4 = lane >> 2, piece = 64 * g_load + 16 * ((lane & 3) ^ ((lane >> 3) & 3));
      const int rope_at = 64 * (wave >> 1) + 16 * (lane >> 4), li = lane & 15;
      if constexpr (SPARSE) {
        const Row r = row_at<true>(p, k * T + 16 * tt_load + t4, 0, idx_sh, tok1 - tok0);
        copy16(r.codes + piece, tile + 1024 * g_load);
        if (wave < 4) {  // uniform
          const Row q = row_at<true>(p, k * T + 16 * tt_load + li, 0, idx_sh, tok1 - tok0);
          copy16(q.rope + rope_at, tile + 1024 * (4 + (wave >> 1)));
        } else if (wave < 6) {
          copy4(r.scale + 4 * (lane & 3), base + kRawScale + 256 * tt_load);
        }
      } else {
        const int row = (k * T & (kPageTokens - 1)) + 16 * tt_load;  // of the tile's first token
        copy16(codes + (int64_t)pg * c_sp + (int64_t)(row * c_st), (uint32_t)(t4 * c_st + piece), tile + 1024 * g_load);
        const uint64_t from = second + (int64_t)pg * second_sp + (int64_t)(row * second_st);
        if (wave < 4)  // uniform
          copy16(from, (uint32_t)(li * second_st + rope_at), tile + 1024 * (4 + (wave >> 1)));
        else if (wave < 6)
          copy4(from, (uint32_t)(t4 * second_st + 4 * (lane & 3)), base + kRawScale + 256 * tt_load);
      }
    };
    if (nst > 0) {
      hold_ids(0);
      copy_stage(0, page_of(0));
    }
    i32x8 qh[4], ql[4];
    int qs_hi;
    {
      const int lane = lane_id<true>();
      const Query q = load_query<true>(p, b, row0 + 16 * wave + (lane & 15), seg.L, lane);
#pragma unroll
      for (int c = 0; c < 4; ++c) qh[c] = q.hi[c], ql[c] = q.lo[c];
      qs_hi = q.scale_hi;
#pragma unroll
      for (int j = 0; j < 2; ++j) *(i32x4 LDS_AS*)at_lds(lds_at(qr_sh) + wave * 2048 + j * 1024 + lane * 16) = q.rope[j];
      lim_sh[wave][lane & 15] = q.lim;
    }
    const int lim_min = seg.L - (p.causal ? p.s_q - 1 : 0);  // every row sees the tokens below it
    const float scale_log2 = p.scale_log2;

    f32x4 o[4][RT];
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < RT; ++r) o[d][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_ref = -INFINITY, l_rnd = 0.f, l_exact = 0.f;

    // ---- q . k of stage k (in buffer `buf`) for row tile `wave`, and this wave's share of V of stage k
    auto scores = [&](int k, auto buf, f32x4 (&s)[2]) __attribute__((always_inline)) {
      constexpr int B = decltype(buf)::value;
      const int t0 = k * T;  // in the segment
      const bool cut = holes || tok0 + t0 + T > tok1 || tok0 + t0 + T > lim_min;  // uniform
      const uint32_t lane16 = 16 * lane_id<true>();
      int qs_lo;  // formed here: one register less to keep
      asm volatile("v_add_u32 %0, 0xf5f5f5f6, %1" : "=v"(qs_lo) : "v"(qs_hi));
      // (the sparse form, with more addresses of copies, has no register for it)
      const uint32_t vw_at = SPARSE ? v_write(lane_id<true>()) : vw_kept;
      i32x4 kf[2][2], qf[2], code;
      int ks[2];
      float scale = 0.f;
      auto read_step = [&](int st) __attribute__((always_inline)) {
        const uint32_t at = st < 2 ? raw_base + lane16 + 1024 * (4 + st) : (frag_at ^ (16 * (st < 2 ? 0 : st - 2)));
#pragma unroll
        for (int i = 0; i < 2; ++i) kf[st & 1][i] = *(const i32x4 LDS_AS*)at_lds(at + B * kRawStage + i * kRawTile);
      };
#pragma unroll
      for (int j = 0; j < 2; ++j) qf[j] = *(const i32x4 LDS_AS*)at_lds(lds_at(qr_sh) + wave * 2048 + j * 1024 + lane16);
      read_step(0);
#pragma unroll
      for (int i = 0; i < 2; ++i) ks[i] = *(const int LDS_AS*)at_lds(word_at + B * kRawStage + i * 256);
      s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < 6; ++st) {
        if (st < 5) read_step(st + 1);
        if (st == 1) {
          code = *(const i32x4 LDS_AS*)at_lds((frag_at ^ (16 * c_conv)) + B * kRawStage + tt_conv * kRawTile);
          scale = __uint_as_float((((uint32_t)(tt_conv ? ks[1] : ks[0]) >> (8 * c_conv)) & 0xFF) << 23);
          // uniform: tokens that do not exist become zeros, and NaN blocks where some rows do not see the token (as above)
          if (cut) {
            const bool none = scale == INFINITY || no_key<SPARSE>(p, t0 + 16 * tt_conv + (lane_id<true>() & 15), idx_sh, tok1 - tok0);
            scale = none ? 1.f : scale;
#pragma unroll
            for (int j = 0; j < 4; ++j) code[j] = none ? 0 : code[j];
          }
        }
        if (st < 2) {
#pragma unroll
          for (int i = 0; i < 2; ++i) s[i] = mfma_bf16(kf[st & 1][i], qf[st], s[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) s[i] = score_packed(st - 2, kf[st & 1][i], qh, s[i], ks[i], qs_hi);
#pragma unroll
          for (int i = 0; i < 2; ++i) s[i] = score_packed(st - 2, kf[st & 1][i], ql, s[i], ks[i], qs_lo);
          *(i32x4 LDS_AS*)at_lds((vw_at ^ (16 * (st - 2))) + B * (T * 1024)) = widen8(code[st - 2], scale);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (cut) {  // uniform
        const int lane = lane_id<true>(), lim = lim_sh[wave][lane & 15];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = t0 + 16 * i + 4 * (lane >> 4) + j;
            s[i][j] = tok0 + t < lim && !no_key<SPARSE>(p, t, idx_sh, tok1 - tok0) ? s[i][j] : -INFINITY;
          }
      }
    };

    // ---- softmax of stage k (SOFT; P to buffer `buf`) in pieces between the products P V of stage k - 1 (PV; from
    // byte offsets p_was and v_was of the buffers).  Where the reference stays, alpha is exactly one.
    auto weigh = [&](auto soft, auto pv, auto buf, int k, uint32_t p_was, uint32_t v_was, int was, f32x4 (&s)[2]) __attribute__((always_inline)) {
      constexpr bool SOFT = decltype(soft)::value, PV = decltype(pv)::value;
      constexpr int B = decltype(buf)::value;
      const uint32_t lane16 = 16 * lane_id<true>();
      i32x4 va[4], pb[2];
      if constexpr (PV) {
        const int any = *(const int LDS_AS*)at_lds(lds_at(&any_sh[0]) + 4 * was);
        pb[0] = *(const i32x4 LDS_AS*)at_lds(lds_at(p_sh) + lane16 + p_was);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint32_t at = (vr_at ^ (32 * d)) + v_was;
          const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)at_lds(at)));
          const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)at_lds(at + 16384)));
          va[d] = i32x4{lo[0], lo[1], hi[0], hi[1]};
        }
        if (__builtin_amdgcn_readfirstlane(any) == k - 1) {  // uniform, rare
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            if (__builtin_amdgcn_readfirstlane(moved_sh[was][r]) == k - 1) {  // uniform
              const float al = alpha_sh[was][r][lane_id<true>() & 15];
#pragma unroll
              for (int d = 0; d < 4; ++d) o[d][r] *= al;
            }
          }
        }
      }
      float top = 0.f, base = 0.f, alpha = 1.f, e[8];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if constexpr (PV) {
          if (r + 1 < RT) pb[(r + 1) & 1] = *(const i32x4 LDS_AS*)at_lds(lds_at(p_sh) + lane16 + p_was + (r + 1) * 1024);
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d][r] = mfma_bf16(va[d], pb[r & 1], o[d][r]);
        }
        if constexpr (SOFT) {
          if (r == 0) {
            // With PV, four of its MFMAs and the reads before them lie between: the empty asm keeps that order.
            if constexpr (PV)
              asm volatile("" : "+v"(s[0]), "+v"(s[1]), "+v"(o[0][0]), "+v"(o[1][0]), "+v"(o[2][0]), "+v"(o[3][0]));
            else
              settled(s);
            top = max3(max3(s[0][0], s[0][1], s[0][2]), max3(s[0][3], s[1][0], s[1][1]), max2(s[1][2], s[1][3]));
            const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = max2(__uint_as_float(x[0]), __uint_as_float(x[1]));
          } else if (r == 1) {
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = max2(__uint_as_float(x[0]), __uint_as_float(x[1])) * scale_log2;
          } else if (r == 2) {
            const float m_old = m_ref;
            m_ref = top > m_ref + kSlack ? top : m_ref;
            moved = __builtin_amdgcn_ballot_w64(m_ref != m_old) != 0;
            base = m_ref == -INFINITY ? 0.f : m_ref;
            if (moved) {  // uniform
              alpha = __builtin_amdgcn_exp2f((m_old == m_ref ? base : m_old) - base);
              l_rnd *= alpha;
              l_exact *= alpha;
              alpha_sh[B][wave][lane_id<true>() & 15] = alpha;
              moved_sh[B][wave] = k;
              any_sh[B] = k;
            }
          } else if (r == 3 || r == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) e[4 * (r - 3) + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r - 3][j], scale_log2, -base));
          } else if (r == 5) {
            const i32x4 w = {(int)pack_bf16(e[0], e[1]), (int)pack_bf16(e[2], e[3]), (int)pack_bf16(e[4], e[5]), (int)pack_bf16(e[6], e[7])};
            *(i32x4 LDS_AS*)at_lds(lds_at(p_sh) + lane16 + (B * RT + wave) * 1024) = w;
#pragma unroll
            for (int j = 0; j < 4; ++j) l_rnd = sum2_bf16((uint32_t)w[j], l_rnd);
          } else if (r == 6) {
            l_exact += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};

    f32x4 s[2];
    auto next_stage = [&](int k, auto buf) __attribute__((always_inline)) {
      copies_landed();
      lds_barrier();  // stage k is in LDS, P and V of stage k - 1 are; their buffers of stage k - 2 are free
      if (k + 1 < nst) copy_stage(k + 1, page_of(k + 1));
      scores(k, buf, s);
    };
    if (nst > 0) {
      constexpr std::integral_constant<int, 0> even{};
      constexpr std::integral_constant<int, 1> odd{};
      next_stage(0, even);
      weigh(yes, no, even, 0, 0, 0, 0, s);
#pragma unroll 1
      for (int k = 1; k < nst; k += 2) {
        next_stage(k, odd);
        weigh(yes, yes, odd, k, 0, 0, 0, s);
        if (k + 1 == nst) break;
        next_stage(k + 1, even);
        weigh(yes, yes, even, k + 1, RT * 1024, T * 1024, 1, s);
      }
    }
    const int lane = lane_id<true>(), g = lane >> 4, li = lane & 15;
    const float l = row_sum(l_rnd), x = row_sum(l_exact);
    sum_sh[wave][li] = l;
    lds_barrier();
    if (nst > 0) {
      const int was = (nst - 1) & 1;
      weigh(no, yes, std::integral_constant<int, 0>{}, nst, was * (RT * 1024), was * (T * 1024), was, s);
    }

    // ---- lse of row tile `wave`, and the output dims of all
    ArgParams& e = params_here();
    const int slot0 = e.splits[b];
    const bool single = e.splits[b + 1] - slot0 == 1;
    const int64_t slot = (int64_t)slot0 + split;
    write_lse(e, b, row0 + 16 * wave + li, g, slot, single, m_ref, x);
    if (single) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float sum = sum_sh[r][li], inv = sum == 0.f ? 0.f : 1.f / sum;
        const int row = row0 + 16 * r + li;
        if (row < e.rows) {
          const int sq = row / e.heads, h = row - sq * e.heads;
          uint16_t* dst = e.out + ((int64_t)b * e.o_sb + (int64_t)sq * e.o_ss + (int64_t)h * e.o_sh) + 64 * wave;
#pragma unroll
          for (int d = 0; d < 4; d += 2) {
            const f32x4 v = o[d][r] * inv, w = o[d + 1][r] * inv;
            store_dims(dst, d, g, i32x2{(int)pack_bf16(v[0], v[1]), (int)pack_bf16(v[2], v[3])},
                       i32x2{(int)pack_bf16(w[0], w[1]), (int)pack_bf16(w[2], w[3])});
          }
        }
      }
    } else {  // scaled fp16; a chunk of 128 dims is two waves' work
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float am = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) am = fmaxf(am, fabsf(o[d][r][j]));
        amax_sh[wave][r][li] = row_max(am);
      }
      lds_barrier();
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float sum = sum_sh[r][li], inv = sum == 0.f ? 0.f : 1.f / sum;
        const int ex = part_exp(fmaxf(amax_sh[wave][r][li], amax_sh[wave ^ 1][r][li]) * inv);
        const int row = row0 + 16 * r + li;
        if (row < e.rows) {
          uint16_t* dst = e.ws_o + (slot * e.rows + row) * kDV + 64 * wave;
#pragma unroll
          for (int d = 0; d < 4; d += 2) {
            const f32x4 v = (o[d][r] * inv) * exp2i(ex), w = (o[d + 1][r] * inv) * exp2i(ex);
            store_dims(dst, d, g, i32x2{(int)pack_f16(v[0], v[1]), (int)pack_f16(v[2], v[3])},
                       i32x2{(int)pack_f16(w[0], w[1]), (int)pack_f16(w[2], w[3])});
          }
          if (g == 0 && (wave & 1) == 0) e.ws_scale[(slot * e.rows + row) * 4 + (wave >> 1)] = exp2i(-ex);
        }
      }
    }
    lds_barrier();  // the sums are read before the next segment's
  }
}

// The schedule's parts are laid out for this many rows a workgroup.  Measured (us; 64 sequences x 4096 tokens, one
// token a sequence), with workgroups of 16, 64 and 128 rows:
//   heads   16: 27.7, 47.9, 63.1     32: 42.6, 50.6, 65.9     33: 61.6, 51.4, 66.8     64: 73.6, 56.7, 69.8
//           72: 94.2, 86.0, 70.2    128: 134,  90.2, 76.7    256: 263,  158,  128
// (32 rows a workgroup took 42.7 at 32 heads, 67.2 at 33 and 69.7 at 64: nowhere ahead, and is not kept.)
int rows_per_workgroup(int64_t rows) { return rows <= 32 ? 16 : rows <= 64 ? 64 : 128; }
int workgroups_per_cu(int R) { return R == 128 ? 1 : 2; }

template <int RT>
static hipError_t launch_rt(const DecodeParams& p, const int32_t* sched, int num_parts, hipStream_t st) {
  const int row_blocks = (p.rows + 16 * RT - 1) / (16 * RT);
  const dim3 grid((uint32_t)num_parts * (uint32_t)row_blocks);
  if (p.indices != nullptr)
    hipLaunchKernelGGL((mla_fp4_kernel<RT, true>), grid, dim3(256), 0, st, sched, row_blocks, num_parts, p);
  else
    hipLaunchKernelGGL((mla_fp4_kernel<RT, false>), grid, dim3(256), 0, st, sched, row_blocks, num_parts, p);
  return hipGetLastError();
}

static hipError_t launch_wide(const DecodeParams& p, const int32_t* sched, int num_parts, hipStream_t st) {
  const int row_blocks = (p.rows + 127) / 128;
  const dim3 grid((uint32_t)num_parts * (uint32_t)row_blocks);
  if (p.indices != nullptr)
    hipLaunchKernelGGL(mla_fp4_wide_kernel<true>, grid, dim3(512), 0, st, sched, row_blocks, num_parts, p);
  else
    hipLaunchKernelGGL(mla_fp4_wide_kernel<false>, grid, dim3(512), 0, st, sched, row_blocks, num_parts, p);
  return hipGetLastError();
}

hipError_t launch_decode(const DecodeParams& p, const int32_t* sched, int num_parts, int cus, hipStream_t st) {
  // Few pages: a part is one or two pages, and what a workgroup does before and after them counts, which is least
  // with 16 rows.  Measured (us, one token a sequence; 16 rows and the form for many pages, each with its schedule):
  //   128 heads: 1 sequence x 64 pages 15.0, 25.3    32 x 11 pages 23.4, 30.9    64 x 11 30.7, 36.7    64 x 22 52.5, 45.7
  //    64 heads: 1 x 64 12.0, 17.3    64 x 11 22.9, 29.9    64 x 22 32.8, 36.4      192 heads: 64 x 11 54.9, 44.0
  // Only with a schedule made for it: 16 rows with the other form's parts are more splits to merge than they save
  // (128 heads, 32 x 11 pages: 35.0); where a sequence is one page there are no splits, and any schedule will do, for
  // one round of workgroups, or two against the form of 128 rows: 64 sequences x 128 heads 11.0 (20.3), 64 x 256 17.9
  // (23.2), 64 x 64 8.2 (13.7), but 256 x 64 17.9 (16.5), 256 x 128 31.8 (27.0).
  const int most = p.indices != nullptr ? pages_of(p.topk) : p.bt_width;  // pages of a sequence
  const int64_t pages = (int64_t)p.batch * most;
  const int64_t tiles = (p.rows + 15) / 16;
  const int64_t round = 2 * cus;
  // A schedule of exactly as many parts as such a form's fill the GPU with was made for it, from the longest length; the
  // table may be as wide as the longest context that is allowed.  (The other forms' parts of such a schedule fill a
  // quarter: 32 x 11 pages x 128 heads in a table of 2048 columns 37.9, and 22.9 with 16 rows.)
  const bool made = num_parts * tiles <= round && num_parts == round / tiles;
  const bool few = made || (pages <= kFewPages / tiles &&
                            (num_parts * tiles <= round || (most <= 1 && pages * tiles <= (p.rows > 64 ? 2 : 1) * round)));
  const int R = few ? 16 : rows_per_workgroup(p.rows);
  if (R == 16) return launch_rt<1>(p, sched, num_parts, st);
  if (R == 64) return launch_rt<4>(p, sched, num_parts, st);
  return launch_wide(p, sched, num_parts, st);
}

}  // namespace mla4
