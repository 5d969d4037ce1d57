// mla_tree.hip -- decoding a tree of drafted tokens (gfx950): the plan of a step, the drafted tokens' part of the
// attention, which drafts the model agrees with, and the kept path's rows in the cache.
//
// A row (query token i of a sequence, head h) sees the sequence's whole prefix and, of the s_q <= 64 drafted tokens
// behind it, those whose bits its mask has.  The prefix is what the split-KV decode already does well, without any
// mask: it runs unchanged.  The drafted tokens are one more split of each sequence, at most 64 keys, which the kernel
// here scores under the masks; the combine merges it with the prefix's splits by their lse, as it merges those.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string>

#include "mla_decode_amd.h"
#include "mla_serving.h"
#include "mla_tree.h"

namespace mla_tree {

constexpr int kPage = MLA_PAGE_TOKENS;
constexpr int kDV = MLA_DIM_V;
constexpr int kKSteps = MLA_DIM_QK / 32;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((__vector_size__(4 * sizeof(short))));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((__vector_size__(8 * sizeof(__bf16))));
typedef _Float16 f16x8 __attribute__((__vector_size__(8 * sizeof(_Float16))));
#define LDS_AS __attribute__((address_space(3)))

template <bool F16>
__device__ __forceinline__ f32x4 mfma32(i32x4 a, i32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2 v = {a, b};
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
// What pack2 left of a and b.
template <bool F16>
__device__ __forceinline__ uint32_t pack2_rest(float a, float b, uint32_t w) {
  if constexpr (F16) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    return pack2<true>(a - (float)h[0], b - (float)h[1]);
  } else {
    return pack2<false>(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xFFFF0000u));
  }
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The exponent that brings a partial's chunk to [2^14, 2^15), as the split-KV decode stores its partials; the workspace
// keeps 2^-e, a normal number (a chunk below 2^-111 lands lower).
__device__ __forceinline__ int part_exp(float amax) {
  const int e = 15 - __builtin_amdgcn_frexp_expf(amax);
  return e < 126 ? e : 126;
}
__device__ __forceinline__ float group_max(float v) {  // over the four lane groups
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
// Whether any of eight 16-bit values is an infinity or a NaN.
template <bool F16>
__device__ __forceinline__ bool non_finite(i32x4 v) {
  constexpr uint32_t kHi = F16 ? 0x7C000000u : 0x7F800000u, kLo = kHi >> 16;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (uint32_t)v[j];
    bad |= (w & kHi) == kHi || (w & kLo) == kLo;
  }
  return bad;
}

// ---------------------------------------------------------------------------------------
// one tile of keys
// ---------------------------------------------------------------------------------------
// A workgroup scores rows of a sequence against one tile of up to 64 keys, its drafted tokens or a page of its prefix,
// and leaves a partial: S^T = K Q^T (16x16x32 MFMA), softmax over the visible keys, O^T = V^T P^T with V^T from
// transposed LDS reads.  All keys are in the tile, so the softmax is one pass.
//
// P goes as two 16-bit halves, its rounding and the rest, in two products beside the same V: 16 bits and more of each weight
// (one half alone: 0.1 to 0.4 us less of 17 to 27, and outputs 20% further off).  A partial output is fp16 with a power of two
// per 128 dims, half of fp32's bytes to write and merge, as the split-KV pass writes the partials that these are merged
// with; that pass rounds P to one half.  Scores, maxima, sums and lse are fp32.  Error of a chain of 5 behind 300 tokens against
// 64 bits, of the outputs' norm: pages by themselves bf16 1.7e-3, fp16 2.8e-4; behind the pass 2.1e-3, 3.3e-4, as the causal decode;
// the exact result rounded once 1.7e-3, 2.1e-4.
//
// Tokens and queries are read row by row, a wave's lanes side by side, and become operands through LDS.  Loaded in operand
// order, 16 rows a quarter wave, each load took the address unit 64 cycles instead of 16: 36 of them 4.2 us.
//
// A drafted token that a row does not see must not reach it, whatever its cache row holds (it may never have been
// written): a weight of 0 times an infinity or a NaN is a NaN.  A token whose latent holds one is zeroed in part,
// remembered, and the rows that do see it become NaN.
constexpr int kPitch = 2 * MLA_DIM_QK + 16;  // bytes of a row in LDS: 16 rows start on 16 different groups of 4 banks
constexpr int kTileBytes = 16 * kPitch;      // 16 rows

// What a lane holds of a wave's share of the tokens, 16 bytes a load whatever the format: of one token 8 dims, of
// two 16 (e4m3) or of four 32 (e2m1).
template <int FMT>
struct Lanes {
  static constexpr int kTokens = FMT == MLA_KV_NATIVE ? 1 : FMT == MLA_KV_FP8_E4M3 ? 2 : 4;  // of a load
  static constexpr int kLanes = 64 / kTokens;                                               // of a token
};
// 8 u .. 8 u + 7 of the dims that a lane holds; coded caches widen to bf16, exactly.
template <int FMT>
__device__ __forceinline__ i32x4 widen8(i32x4 raw, float sc, int u) {
  if constexpr (FMT == MLA_KV_FP8_E4M3) {
    const int a = raw[2 * u], b = raw[2 * u + 1];
    return i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, true)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, true))};
  } else if constexpr (FMT == MLA_KV_FP4_E2M1) {
    const int w = raw[u];
    return i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3))};
  } else {
    return raw;
  }
}

// A prefix's splits where every page is one: an empty prefix has an empty one (the merge passes over sequences of one split).
__device__ __forceinline__ int page_splits(int tokens) { return tokens > 0 ? (tokens + kPage - 1) / kPage : 1; }

// The tile of a workgroup; grid (row blocks, tiles, batch): tile 0 is the drafted tokens; with `pages`, tile 1 + i is page
// i of the prefix.
struct Tile {
  bool drafts;
  int held;       // keys
  int at;         // the first one's row in the first page
  int pages[2];   // 64 keys lie in one page or two
  uint64_t known; // bits of the keys
  int prefix_raw, prefix, cap;
};
// False where the sequence has no such tile.
__device__ __forceinline__ bool find_tile(const TreeParams& p, int b, int tile, Tile& t) {
  t.drafts = tile == 0;
  t.cap = p.bt_width * kPage;
  const int raw = p.prefix[b];
  t.prefix_raw = raw > 0 ? raw : 0;
  t.prefix = t.prefix_raw < t.cap ? t.prefix_raw : t.cap;
  if (!t.drafts && tile > page_splits(t.prefix)) return false;
  const int64_t room = (int64_t)t.cap - t.prefix_raw;  // of the table's row, for drafted tokens
  t.at = t.drafts ? t.prefix_raw & (kPage - 1) : 0;
  t.held = !t.drafts ? min(t.prefix - (tile - 1) * kPage, kPage) : room < 0 ? 0 : room < p.s_q ? (int)room : p.s_q;
  t.known = t.held >= 64 ? ~0ull : (1ull << t.held) - 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int col = (t.drafts ? t.prefix_raw / kPage : tile - 1) + i;
    col = col < p.bt_width ? col : p.bt_width - 1;
    const int id = p.block_table[(int64_t)b * p.bt_stride + col];
    t.pages[i] = id < 0 ? 0 : id < p.num_blocks ? id : p.num_blocks - 1;
  }
  return true;
}

// The tile's slot; the drafted tokens' workgroup also writes what the merge (and the split-KV pass) are told.
__device__ __forceinline__ int find_slot(const TreeParams& p, int b, int tile, const Tile& t, int lane) {
  int slot;
  if (p.pages) {  // uniform: every page a split, in order, then the drafted tokens
    int before = 0;
    for (int i = lane; i < b; i += 64) {
      const int n = p.prefix[i];
      before += 1 + page_splits(n < t.cap ? n : t.cap);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d);
    slot = __builtin_amdgcn_readfirstlane(before) + (t.drafts ? page_splits(t.prefix) : tile - 1);
  } else {
    slot = p.splits[b + 1] + b;  // one more split for this sequence and each before it
  }
  if (t.drafts && blockIdx.x == 0 && threadIdx.x == 0) {
    if (b == 0) p.splits_out[0] = p.pages ? 0 : p.splits[0];
    p.splits_out[b + 1] = slot + 1;
    if (p.pages && t.prefix_raw > t.cap && p.status != nullptr) *p.status = 1;
  }
  return slot;
}

// N tokens first, first + 1, .. of the tile (rows past its keys as zeros): their latents, the coded ones' scales, and the
// rope dims, 8 tokens a register.
template <int FMT, int N>
struct Share {
  static constexpr int kLoads = N / Lanes<FMT>::kTokens;
  i32x4 v[kLoads], r[N / 8];
  float sc[FMT == MLA_KV_NATIVE ? 1 : kLoads];
};
template <int FMT, int N>
__device__ __forceinline__ void load_tokens(const TreeParams& p, const Tile& t, int first, int lane, Share<FMT, N>& x) {
  constexpr int kTokens = Lanes<FMT>::kTokens, kLanes = Lanes<FMT>::kLanes;
#pragma unroll
  for (int i = 0; i < N / kTokens; ++i) {
    const int j = first + kTokens * i + (kTokens > 1 ? lane / kLanes : 0);  // 16-bit caches: uniform
    x.v[i] = i32x4{0, 0, 0, 0};
    if constexpr (FMT != MLA_KV_NATIVE) x.sc[i] = 1.f;
    if (j < t.held) {
      const int64_t page = t.at + j < kPage ? t.pages[0] : t.pages[1];
      const int row = (t.at + j) & (kPage - 1), piece = lane % kLanes;
      x.v[i] = *(const i32x4*)(p.nope + page * p.sp + row * p.st + 16 * piece);
      if constexpr (FMT == MLA_KV_FP8_E4M3)
        x.sc[i] = *(const float*)(p.scale + page * p.cp + (piece >> 3) * p.ct + 4 * row);
      else if constexpr (FMT == MLA_KV_FP4_E2M1)
        x.sc[i] = __uint_as_float((uint32_t)p.scale[page * p.cp + row * p.ct + piece] << 23);
    }
  }
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    const int j = first + 8 * i + (lane >> 3);
    x.r[i] = i32x4{0, 0, 0, 0};
    if (j < t.held) {
      const int64_t page = t.at + j < kPage ? t.pages[0] : t.pages[1];
      x.r[i] = *(const i32x4*)(p.rope + page * p.rp + ((t.at + j) & (kPage - 1)) * p.rt + 16 * (lane & 7));
    }
  }
}
// The same to rows of LDS.  Of drafted tokens, what is not finite is left out; bits of such tokens come back.
template <int FMT, bool F16, int N>
__device__ __forceinline__ uint32_t put_tokens(uint8_t* dst, bool drafts, int lane, const Share<FMT, N>& x) {
  constexpr int kTokens = Lanes<FMT>::kTokens, kLanes = Lanes<FMT>::kLanes;
  uint32_t spoilt = 0;
#pragma unroll
  for (int i = 0; i < N / kTokens; ++i) {
    uint8_t* row = dst + (kTokens * i + lane / kLanes) * kPitch + 16 * kTokens * (lane % kLanes);
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      i32x4 v = widen8<FMT>(x.v[i], FMT == MLA_KV_NATIVE ? 0.f : x.sc[FMT == MLA_KV_NATIVE ? 0 : i], u);
      if (drafts) {  // uniform
        const bool bad = non_finite<F16>(v);
        const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
        if (any != 0) {  // uniform, rare
          if (bad) v = i32x4{0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < kTokens; ++w) spoilt |= (uint32_t)((any >> (w * kLanes) << (64 - kLanes)) != 0) << (kTokens * i + w);
        }
      }
      *(i32x4*)(row + 16 * u) = v;
    }
  }
#pragma unroll
  for (int i = 0; i < N / 8; ++i) *(i32x4*)(dst + (8 * i + (lane >> 3)) * kPitch + 2 * kDV + 16 * (lane & 7)) = x.r[i];
  return spoilt;
}
// Rows first .. of the queries (past the last: the last), alike.
template <int N>
__device__ __forceinline__ void load_queries(const TreeParams& p, int b, int first, int lane, i32x4 (&v)[N], i32x4 (&r)[(N + 7) / 8]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int row = first + i < p.rows ? first + i : p.rows - 1;  // uniform
    const int s = row / p.heads, h = row - s * p.heads;
    v[i] = *(const i32x4*)(p.q_nope + (b * p.q_sb + s * p.q_ss + h * p.q_sh) + 8 * lane);
  }
#pragma unroll
  for (int i = 0; i < (N + 7) / 8; ++i) {
    const int j = first + 8 * i + ((lane >> 3) & (N < 8 ? N - 1 : 7));
    const int row = j < p.rows ? j : p.rows - 1;
    const int s = row / p.heads, h = row - s * p.heads;
    r[i] = *(const i32x4*)(p.q_rope + (b * p.qr_sb + s * p.qr_ss + h * p.qr_sh) + 8 * (lane & 7));
  }
}
template <int N>
__device__ __forceinline__ void put_queries(uint8_t* dst, int lane, const i32x4 (&v)[N], const i32x4 (&r)[(N + 7) / 8]) {
#pragma unroll
  for (int i = 0; i < N; ++i) *(i32x4*)(dst + i * kPitch + 16 * lane) = v[i];
#pragma unroll
  for (int i = 0; i < (N + 7) / 8; ++i)
    if (N >= 8 || lane < 8 * N) *(i32x4*)(dst + (8 * i + (lane >> 3)) * kPitch + 2 * kDV + 16 * (lane & 7)) = r[i];
}
// Fragments of 16 rows: lane (g, i) holds dims 32 kk + 8 g .. +7 of row i.
__device__ __forceinline__ void read_fragments(const uint8_t* src, int g, int li, i32x4 (&f)[kKSteps]) {
#pragma unroll
  for (int kk = 0; kk < kKSteps; ++kk) f[kk] = *(const i32x4*)(src + li * kPitch + 64 * kk + 16 * g);
}
// V^T (A operand): transposed reads give lane (g, i) keys 4 g .. +3 and 16 + 4 g .. +3 of 32 at dim 16 d + i.
__device__ __forceinline__ i32x4 read_vt(const uint8_t* rows32, int d, int g, int li) {
  const uint8_t LDS_AS* a = (const uint8_t LDS_AS*)(rows32 + (4 * g + (li >> 2)) * kPitch + 32 * d + 8 * (li & 3));
  const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)a));
  const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)(a + kTileBytes)));
  return i32x4{lo[0], lo[1], hi[0], hi[1]};
}

__device__ __forceinline__ float largest(f32x4 v, float a) {
  return fmaxf(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))), a);
}
// A row's divisor and lse.  A NaN in the lse makes the merged one -inf, as any NaN row's is.
__device__ __forceinline__ void finish_row(bool spoilt, float l, float ref, float& inv, float& lse2) {
  const float nan = __builtin_nanf("");
  inv = spoilt ? nan : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  lse2 = spoilt ? nan : l > 0.f ? ref + __log2f(l) : l == 0.f ? -INFINITY : l;
}

// The rows of one 128-dim chunk on their way out: 16 rows of 256 bytes in LDS, 16-byte pieces swizzled by the row, so
// that a store writes four rows' whole chunks (fragments stored directly write pieces of 32 bytes of 16 rows).
__device__ __forceinline__ void stage_chunk(uint8_t* stage, int d, int g, int li, f32x4 x) {
  *(i32x2*)(stage + li * 256 + (((2 * d + (g >> 1)) ^ li) << 4) + 8 * (g & 1)) =
      i32x2{(int)pack2<true>(x[0], x[1]), (int)pack2<true>(x[2], x[3])};
}
__device__ __forceinline__ void store_chunk(const TreeParams& p, const uint8_t* stage, int64_t slot, int first, int chunk, int g, int li) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 4 * j + g;
    const i32x4 x = *(const i32x4*)(stage + r * 256 + ((li ^ r) << 4));
    if (first + r < p.rows) *(i32x4*)(p.ws_o + (slot * p.rows + first + r) * kDV + 128 * chunk + 8 * li) = x;
  }
}

// 64 rows, a wave 16 of them: few synchronisations, for many rows.  The waves read their own 16 queries and a quarter of
// the keys; the queries become operands in the place that the keys take afterwards.  Drafted tokens alone are bound by latency
// (length, table, tokens, LDS, products, store, one after the other): 32 x 256 rows 12 us (fp8), 8 x 4096 rows 19 us (bf16, 71 MB
// in and out, 3.7 TB/s).
template <int FMT, bool F16, int KT>
__global__ __launch_bounds__(256, 2) void mla_tree_rows_kernel(TreeParams p) {
  constexpr int kTok = 32 * KT, kShare = kTok / 4;
  __shared__ __attribute__((aligned(16))) uint8_t kv_sh[4 * kTileBytes];
  __shared__ uint32_t spoilt_sh[4];
  const int b = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, li = lane & 15;
  const int first = blockIdx.x * 64 + 16 * wave;
  i32x4 q[kKSteps];
  Share<FMT, kShare> x;
  Tile t;
  {
    i32x4 qv[16], qr[2];
    load_queries<16>(p, b, first, lane, qv, qr);
    if (!find_tile(p, b, blockIdx.y, t)) return;
    load_tokens(p, t, wave * kShare, lane, x);
    put_queries<16>(kv_sh + wave * kTileBytes, lane, qv, qr);
  }
  __builtin_amdgcn_wave_barrier();  // the wave's own rows: LDS runs its accesses in order
  read_fragments(kv_sh + wave * kTileBytes, g, li, q);
  const int row_raw = first + li;
  const int row = row_raw < p.rows ? row_raw : p.rows - 1;
  uint64_t mask = t.known;
  if (t.drafts) {  // uniform
    const uint64_t nodes = p.s_q == 64 ? ~0ull : (1ull << p.s_q) - 1;
    mask = p.mask[(int64_t)b * p.s_q + row / p.heads];
    if ((mask & nodes & ~t.known) != 0 && p.status != nullptr) *p.status = 1;
    mask &= t.known;
  }
  const int64_t slot = find_slot(p, b, blockIdx.y, t, lane);
  __syncthreads();  // the queries are read
  spoilt_sh[wave] = put_tokens<FMT, F16, kShare>(kv_sh + wave * kShare * kPitch, t.drafts, lane, x);
  __syncthreads();
  uint64_t spoilt = 0;
  if (t.drafts)
#pragma unroll
    for (int w = 0; w < 4; ++w) spoilt |= (uint64_t)spoilt_sh[w] << (w * kShare);

  // S^T: lane (g, i) gets keys 16 u + 4 g .. +3 of row i
  f32x4 sc[2 * KT];
#pragma unroll
  for (int u = 0; u < 2 * KT; ++u) {
    const uint8_t* k = kv_sh + (16 * u + li) * kPitch + 16 * g;
    sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < kKSteps; ++kk) sc[u] = mfma32<F16>(*(const i32x4*)(k + 64 * kk), q[kk], sc[u]);
  }
  float mx = -INFINITY;
#pragma unroll
  for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool seen = (mask >> (16 * u + 4 * g + i)) & 1;
      sc[u][i] = seen ? sc[u][i] * p.scale_log2 : -INFINITY;
      mx = fmaxf(mx, sc[u][i]);
    }
  mx = group_max(mx);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  i32x4 pb[KT], pr[KT];  // P^T as it is: the B operand in the key order of the transposed reads, and its rest
#pragma unroll
  for (int u = 0; u < 2 * KT; ++u) {
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = __builtin_amdgcn_exp2f(sc[u][i] - ref);
      l += e[i];
    }
    const uint32_t w0 = pack2<F16>(e[0], e[1]), w1 = pack2<F16>(e[2], e[3]);
    pb[u >> 1][2 * (u & 1)] = (int)w0;
    pb[u >> 1][2 * (u & 1) + 1] = (int)w1;
    pr[u >> 1][2 * (u & 1)] = (int)pack2_rest<F16>(e[0], e[1], w0);
    pr[u >> 1][2 * (u & 1) + 1] = (int)pack2_rest<F16>(e[2], e[3], w1);
  }
  f32x4 o[kDV / 16];
#pragma unroll
  for (int d = 0; d < kDV / 16; ++d) {
    o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < KT; ++u) {
      const i32x4 vt = read_vt(kv_sh + 2 * u * kTileBytes, d, g, li);
      o[d] = mfma32<F16>(vt, pb[u], o[d]);
      o[d] = mfma32<F16>(vt, pr[u], o[d]);
    }
  }
  float inv, lse2;
  finish_row((mask & spoilt) != 0, group_sum(l), mx, inv, lse2);
  __syncthreads();  // V is read: its place takes the rows on their way out
  uint8_t* stage = kv_sh + wave * kTileBytes;  // 4 KiB a chunk
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float a = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) a = largest(o[8 * c + d], a);
    const int e = part_exp(group_max(a * inv));
#pragma unroll
    for (int d = 0; d < 8; ++d) stage_chunk(stage + 4096 * c, d, g, li, (o[8 * c + d] * inv) * exp2i(e));
    if (g == c && row_raw < p.rows) p.ws_scale[(slot * p.rows + row) * 4 + c] = exp2i(-e);
  }
  if (g == 0 && row_raw < p.rows) p.ws_lse[slot * p.rows + row] = lse2;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int c = 0; c < 4; ++c) store_chunk(p, stage + 4096 * c, slot, first, c, g, li);
}

// 16 rows: wave w scores keys 16 w .. +15 and owns dims 128 w .. +127 of the output; the row maximum and P^T cross the
// waves through LDS.  The work of a tile in a quarter of the time, for few rows: 33 tiles of 64 keys x 128 rows 10.5 us.
template <int FMT, bool F16>
__global__ __launch_bounds__(256, 2) void mla_tree_keys_kernel(TreeParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t kv_sh[4 * kTileBytes];
  __shared__ __attribute__((aligned(16))) uint8_t p_sh[2][2][1024];  // P^T, and its rest
  __shared__ float max_sh[4][16], sum_sh[4][16];
  __shared__ uint32_t spoilt_sh[4];
  const int b = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, li = lane & 15;
  const int first = blockIdx.x * 16;
  Share<FMT, 16> x;
  Tile t;
  {
    i32x4 qv[4], qr[1];
    load_queries<4>(p, b, first + 4 * wave, lane, qv, qr);
    if (!find_tile(p, b, blockIdx.y, t)) return;
    load_tokens(p, t, 16 * wave, lane, x);
    put_queries<4>(kv_sh + 4 * wave * kPitch, lane, qv, qr);
  }
  const int row_raw = first + li;
  const int row = row_raw < p.rows ? row_raw : p.rows - 1;
  uint64_t mask = t.known;
  if (t.drafts) {  // uniform
    const uint64_t nodes = p.s_q == 64 ? ~0ull : (1ull << p.s_q) - 1;
    mask = p.mask[(int64_t)b * p.s_q + row / p.heads];
    if ((mask & nodes & ~t.known) != 0 && p.status != nullptr) *p.status = 1;
    mask &= t.known;
  }
  const int64_t slot = find_slot(p, b, blockIdx.y, t, lane);
  __syncthreads();
  i32x4 q[kKSteps], k[kKSteps];
  read_fragments(kv_sh, g, li, q);
  __syncthreads();  // the queries are read
  spoilt_sh[wave] = put_tokens<FMT, F16, 16>(kv_sh + wave * kTileBytes, t.drafts, lane, x);
  __builtin_amdgcn_wave_barrier();  // the wave's own rows: LDS runs its accesses in order
  read_fragments(kv_sh + wave * kTileBytes, g, li, k);
  f32x4 even = {0.f, 0.f, 0.f, 0.f}, odd = even;
#pragma unroll
  for (int kk = 0; kk < kKSteps; kk += 2) {
    even = mfma32<F16>(k[kk], q[kk], even);
    odd = mfma32<F16>(k[kk + 1], q[kk + 1], odd);
  }
  float sc[4], mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool seen = (mask >> (16 * wave + 4 * g + i)) & 1;
    sc[i] = seen ? (even[i] + odd[i]) * p.scale_log2 : -INFINITY;
    mx = fmaxf(mx, sc[i]);
  }
  max_sh[wave][li] = group_max(mx);  // four lane groups, one value
  __syncthreads();
  mx = fmaxf(fmaxf(max_sh[0][li], max_sh[1][li]), fmaxf(max_sh[2][li], max_sh[3][li]));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float e[4], l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e[i] = __builtin_amdgcn_exp2f(sc[i] - ref);
    l += e[i];
  }
  // P^T as it is: half of the B operand of 32 keys in the order of the transposed reads
  const uint32_t w0 = pack2<F16>(e[0], e[1]), w1 = pack2<F16>(e[2], e[3]);
  *(i32x2*)&p_sh[0][wave >> 1][16 * lane + 8 * (wave & 1)] = i32x2{(int)w0, (int)w1};
  *(i32x2*)&p_sh[1][wave >> 1][16 * lane + 8 * (wave & 1)] =
      i32x2{(int)pack2_rest<F16>(e[0], e[1], w0), (int)pack2_rest<F16>(e[2], e[3], w1)};
  sum_sh[wave][li] = group_sum(l);
  __syncthreads();
  const i32x4 pb[2] = {*(const i32x4*)&p_sh[0][0][16 * lane], *(const i32x4*)&p_sh[0][1][16 * lane]};
  const i32x4 pr[2] = {*(const i32x4*)&p_sh[1][0][16 * lane], *(const i32x4*)&p_sh[1][1][16 * lane]};
  f32x4 o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const i32x4 vt = read_vt(kv_sh + 2 * u * kTileBytes, 8 * wave + d, g, li);
      o[d] = mfma32<F16>(vt, pb[u], o[d]);
      o[d] = mfma32<F16>(vt, pr[u], o[d]);
    }
  }
  uint64_t spoilt = 0;
  if (t.drafts)
#pragma unroll
    for (int w = 0; w < 4; ++w) spoilt |= (uint64_t)spoilt_sh[w] << (16 * w);
  float inv, lse2;
  finish_row((mask & spoilt) != 0, sum_sh[0][li] + sum_sh[1][li] + sum_sh[2][li] + sum_sh[3][li], mx, inv, lse2);
  float a = 0.f;
#pragma unroll
  for (int d = 0; d < 8; ++d) a = largest(o[d], a);
  const int ex = part_exp(group_max(a * inv));
  __syncthreads();  // V is read: its place takes the rows on their way out
  uint8_t* stage = kv_sh + 4096 * wave;
#pragma unroll
  for (int d = 0; d < 8; ++d) stage_chunk(stage, d, g, li, (o[d] * inv) * exp2i(ex));
  if (g == 0 && row_raw < p.rows) {
    p.ws_scale[(slot * p.rows + row) * 4 + wave] = exp2i(-ex);
    if (wave == 0) p.ws_lse[slot * p.rows + row] = lse2;
  }
  __builtin_amdgcn_wave_barrier();
  store_chunk(p, stage, slot, first, wave, g, li);
}

// Whether the prefixes' pages are tiles of the launch too, each its own split, instead of parts of the split-KV pass: where
// they are few the pass is mostly start and end, a launch more, and wants a schedule.  By tiles of 16 rows x pages (the
// table's width for all sequences; `slots`: what the workspace has), the whole decode in us, the pass -> pages:
//   bf16  264 34.6 -> 14.7    528 36.2 -> 19.9    1056 41.7 -> 27.6    1152 31.6 -> 25.3    2112 41.4 -> 38.3, 44.1 -> 37.6
//   fp8   264 36.5 -> 14.4    528 37.6 -> 19.7    1056 43.3 -> 28.2    1152 31.2 -> 24.5    2112 42.9 -> 37.3, 46.2 -> 39.3
//   fp4   264 19.9 -> 14.9    528 23.3 -> 20.0    640 23.0 -> 23.6 (a form for few pages of its own)
bool takes_pages(int64_t batch, int64_t rows, int format, int64_t bt_width, int64_t slots, int cus) {
  const int64_t tiles = (rows + 15) / 16 * batch * bt_width;
  return batch * (bt_width + 1) <= slots && 4 * tiles <= (format == MLA_KV_FP4_E2M1 ? 9 : 36) * (int64_t)cus;
}

// 16 rows a workgroup where there are few tiles for the CUs, else 64; the whole decode in us, 16 -> 64 (bf16):
//   72 tiles 12.0 -> 15.5    136 12.4 -> 15.6    264 (272 with the drafted tokens') 14.7 -> 17.1    256 47.6 -> 48.7
//   512 56.0 -> 56.0    528 22.0 -> 20.3    640 73.2 -> 70.5    1024 78.5 -> 73.2    2048 124 -> 108    4096 194 -> 160
template <int FMT, bool F16>
static void launch_format(const TreeParams& p, int cus, hipStream_t st) {
  const int64_t rows16 = (p.rows + 15) / 16;
  const int tiles = p.pages ? 1 + p.bt_width : 1;
  const bool few = 4 * rows16 * tiles * p.batch <= 5 * (int64_t)cus;
  const dim3 grid((uint32_t)(few ? rows16 : (rows16 + 3) / 4), tiles, p.batch);
  if (few)
    hipLaunchKernelGGL((mla_tree_keys_kernel<FMT, F16>), grid, dim3(256), 0, st, p);
  else if (!p.pages && p.s_q <= 32)
    hipLaunchKernelGGL((mla_tree_rows_kernel<FMT, F16, 1>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((mla_tree_rows_kernel<FMT, F16, 2>), grid, dim3(256), 0, st, p);
}

hipError_t launch_tiles(const TreeParams& p, int cus, hipStream_t st) {
  if (p.format == MLA_KV_FP8_E4M3) launch_format<MLA_KV_FP8_E4M3, false>(p, cus, st);
  else if (p.format == MLA_KV_FP4_E2M1) launch_format<MLA_KV_FP4_E2M1, false>(p, cus, st);
  else if (p.f16) launch_format<MLA_KV_NATIVE, true>(p, cus, st);
  else launch_format<MLA_KV_NATIVE, false>(p, cus, st);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// plan: parents -> masks, positions, cache rows, prefix lengths
// ---------------------------------------------------------------------------------------
// A wave a sequence, a lane a node.  A node's mask is its own bit and its parent's mask.  Each of six rounds takes
// over the mask of the node that the lane points at and then points where that one does: 2, 4, .. 64 generations.
// Bound by latency: two loads, six rounds of lane reads, a table lookup: 128 trees of 16 nodes 2.7 us,
// 4096 of them 3.2.
struct PlanParams {
  const int32_t* parents;
  const int32_t* seqlens;
  const int32_t* tree_lens;  // may be NULL: s_q each
  const int32_t* block_table;
  int32_t bt_stride, bt_width, batch, s_q;
  uint64_t* mask;
  int32_t* positions;
  int32_t* slots;
  int32_t* prefix;
};

__global__ __launch_bounds__(256) void mla_tree_plan_kernel(PlanParams p) {
  const int b = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (b >= p.batch) return;
  const int L = p.seqlens[b];
  int n = p.s_q;
  if (p.tree_lens != nullptr) {
    const int m = p.tree_lens[b];
    n = m < 0 ? 0 : m < n ? m : n;
  }
  const bool fits = L >= n;  // a sequence shorter than its tree holds none of it
  const int prefix = fits ? L - n : 0;
  const bool in = lane < p.s_q;
  int up = in ? p.parents[(int64_t)b * p.s_q + lane] : -2;
  bool dead = !fits || lane >= n || up < -1 || up >= lane;
  if (dead) up = -1;
  uint64_t mask = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int from = up < 0 ? lane : up;
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)mask, from), hi = (uint32_t)__shfl((int)(mask >> 32), from);
    const int next = __shfl((up + 1) | (dead ? 128 : 0), from);  // the node's pointer + 1, and whether it is dead
    mask |= (uint64_t)hi << 32 | lo;
    dead |= (next & 128) != 0;
    up = up < 0 ? -1 : (next & 127) - 1;
  }
  if (lane == 0) p.prefix[b] = prefix;
  if (!in) return;
  const int64_t at = (int64_t)b * p.s_q + lane;
  int slot = -1;
  const int64_t pos = (int64_t)prefix + lane;
  if (fits && lane < n && pos / kPage < p.bt_width) {
    const int page = p.block_table[(int64_t)b * p.bt_stride + pos / kPage];
    if (page >= 0 && page < INT32_MAX / kPage) slot = page * kPage + (int)(pos % kPage);
  }
  p.mask[at] = dead ? 0 : mask;
  p.positions[at] = dead ? -1 : prefix + __builtin_popcountll(mask) - 1;
  p.slots[at] = slot;
}

// ---------------------------------------------------------------------------------------
// accept: the drafted path that the model agrees with
// ---------------------------------------------------------------------------------------
// A wave a sequence, a lane a node.  From node 0 on, the walk goes to the lowest child whose token is the one the model
// chose after the node: a ballot a step.  A child of `cur` is a node whose mask is cur's and its own bit.
// Bound by latency: 128 trees of 16 nodes 2.3 us, a launch.
struct AcceptParams {
  const uint64_t* mask;
  const int32_t* prefix;
  const void* tokens;
  const void* targets;
  int32_t batch, s_q;
  int32_t* path;
  int32_t* counts;
  void* next;
  int32_t* keep_lens;
};

template <class T>
__global__ __launch_bounds__(256) void mla_tree_accept_kernel(AcceptParams p) {
  const int b = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (b >= p.batch) return;
  const int64_t at = (int64_t)b * p.s_q + lane;
  const bool in = lane < p.s_q;
  const uint64_t mask = in ? p.mask[at] : 0;
  const T token = in ? ((const T*)p.tokens)[at] : 0;
  const T target = in ? ((const T*)p.targets)[at] : 0;
  const uint64_t own = 1ull << lane;
  const bool alive = (mask & own) != 0;
  auto lane_of = [](uint64_t v, int l) __attribute__((always_inline)) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
  };
  int count = 0, place = -1;  // place: the lane's entry of the path
  T after = -1;
  const int root = __builtin_amdgcn_readfirstlane(mask == 1ull ? 1 : 0);  // node 0 sees itself alone
  if (root) {
    int cur = 0;
    do {  // every step goes to a higher node
      if (lane == count) place = cur;
      ++count;
      const uint64_t line = lane_of(mask, cur);
      after = (T)lane_of((uint64_t)target, cur);
      const uint64_t next = __builtin_amdgcn_ballot_w64(alive && lane > cur && mask == (line | own) && token == after);
      cur = next ? __builtin_ctzll(next) : -1;
    } while (cur >= 0);
  }
  if (in) p.path[at] = place;
  if (lane == 0) {
    p.counts[b] = count;
    ((T*)p.next)[b] = after;
    p.keep_lens[b] = p.prefix[b] + count;
  }
}

// ---------------------------------------------------------------------------------------
// keep: the path's rows together
// ---------------------------------------------------------------------------------------
// Row slots[k] <- row slots[path[k]] for the entries of the path, as if all were read before any is written.  A thread
// takes one 16-byte piece of the rows (4 bytes of the fp8 cache's scales) and walks the path in order, 16 rows
// read ahead of their writes.  No read can meet an earlier write: an entry is at least its own place (others are
// passed over), so the rows written before it lie below the one that it reads.  Lane k of each wave holds entry k, its
// row and that of path[k]: what a round moves is known without another load.  Bound by latency, a read and a write per 16
// rows: 128 sequences that move 15 rows each 3.9 us (bf16; with the rows' indices loaded for every item 8.6, and in the
// fp8 cache, whose parts went one after the other, 21.7 -> 3.7), 256 that move 63 10.9 us (32.1); 4096 that move 15 24 us
// (5.9 TB/s: the 140 MB stay in the last-level cache; a copy past it makes 4.8).
struct KeepParams {
  uint8_t* nope;
  uint8_t* rope;
  uint8_t* scale;
  int64_t sp, st, rp, rt, cp, ct;
  int64_t tokens;
  const int32_t* slots;
  const int32_t* path;
  int32_t s_q, format;
};

// The next N moves, all read, then all written; where fewer are left, the last of them again, the same bytes (a branch an
// item would have each write wait for the one before it).  from, to: lane k's rows.  The strides are the thread's own; the
// moves are uniform.
template <class V, int N>
__device__ __forceinline__ uint64_t keep_some(uint8_t* base, int64_t page_stride, int64_t row_stride, int from, int to, uint64_t moves) {
  V v[N];
  uint8_t* dst[N];
  int k = 0;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    k = moves ? __builtin_ctzll(moves) : k;
    moves &= moves - 1;
    const int i = __builtin_amdgcn_readlane(from, k), o = __builtin_amdgcn_readlane(to, k);
    v[u] = *(const V*)(base + i / kPage * page_stride + i % kPage * row_stride);
    dst[u] = base + o / kPage * page_stride + o % kPage * row_stride;
  }
#pragma unroll
  for (int u = 0; u < N; ++u) *(V*)dst[u] = v[u];
  return moves;
}
template <class V>
__device__ __forceinline__ void keep_pieces(uint8_t* base, int64_t page_stride, int64_t row_stride, int from, int to, uint64_t moves) {
  while (__builtin_popcountll(moves) > 4) moves = keep_some<V, 16>(base, page_stride, row_stride, from, to, moves);
  if (moves) keep_some<V, 4>(base, page_stride, row_stride, from, to, moves);
}

__global__ __launch_bounds__(128) void mla_keep_path_kernel(KeepParams p) {
  const int t = threadIdx.x, lane = t & 63;
  const int64_t at = (int64_t)blockIdx.x * p.s_q + lane;
  const bool in = lane < p.s_q;
  const int slot = in ? p.slots[at] : -1, j = in ? p.path[at] : -1;
  const bool goes = j > lane && j < p.s_q;
  const int from = __shfl(slot, goes ? j : lane);
  const bool moved = goes && slot >= 0 && from >= 0 && slot < p.tokens && from < p.tokens;
  const uint64_t moves = __builtin_amdgcn_ballot_w64(moved);
  const int pieces = p.format == MLA_KV_NATIVE ? 64 : p.format == MLA_KV_FP8_E4M3 ? 32 : 16;  // of the latent
  if (p.format == MLA_KV_FP8_E4M3 && t >= 64) {
    if (t < 68) keep_pieces<int32_t>(p.scale + (t - 64) * p.ct, p.cp, 4, from, slot, moves);
    return;
  }
  uint8_t* base = p.nope + 16 * t;
  int64_t page_stride = p.sp, row_stride = p.st;
  if (t >= pieces) {
    base = p.rope + 16 * (t - pieces);
    page_stride = p.rp;
    row_stride = p.rt;
  }
  if (t >= pieces + 8) {
    base = p.scale;
    page_stride = p.cp;
    row_stride = p.ct;
  }
  if (t < pieces + 8 || (p.format == MLA_KV_FP4_E2M1 && t == pieces + 8))
    keep_pieces<i32x4>(base, page_stride, row_stride, from, slot, moves);
}

static bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
static int bad(const char* what) { return mla_srv::set_error(MLA_ERR_INVALID, what); }
static int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mla_srv::set_error(MLA_ERR_HIP, std::string(what) + " launch failed: " + hipGetErrorString(e));
  return MLA_OK;
}
static int check_shape(int32_t batch, int32_t s_q) {
  if (batch < 0 || batch > (1 << 20)) return bad("batch must be in [0, 2^20]");
  if (s_q < 1 || s_q > kMaxNodes) return bad("s_q must be in [1, 64]");
  return MLA_OK;
}

}  // namespace mla_tree

using namespace mla_tree;

extern "C" {

int mla_tree_plan(const mla_tree_plan_args* a, void* stream) {
  if (!a) return bad("args is NULL");
  const int rc = check_shape(a->batch, a->s_q);
  if (rc != MLA_OK) return rc;
  if (a->batch == 0) return MLA_OK;
  if (!a->parents || !a->cache_seqlens || !a->block_table || !a->mask || !a->positions || !a->slots || !a->prefix_lens)
    return bad("a required pointer is NULL");
  if (!aligned(a->mask, 8)) return bad("mask must be 8-byte aligned");
  if (a->block_table_width < 1 || a->block_table_stride < a->block_table_width || a->block_table_width > (1 << 24))
    return bad("block_table_width must be in [1, min(block_table_stride, 2^24)]");
  const PlanParams k = {a->parents, a->cache_seqlens, a->tree_lens, a->block_table, a->block_table_stride, a->block_table_width,
                        a->batch, a->s_q, a->mask, a->positions, a->slots, a->prefix_lens};
  hipLaunchKernelGGL(mla_tree_plan_kernel, dim3((a->batch + 3) / 4), dim3(256), 0, (hipStream_t)stream, k);
  return launched("tree plan");
}

int mla_tree_accept(const uint64_t* mask, const int32_t* prefix_lens, const void* tokens, const void* targets, int32_t wide,
                    int32_t batch, int32_t s_q, int32_t* path, int32_t* counts, void* next_tokens, int32_t* keep_lens, void* stream) {
  const int rc = check_shape(batch, s_q);
  if (rc != MLA_OK) return rc;
  if (wide != 0 && wide != 1) return bad("wide must be 0 (int32 tokens) or 1 (int64)");
  if (batch == 0) return MLA_OK;
  if (!mask || !prefix_lens || !tokens || !targets || !path || !counts || !next_tokens || !keep_lens)
    return bad("a required pointer is NULL");
  const size_t es = wide ? 8 : 4;
  if (!aligned(mask, 8) || !aligned(tokens, es) || !aligned(targets, es) || !aligned(next_tokens, es))
    return bad("mask and tokens must be aligned to their elements");
  const AcceptParams k = {mask, prefix_lens, tokens, targets, batch, s_q, path, counts, next_tokens, keep_lens};
  const dim3 grid((batch + 3) / 4);
  if (wide)
    hipLaunchKernelGGL(mla_tree_accept_kernel<int64_t>, grid, dim3(256), 0, (hipStream_t)stream, k);
  else
    hipLaunchKernelGGL(mla_tree_accept_kernel<int32_t>, grid, dim3(256), 0, (hipStream_t)stream, k);
  return launched("tree accept");
}

int mla_kv_keep_path(const mla_kv_cache* cache, const int32_t* slots, const int32_t* path, int32_t batch, int32_t s_q, void* stream) {
  if (!cache) return bad("args is NULL");
  mla_srv::Cache c{};
  int rc = mla_srv::check_cache(cache, &c);
  if (rc != MLA_OK) return rc;
  if ((rc = check_shape(batch, s_q)) != MLA_OK) return rc;
  if (batch == 0) return MLA_OK;
  if (!slots || !path) return bad("a required pointer is NULL");
  const KeepParams k = {c.nope, c.rope, c.scale, c.sp, c.st, c.rp, c.rt, c.cp, c.ct, c.tokens, slots, path, s_q, c.format};
  hipLaunchKernelGGL(mla_keep_path_kernel, dim3(batch), dim3(128), 0, (hipStream_t)stream, k);
  return launched("keep path");
}

}  // extern "C"
