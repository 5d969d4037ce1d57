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
constexpr int kDimTiles = kDV / 16;

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
template <bool F16>
__device__ __forceinline__ float sum2(uint32_t w) {
  if constexpr (F16) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    return (float)h[0] + (float)h[1];
  } else {
    return __uint_as_float(w << 16) + __uint_as_float(w & 0xFFFF0000u);
  }
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The exponent that brings a partial's chunk to [2^14, 2^15), as the split-KV decode stores its partials.
__device__ __forceinline__ int part_exp(float amax) {
  const int e = 15 - __builtin_amdgcn_frexp_expf(amax);
  return e < 127 ? e : 127;
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

// Eight latent values (dims 8 lane ..) of a cached token as 16-bit words; coded caches widen to bf16, exactly.
template <int FMT>
__device__ __forceinline__ i32x4 latent8(const TreeParams& p, int64_t page, int row, int lane) {
  const uint8_t* src = p.nope + page * p.sp + row * p.st;
  if constexpr (FMT == MLA_KV_NATIVE) {
    return *(const i32x4*)(src + 16 * lane);
  } else if constexpr (FMT == MLA_KV_FP8_E4M3) {
    const i32x2 w = *(const i32x2*)(src + 8 * lane);
    const float sc = *(const float*)(p.scale + page * p.cp + (lane >> 4) * p.ct + 4 * row);
    const int a = w[0], b = w[1];
    return i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, true)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, true))};
  } else {
    const int w = *(const int*)(src + 4 * lane);
    const float sc = __uint_as_float((uint32_t)p.scale[page * p.cp + row * p.ct + (lane >> 2)] << 23);
    return i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3))};
  }
}

// ---------------------------------------------------------------------------------------
// the drafted tokens' split
// ---------------------------------------------------------------------------------------
// For 64 rows of a sequence, a wave 16 of them: S^T = K Q^T over the drafted tokens (16x16x32 MFMA, K rows from LDS,
// queries in registers), softmax over the row's visible ones, O^T = V^T P^T.  All keys are in one tile (32 KT of
// them), so the softmax is one pass and P^T never leaves the registers: the S^T accumulators of two token tiles, packed
// to 16 bits, are the B operand of PV in the k order of the transposed V reads.  P is rounded to 16 bits (the operand's
// type) and the sum that divides the output is of the rounded weights, so that the rounding cancels in it.
//
// A drafted token that a row does not see must not reach it, whatever its cache row holds (it may never have been
// written): a weight of 0 times an infinity or a NaN is a NaN.  A chunk that holds one is zeroed in LDS, the token is
// remembered, and rows that do see it become NaN.
constexpr int kPitch = 2 * MLA_DIM_QK + 16;  // bytes of a token in LDS: 16 rows start on 16 different groups of 4 banks

template <int FMT, bool F16, int KT>
__global__ __launch_bounds__(256, 2) void mla_tree_kernel(TreeParams p) {
  constexpr int kTok = 32 * KT;
  __shared__ __attribute__((aligned(16))) uint8_t kv_sh[kTok * kPitch];
  __shared__ unsigned long long bad_sh;
  const int b = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, li = lane & 15;
  const int last = p.splits[b + 1] + b;  // the sequence's last slot, with one more split for it and those before it
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (b == 0) p.splits_out[0] = p.splits[0];
    p.splits_out[b + 1] = last + 1;
  }
  if (threadIdx.x == 0) bad_sh = 0;
  int prefix = p.prefix[b];
  prefix = prefix > 0 ? prefix : 0;
  // drafted tokens that the table's row has room for, and the one or two pages that they lie in
  const int64_t room = (int64_t)p.bt_width * kPage - prefix;
  const int held = room < 0 ? 0 : room < p.s_q ? (int)room : p.s_q;
  const int at = prefix & (kPage - 1);
  int pages[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int col = prefix / kPage + i;
    col = col < p.bt_width ? col : p.bt_width - 1;
    const int id = p.block_table[(int64_t)b * p.bt_stride + col];
    pages[i] = id < 0 ? 0 : id < p.num_blocks ? id : p.num_blocks - 1;
  }

  // queries (B operand): lane (g, i) holds dims 32 kk + 8 g .. +7 of row i
  const int row_raw = blockIdx.x * 64 + 16 * wave + li;
  const int row = row_raw < p.rows ? row_raw : p.rows - 1;
  const int s = row / p.heads, h = row - s * p.heads;
  const uint16_t* qn = p.q_nope + (b * p.q_sb + s * p.q_ss + h * p.q_sh) + 8 * g;
  const uint16_t* qr = p.q_rope + (b * p.qr_sb + s * p.qr_ss + h * p.qr_sh) + 8 * g;
  i32x4 q[kKSteps];
#pragma unroll
  for (int kk = 0; kk < kKSteps; ++kk) q[kk] = *(const i32x4*)(kk < 16 ? qn + 32 * kk : qr + 32 * (kk - 16));
  uint64_t mask = p.mask[(int64_t)b * p.s_q + s];
  const uint64_t nodes = p.s_q == 64 ? ~0ull : (1ull << p.s_q) - 1;
  const uint64_t known = held == 64 ? ~0ull : (1ull << held) - 1;
  if ((mask & nodes & ~known) != 0 && p.status != nullptr) *p.status = 1;
  mask &= known;

  // the tokens into LDS: wave w takes tokens w, w + 4, .., a lane 8 dims of each
  i32x4 v[kTok / 4], r[KT];
#pragma unroll
  for (int i = 0; i < kTok / 4; ++i) {
    const int j = 4 * i + wave;  // uniform
    v[i] = i32x4{0, 0, 0, 0};
    if (j < held) v[i] = latent8<FMT>(p, at + j < kPage ? pages[0] : pages[1], (at + j) & (kPage - 1), lane);
  }
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    const int j = 32 * i + 8 * wave + (lane >> 3);
    r[i] = i32x4{0, 0, 0, 0};
    if (j < held) {
      const int64_t page = at + j < kPage ? pages[0] : pages[1];
      r[i] = *(const i32x4*)(p.rope + page * p.rp + ((at + j) & (kPage - 1)) * p.rt + 16 * (lane & 7));
    }
  }
  __syncthreads();  // bad_sh is clear
#pragma unroll
  for (int i = 0; i < kTok / 4; ++i) {
    const int j = 4 * i + wave;
    const bool bad = non_finite<F16>(v[i]);
    if (__builtin_amdgcn_ballot_w64(bad) != 0) {  // uniform, rare
      if (bad) v[i] = i32x4{0, 0, 0, 0};
      if (lane == 0) atomicOr(&bad_sh, 1ull << j);
    }
    *(i32x4*)(kv_sh + j * kPitch + 16 * lane) = v[i];
  }
#pragma unroll
  for (int i = 0; i < KT; ++i)
    *(i32x4*)(kv_sh + (32 * i + 8 * wave + (lane >> 3)) * kPitch + 2 * kDV + 16 * (lane & 7)) = r[i];
  __syncthreads();
  const uint64_t bad = bad_sh;

  // S^T: lane (g, i) gets tokens 16 t + 4 g .. +3 of row i
  f32x4 sc[2 * KT];
#pragma unroll
  for (int t = 0; t < 2 * KT; ++t) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const uint8_t* k = kv_sh + (16 * t + li) * kPitch + 16 * g;
#pragma unroll
    for (int kk = 0; kk < kKSteps; ++kk) acc = mfma32<F16>(*(const i32x4*)(k + 64 * kk), q[kk], acc);
    sc[t] = acc;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int t = 0; t < 2 * KT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool seen = (mask >> (16 * t + 4 * g + i)) & 1;
      sc[t][i] = seen ? sc[t][i] * p.scale_log2 : -INFINITY;
      mx = fmaxf(mx, sc[t][i]);
    }
  mx = group_max(mx);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, lx = 0.f;
  i32x4 pb[KT];
#pragma unroll
  for (int t = 0; t < 2 * KT; ++t) {
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = __builtin_amdgcn_exp2f(sc[t][i] - ref);
      lx += e[i];
    }
    const uint32_t w0 = pack2<F16>(e[0], e[1]), w1 = pack2<F16>(e[2], e[3]);
    l += sum2<F16>(w0) + sum2<F16>(w1);
    pb[t >> 1][2 * (t & 1)] = (int)w0;
    pb[t >> 1][2 * (t & 1) + 1] = (int)w1;
  }
  l = group_sum(l);
  lx = group_sum(lx);

  // O^T: transposed reads give lane (g, i) tokens 4 g .. +3 and 16 + 4 g .. +3 of dim 16 d + i
  f32x4 o[kDimTiles];
  const uint8_t* vt = kv_sh + (4 * g + (li >> 2)) * kPitch + 8 * (li & 3);
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const uint8_t LDS_AS* a = (const uint8_t LDS_AS*)(vt + 32 * t * kPitch + 32 * d);
      const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)a));
      const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 LDS_AS*)(a + 16 * kPitch)));
      acc = mfma32<F16>(i32x4{lo[0], lo[1], hi[0], hi[1]}, pb[t], acc);
    }
    o[d] = acc;
  }

  // the partial, as the split-KV decode writes its own: fp16 rows, each 128-dim chunk times a power of two
  const bool spoilt = (mask & bad) != 0;
  const float inv = spoilt ? __builtin_nanf("") : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  // a NaN here makes the merged lse -inf, as any NaN row's is
  const float lse2 = spoilt ? __builtin_nanf("") : lx > 0.f ? mx + __log2f(lx) : lx == 0.f ? -INFINITY : lx;
  int e[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float a = 0.f;
#pragma unroll
    for (int d = 8 * c; d < 8 * c + 8; ++d)
      a = fmaxf(fmaxf(fmaxf(fabsf(o[d][0]), fabsf(o[d][1])), fmaxf(fabsf(o[d][2]), fabsf(o[d][3]))), a);
    e[c] = part_exp(group_max(a * inv));
  }
  if (row_raw >= p.rows) return;
  const int64_t dst_row = (int64_t)last * p.rows + row;
  uint16_t* dst = p.ws_o + dst_row * kDV + 4 * g;
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d) {
    const f32x4 x = (o[d] * inv) * exp2i(e[d >> 3]);
    *(i32x2*)(dst + 16 * d) = i32x2{(int)pack2<true>(x[0], x[1]), (int)pack2<true>(x[2], x[3])};
  }
  const int eg = g == 0 ? e[0] : g == 1 ? e[1] : g == 2 ? e[2] : e[3];
  p.ws_scale[dst_row * 4 + g] = exp2i(-eg);
  if (g == 0) p.ws_lse[dst_row] = lse2;
}

template <int FMT, bool F16>
static void launch_format(const TreeParams& p, hipStream_t st) {
  const dim3 grid((p.rows + 63) / 64, p.batch);
  if (p.s_q <= 32)
    hipLaunchKernelGGL((mla_tree_kernel<FMT, F16, 1>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((mla_tree_kernel<FMT, F16, 2>), grid, dim3(256), 0, st, p);
}

hipError_t launch_drafts(const TreeParams& p, hipStream_t st) {
  if (p.format == MLA_KV_FP8_E4M3) launch_format<MLA_KV_FP8_E4M3, false>(p, st);
  else if (p.format == MLA_KV_FP4_E2M1) launch_format<MLA_KV_FP4_E2M1, false>(p, st);
  else if (p.f16) launch_format<MLA_KV_NATIVE, true>(p, st);
  else launch_format<MLA_KV_NATIVE, false>(p, st);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// plan: parents -> masks, positions, cache rows, prefix lengths
// ---------------------------------------------------------------------------------------
// A wave a sequence, a lane a node.  A node's mask is its own bit and its parent's mask.  Each of six rounds takes
// over the mask of the node that the lane points at and then points where that one does: 2, 4, .. 64 generations.
// Bound by latency: two loads, six rounds of lane reads, a table lookup: a step's 128 trees of 16 nodes 2.7 us.
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
// takes one 16-byte piece of the rows (4 bytes of the fp8 cache's scales) and walks the path in order, kAhead rows
// read ahead of their writes.  No read can meet an earlier write: an entry is at least its own place (others are
// passed over), so the rows written before it lie below the one that it reads.  Bound by latency: rows read in turns
// of kAhead; paths are a few nodes long.
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
constexpr int kAhead = 8;

template <class V>
__device__ __forceinline__ void keep_pieces(uint8_t* base, int64_t page_stride, int64_t row_stride, const int32_t* slots,
                                            const int32_t* path, int s_q, int64_t tokens) {
  for (int k0 = 0; k0 < s_q; k0 += kAhead) {
    V v[kAhead];
    int64_t to[kAhead];
    bool more = false;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int k = k0 + u;
      to[u] = -1;
      if (k >= s_q) continue;
      const int j = path[k];
      more = j >= 0;
      if (j <= k || j >= s_q) continue;
      const int64_t src = slots[j], dst = slots[k];
      if (src < 0 || dst < 0 || src >= tokens || dst >= tokens) continue;
      to[u] = dst / kPage * page_stride + dst % kPage * row_stride;
      v[u] = *(const V*)(base + src / kPage * page_stride + src % kPage * row_stride);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (to[u] >= 0) *(V*)(base + to[u]) = v[u];
    if (!more) break;  // the path's end
  }
}

__global__ __launch_bounds__(128) void mla_keep_path_kernel(KeepParams p) {
  const int t = threadIdx.x;
  const int32_t* slots = p.slots + (int64_t)blockIdx.x * p.s_q;
  const int32_t* path = p.path + (int64_t)blockIdx.x * p.s_q;
  const int pieces = p.format == MLA_KV_NATIVE ? 64 : p.format == MLA_KV_FP8_E4M3 ? 32 : 16;  // of the latent
  if (t < pieces) {
    keep_pieces<i32x4>(p.nope + 16 * t, p.sp, p.st, slots, path, p.s_q, p.tokens);
  } else if (t < pieces + 8) {
    keep_pieces<i32x4>(p.rope + 16 * (t - pieces), p.rp, p.rt, slots, path, p.s_q, p.tokens);
  } else if (p.format == MLA_KV_FP8_E4M3 && t < pieces + 12) {
    keep_pieces<int32_t>(p.scale + (t - pieces - 8) * p.ct, p.cp, 4, slots, path, p.s_q, p.tokens);
  } else if (p.format == MLA_KV_FP4_E2M1 && t == pieces + 8) {
    keep_pieces<i32x4>(p.scale, p.cp, p.ct, slots, path, p.s_q, p.tokens);
  }
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
