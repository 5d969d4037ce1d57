// mla_serving.hip -- what a serving step does around the decode (gfx950): rotary positions, the append
// of ragged token counts by slot map with the rotation fused in, the append to the 4-bit cache, reading
// cached tokens back, and the bookkeeping of pages, block tables and slot maps.
//
// All of it is bound by memory or by latency: a decode step's calls move a few hundred KiB, so they
// are one launch each, with independent loads requested together; a prefill's stream through HBM.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string>

#include "mla_decode_amd.h"
#include "mla_serving.h"

namespace mla_srv {

constexpr int kPage = MLA_PAGE_TOKENS;
constexpr int kDV = MLA_DIM_V;
constexpr int kRope = MLA_DIM_QK - MLA_DIM_V;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Cache {
  int32_t format;
  int32_t f16;  // native: fp16 (else bf16)
  int64_t tokens;
  uint8_t* nope;
  uint8_t* rope;
  uint8_t* scale;
  int64_t sp, st, rp, rt, cp, ct;  // page and token (fp8 scale: block) strides in bytes
};

// ---------------------------------------------------------------------------------------
// values of the three element types
// ---------------------------------------------------------------------------------------
struct Bf16 {
  static constexpr int kBytes = 2;
  typedef uint16_t bits;
  __device__ static float value(bits b) { return __uint_as_float((uint32_t)b << 16); }
  __device__ static bits of(float v) { return __builtin_bit_cast(bits, (__bf16)v); }
};
struct F16 {
  static constexpr int kBytes = 2;
  typedef uint16_t bits;
  __device__ static float value(bits b) { return (float)__builtin_bit_cast(_Float16, b); }
  __device__ static bits of(float v) { return __builtin_bit_cast(bits, (_Float16)v); }
};
struct F32 {
  static constexpr int kBytes = 4;
  typedef uint32_t bits;
  __device__ static float value(bits b) { return __uint_as_float(b); }
  __device__ static bits of(float v) { return __float_as_uint(v); }
};

// 16 bytes to floats and back (8 values, or 4 of fp32)
template <class E>
__device__ __forceinline__ void unpack(const i32x4 v, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (uint32_t)v[j];
    if constexpr (E::kBytes == 4) {
      x[j] = __uint_as_float(w);
    } else if constexpr (__is_same(E, Bf16)) {
      x[2 * j] = __uint_as_float(w << 16);
      x[2 * j + 1] = __uint_as_float(w & 0xFFFF0000u);
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      x[2 * j] = (float)h[0];
      x[2 * j + 1] = (float)h[1];
    }
  }
}
template <class E>
__device__ __forceinline__ i32x4 pack(const float* x) {
  i32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (E::kBytes == 4)
      v[j] = (int)__float_as_uint(x[j]);
    else if constexpr (__is_same(E, Bf16))
      v[j] = __builtin_bit_cast(int, __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), bf16x2));
    else
      v[j] = __builtin_bit_cast(int, __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), f16x2));
  }
  return v;
}

// ---------------------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------------------
// Pair i of a head at position p is multiplied, as a complex number, by amp * e^(2 pi i p f_i), f in turns
// per position.  p * f is formed and reduced to half a turn in 64 bits: at position 10^6 a 32-bit
// product would be off by a sixteenth of a turn's 2 pi.  Everything after it is fp32, rounded once.
__device__ __forceinline__ f32x2 turn(int pos, double f, float amp) {
  double t = (double)pos * f;
  t -= rint(t);
  float s, c;
  sincospif(2.f * (float)t, &s, &c);
  return f32x2{c * amp, s * amp};
}
__device__ __forceinline__ void rotate(float& a, float& b, f32x2 cs) {
  const float x = a * cs[0] - b * cs[1];
  b = a * cs[1] + b * cs[0];
  a = x;
}
// A token without a position stays as it is, bit for bit (a turn of zero would spread an infinity or a NaN to its pair,
// and make some -0 a 0): its cosines hold a signalling NaN, which no arithmetic gives.
constexpr uint32_t kStill = 0x7F800001u;
__device__ __forceinline__ f32x2 turn_or_still(int pos, double f, float amp) {
  return pos < 0 ? f32x2{__uint_as_float(kStill), 0.f} : turn(pos, f, amp);
}
__device__ __forceinline__ bool is_still(f32x2 cs) { return __float_as_uint(cs[0]) == kStill; }
// Whether any of the four waves' lanes set `mine`, the same for all of them; a barrier.
__device__ __forceinline__ bool any_of_256(bool mine, int (&any_sh)[4]) {
  any_sh[threadIdx.x >> 6] = __builtin_amdgcn_ballot_w64(mine) != 0;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(any_sh[0] | any_sh[1] | any_sh[2] | any_sh[3]) != 0;
}
template <class E>
__device__ __forceinline__ void rotate_bits(typename E::bits& a, typename E::bits& b, f32x2 cs) {
  float x = E::value(a), y = E::value(b);
  rotate(x, y, cs);
  const bool keep = is_still(cs);
  a = keep ? a : E::of(x);
  b = keep ? b : E::of(y);
}

// Item `i` of [tokens][heads][items] as (t, h, it), in steps of 256 items without a division.
struct Walk {
  int t, h, it;
  int items, heads, step_t, step_h, step_it;
  __device__ __forceinline__ Walk(int i, int items_, int heads_) : items(items_), heads(heads_) {
    const int th = i / items;
    it = i - th * items;
    t = th / heads;
    h = th - t * heads;
    const int s = 256 / items;
    step_it = 256 - s * items;
    step_t = s / heads;
    step_h = s - step_t * heads;
  }
  __device__ __forceinline__ void step() {
    it += step_it;
    h += step_h;
    t += step_t;
    if (it >= items) it -= items, ++h;
    if (h >= heads) h -= heads, ++t;
  }
};

struct RopeParams {
  const uint8_t* x;
  uint8_t* out;
  int64_t x_st, x_sh, o_st, o_sh;  // bytes
  const int32_t* positions;
  const double* freqs;
  int32_t tokens, heads, dim, rot, first, half;
  float amp;
  int32_t tile;   // tokens per workgroup
  int32_t split;  // workgroups that share a token tile's heads
};

// 256 threads take `tile` tokens (tile * rot / 2 <= kPairs): each pair's cosine and sine once per token into LDS,
// then every head.  VEC: 16-byte chunks; a chunk of the rotated dims holds whole pairs (interleaved), or is
// taken together with the chunk half the rotated dims further on (half layout).
// Bound by memory: 8191 tokens x 32 heads of 128 fp16 dims, 64 of them rotated, 23.3 us (134 MB; 24.8 with one chunk
// a thread in flight and a division an item, 23.4 with four chunks).  128 tokens x 128 heads: 4.0 us, a launch.
// Rows that no 16-byte chunk fits (71 dims a head) go value by value, in 2- or 4-byte accesses: 8191 x 32 heads, 75 MB,
// 34.9 us; rows that start on odd elements have no wider ones.
constexpr int kPairs = 512, kRopeTile = 8;
template <class E, bool VEC>
__global__ __launch_bounds__(256) void mla_rope_kernel(RopeParams p) {
  __shared__ f32x2 cs[kPairs];
  __shared__ int any_sh[4];
  const int pairs = p.rot / 2;
  const int wg = blockIdx.x / p.split, sub = blockIdx.x - wg * p.split;
  const int t0 = wg * p.tile;
  const int nt = p.tokens - t0 < p.tile ? p.tokens - t0 : p.tile;
  bool mine = false;
  for (int i = threadIdx.x; i < nt * pairs; i += 256) {
    const int t = i / pairs;
    const int pos = p.positions[t0 + t];
    cs[i] = turn_or_still(pos, p.freqs[i - t * pairs], p.amp);
    mine |= pos < 0;
  }
  const bool some_still = any_of_256(mine, any_sh);  // rare: the loop looks for them only then
  const int h0 = (int)((int64_t)p.heads * sub / p.split), h1 = (int)((int64_t)p.heads * (sub + 1) / p.split);
  const int nh = h1 - h0;
  constexpr int W = VEC ? 16 / E::kBytes : 1;  // values per item
  // items of a head: chunks of W values (half layout: the second halves come with the first ones); the
  // scalar form takes a pair or a single value per item
  const int rot_items = VEC ? (p.half ? pairs / W : p.rot / W) : pairs;
  const int lead = p.first / W, tail = (p.dim - p.first - p.rot) / W;
  const bool in_place = p.out == p.x;
  const int items = rot_items + (in_place ? 0 : lead + tail);
  const int total = nt * nh * items;
  Walk at(threadIdx.x, items, nh);
  if constexpr (VEC) {
    constexpr int U = 2;  // a thread's chunks in flight
#pragma unroll 1
    for (int i = threadIdx.x; i < total; i += 256 * U) {
      i32x4 v[U], w[U];
      uint8_t* dst[U];
      int pair[U];  // the chunk's first pair among its tile's, -1: a chunk that is copied
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + 256 * u < total) {
          const bool turns = at.it < rot_items;
          const int c = at.it - rot_items;
          const int a = (turns ? p.first + at.it * W : c < lead ? c * W : p.first + p.rot + (c - lead) * W) * E::kBytes;
          const uint8_t* src = p.x + (int64_t)(t0 + at.t) * p.x_st + (int64_t)(h0 + at.h) * p.x_sh + a;
          dst[u] = p.out + (int64_t)(t0 + at.t) * p.o_st + (int64_t)(h0 + at.h) * p.o_sh + a;
          pair[u] = turns ? at.t * pairs + at.it * (p.half ? W : W / 2) : -1;
          v[u] = *(const i32x4*)src;
          if (p.half && turns) w[u] = *(const i32x4*)(src + pairs * E::kBytes);
        }
        at.step();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + 256 * u >= total) break;
        if (pair[u] >= 0) {
          const f32x2* c = cs + pair[u];
          if (!(some_still && is_still(c[0]))) {
            float x[W], y[W];
            unpack<E>(v[u], x);
            if (p.half) {
              unpack<E>(w[u], y);
#pragma unroll
              for (int j = 0; j < W; ++j) rotate(x[j], y[j], c[j]);
              w[u] = pack<E>(y);
            } else {
#pragma unroll
              for (int j = 0; j < W / 2; ++j) rotate(x[2 * j], x[2 * j + 1], c[j]);
            }
            v[u] = pack<E>(x);
          }
          if (p.half) *(i32x4*)(dst[u] + pairs * E::kBytes) = w[u];
        }
        *(i32x4*)dst[u] = v[u];
      }
    }
  } else {
    for (int i = threadIdx.x; i < total; i += 256, at.step()) {
      const uint8_t* src = p.x + (int64_t)(t0 + at.t) * p.x_st + (int64_t)(h0 + at.h) * p.x_sh;
      uint8_t* dst = p.out + (int64_t)(t0 + at.t) * p.o_st + (int64_t)(h0 + at.h) * p.o_sh;
      if (at.it < rot_items) {
        const int a = (p.first + (p.half ? at.it : 2 * at.it)) * E::kBytes, b = a + (p.half ? pairs : 1) * E::kBytes;
        typename E::bits x = *(const typename E::bits*)(src + a), y = *(const typename E::bits*)(src + b);
        rotate_bits<E>(x, y, cs[at.t * pairs + at.it]);
        *(typename E::bits*)(dst + a) = x;
        *(typename E::bits*)(dst + b) = y;
      } else {
        const int c = at.it - rot_items;
        const int a = (c < lead ? c : p.first + p.rot + (c - lead)) * E::kBytes;
        *(typename E::bits*)(dst + a) = *(const typename E::bits*)(src + a);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// one token into the cache
// ---------------------------------------------------------------------------------------
// k of a block's scale from its bf16 amax (bit pattern `bits`): the smallest with amax <= top * 2^k,
// top = 1.m * 2^e (e2m1: 6 = 1.5 * 2^2, e4m3: 448 = 1.75 * 2^8), in [-126, 127]; amax = 0 gives 0.
__device__ __forceinline__ int block_exp(uint32_t bits, int e, uint32_t m) {
  int k = (int)(bits >> 7) - 127 - e + ((bits & 0x7F) > m ? 1 : 0);
  k = k < -126 ? -126 : k;
  return bits == 0 ? 0 : k;
}

// The wave's lane l holds dims 8l .. 8l+7 of the token's latent (v); written to (page, row) of the cache.
// A 4-bit block with a NaN or an infinity in it is marked whole (scale byte 255): the format has neither.  A value past
// 1.5 * 2^127, the largest that e2m1 and bf16 both hold, is stored as that one: the next, 4 * 2^126, would read back
// as an infinity.
__device__ __forceinline__ void put_latent(const Cache& c, int64_t page, int row, int lane, i32x4 v) {
  uint8_t* dst = c.nope + page * c.sp + row * c.st;
  if (c.format == MLA_KV_NATIVE) {
    *(i32x4*)(dst + 16 * lane) = v;
    return;
  }
  float x[8];
  unpack<Bf16>(v, x);
  uint32_t top = 0;  // |x| as bits: ordered like the values, with infinities and NaNs at the end
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (uint32_t)v[j] & 0x7FFF7FFFu;
    const uint32_t lo = w & 0xFFFFu, hi = w >> 16;
    top = top > lo ? top : lo;
    top = top > hi ? top : hi;
  }
  const int width = c.format == MLA_KV_FP4_E2M1 ? 4 : 16;  // lanes per block
  for (int m = 1; m < width; m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)top, m);
    top = top > o ? top : o;
  }
  if (c.format == MLA_KV_FP4_E2M1) {
    const bool bad = top >= 0x7F80u;
    const int k = bad ? 0 : block_exp(top, 2, 0x40);
    const float sc = __uint_as_float((uint32_t)(k + 127) << 23);
    if (__builtin_amdgcn_ballot_w64(k > 125) != 0) {  // uniform, rare
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_fmed3f(x[j], -0x1.8p127f, 0x1.8p127f);
    }
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], sc, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], sc, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], sc, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], sc, 3);
    *(uint32_t*)(dst + 4 * lane) = bad ? 0u : w;
    if ((lane & 3) == 0) c.scale[page * c.cp + row * c.ct + (lane >> 2)] = bad ? 255 : (uint8_t)(k + 127);
  } else {
    float amax = 0.f;  // as mla_kv_append: a NaN is passed over by the maximum
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 16));
    const uint32_t bits = __float_as_uint(amax) >> 16;
    const int k = bits == 0 ? 0 : (bits >> 7) == 0 ? -126 : block_exp(bits, 8, 0x60);
    const int kc = k > 127 ? 127 : k;
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(x[0], -kc), __builtin_ldexpf(x[1], -kc), lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(x[2], -kc), __builtin_ldexpf(x[3], -kc), lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(x[4], -kc), __builtin_ldexpf(x[5], -kc), hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(x[6], -kc), __builtin_ldexpf(x[7], -kc), hi, true);
    *(i32x2*)(dst + 8 * lane) = i32x2{lo, hi};
    if ((lane & 15) == 0)
      *(uint32_t*)(c.scale + page * c.cp + (lane >> 4) * c.ct + 4 * row) = (uint32_t)(kc + 127) << 23;
  }
}

// ---------------------------------------------------------------------------------------
// append by slot map
// ---------------------------------------------------------------------------------------
struct AppendParams {
  Cache cache;
  const uint8_t* kv_new;
  int64_t n_st;  // bytes
  const int32_t* slots;
  const int32_t* positions;
  const double* freqs;  // null: nothing is rotated
  int32_t half;
  float amp;
  const uint8_t* q_pe;  // null: no queries
  uint8_t* q;           // its rope dims
  int64_t pe_st, pe_sh, q_st, q_sh;
  int32_t tokens, heads, tile;
};

// Workgroups of four waves take `tile` tokens: the 32 pairs' cosines and sines of each token into LDS, a
// wave per token for its cache row, and all threads for the queries' rope dims in 16-byte chunks.  One launch for
// the three.  What is not rotated is copied bit for bit.  Bound by memory where there is any: 76 MB of a ragged prefill
// (16 heads, 4-bit cache) in 16.1 us, 4.7 TB/s, a large copy's rate; 65536 tokens without queries into the 4-bit cache
// 22.8 us (floor 21), into the fp8 one 27.5 (24.5: its scales leave four bytes a token and block).  A decode step's
// 128 tokens x 16 heads 3.5 us.
constexpr int kAppendTile = 8;
template <class E>
__global__ __launch_bounds__(256) void mla_append_slots_kernel(AppendParams p) {
  __shared__ f32x2 cs[kAppendTile][32];
  __shared__ int32_t slot_sh[kAppendTile];  // -1: names no row
  __shared__ int any_sh[4];
  const int t0 = blockIdx.x * p.tile;
  const int nt = p.tokens - t0 < p.tile ? p.tokens - t0 : p.tile;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (threadIdx.x < nt) {
    const int slot = p.slots[t0 + threadIdx.x];
    slot_sh[threadIdx.x] = slot >= 0 && slot < p.cache.tokens ? slot : -1;
  }
  bool mine = false;
  if (p.freqs != nullptr) {
    const int t = threadIdx.x >> 5;
    if (t < nt) {
      const int pos = p.positions[t0 + t];
      mine = pos < 0;
      cs[t][threadIdx.x & 31] = turn_or_still(pos, p.freqs[threadIdx.x & 31], p.amp);
    }
  }
  // a wave's tokens, loaded together, whatever their slots
  i32x4 v[kAppendTile / 4];
  uint16_t x[kAppendTile / 4], y[kAppendTile / 4];
  const int rope_a = (p.half ? lane : 2 * lane) * 2, rope_b = rope_a + (p.half ? 64 : 2);  // a rope pair per lane < 32
#pragma unroll
  for (int u = 0; u < kAppendTile / 4; ++u) {
    const int t = wave + 4 * u;
    if (t < nt) {  // uniform
      const uint8_t* src = p.kv_new + (int64_t)(t0 + t) * p.n_st;
      v[u] = *(const i32x4*)(src + 16 * lane);
      if (lane < 32) x[u] = *(const uint16_t*)(src + 2 * kDV + rope_a), y[u] = *(const uint16_t*)(src + 2 * kDV + rope_b);
    }
  }
  const bool some_still = any_of_256(mine, any_sh);
#pragma unroll
  for (int u = 0; u < kAppendTile / 4; ++u) {
    const int t = wave + 4 * u;
    if (t >= nt) break;  // uniform
    const int64_t slot = __builtin_amdgcn_readfirstlane(slot_sh[t]);
    if (slot < 0) continue;
    const int64_t page = slot / kPage;
    const int row = (int)(slot % kPage);
    if (lane < 32) {
      if (p.freqs != nullptr) rotate_bits<E>(x[u], y[u], cs[t][lane]);
      uint8_t* dst = p.cache.rope + page * p.cache.rp + row * p.cache.rt;
      *(uint16_t*)(dst + rope_a) = x[u];
      *(uint16_t*)(dst + rope_b) = y[u];
    }
    put_latent(p.cache, page, row, lane, v[u]);
  }
  if (p.q_pe == nullptr) return;
  const int per_head = p.half ? 4 : 8;
  const int total = nt * p.heads * per_head;
  constexpr int U = 2;  // a thread's chunks in flight
  const int first = (threadIdx.x + 256 - 64 * (nt & 3)) & 255;  // the waves after the tokens' own start first
  Walk at(first, per_head, p.heads);
#pragma unroll 1
  for (int i = first; i < total; i += 256 * U) {
    i32x4 a[U], b[U];
    uint8_t* dst[U];
    const f32x2* turns[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      turns[u] = nullptr;
      if (i + 256 * u < total && slot_sh[at.t] >= 0) {
        const uint8_t* src = p.q_pe + (int64_t)(t0 + at.t) * p.pe_st + (int64_t)at.h * p.pe_sh + 16 * at.it;
        dst[u] = p.q + (int64_t)(t0 + at.t) * p.q_st + (int64_t)at.h * p.q_sh + 16 * at.it;
        turns[u] = &cs[at.t][(p.half ? 8 : 4) * at.it];
        a[u] = *(const i32x4*)src;
        if (p.half) b[u] = *(const i32x4*)(src + 64);
      }
      at.step();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (turns[u] == nullptr) continue;
      if (some_still && is_still(turns[u][0])) {
        *(i32x4*)dst[u] = a[u];
        if (p.half) *(i32x4*)(dst[u] + 64) = b[u];
        continue;
      }
      float x[8], y[8];
      unpack<E>(a[u], x);
      if (p.half) {
        unpack<E>(b[u], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) rotate(x[j], y[j], turns[u][j]);
        *(i32x4*)(dst[u] + 64) = pack<E>(y);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) rotate(x[2 * j], x[2 * j + 1], turns[u][j]);
      }
      *(i32x4*)dst[u] = pack<E>(x);
    }
  }
}

// The 4-bit form of mla_kv_append: n_new tokens of each sequence at its length, which then advances.  One
// workgroup per sequence, a wave per token; every wave checks all of the sequence's pages first.  What bounds it
// is latency: the length, the table's entry, the token, one after the other: a token of each of 128 sequences 3.2 us.
// Whole pages (a quantised cache of 138496 tokens, 215 MB) 39.5 us, 5.4 TB/s.
struct SeqAppendParams {
  Cache cache;
  const uint8_t* kv_new;
  int64_t n_sb, n_st;
  const int32_t* block_table;
  int32_t bt_stride, max_pages, n_new;
  int32_t* seqlens;
  int32_t* status;
};
__global__ __launch_bounds__(1024) void mla_append_fp4_kernel(SeqAppendParams p) {
  const int b = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int waves = blockDim.x >> 6;
  const int L = p.seqlens[b];
  const uint32_t pos = (uint32_t)L + (uint32_t)lane;  // token `lane`'s position (n_new <= 64)
  int page = -1;
  if (lane < p.n_new && L >= 0 && (int)pos >= 0 && (int)(pos / kPage) < p.max_pages)
    page = p.block_table[(int64_t)b * p.bt_stride + pos / kPage];
  const bool ok = __builtin_amdgcn_ballot_w64(lane < p.n_new && (page < 0 || page >= p.cache.tokens / kPage)) == 0;
  __syncthreads();  // every wave has read the length
  if (threadIdx.x == 0) {
    if (ok)
      p.seqlens[b] = L + p.n_new;
    else if (p.status != nullptr)
      *p.status = 1;
  }
  if (!ok) return;
  for (int t = wave; t < p.n_new; t += waves) {  // uniform
    const uint8_t* src = p.kv_new + b * p.n_sb + t * p.n_st;
    const int64_t pg = __builtin_amdgcn_readlane(page, t);
    const int row = (L + t) & (kPage - 1);
    const i32x4 v = *(const i32x4*)(src + 16 * lane);
    if (lane < 8) *(i32x4*)(p.cache.rope + pg * p.cache.rp + row * p.cache.rt + 16 * lane) = *(const i32x4*)(src + 2 * kDV + 16 * lane);
    put_latent(p.cache, pg, row, lane, v);
  }
}

// ---------------------------------------------------------------------------------------
// cached tokens back as rows
// ---------------------------------------------------------------------------------------
struct GatherParams {
  Cache cache;
  const int32_t* slots;
  uint8_t* out;
  int64_t o_st;  // bytes
  int32_t tokens;
};
// A wave a token: its row is read in one load of 16 bytes a lane (8 of fp8, 4 of 4-bit codes) and one of rope, and
// written in two.  Bound by memory: 65536 fp8 tokens (118 MB) in 25.5 us, 4.6 TB/s, where a large copy reaches 4.9.
template <int FMT>
__global__ __launch_bounds__(256) void mla_gather_kernel(GatherParams p) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + wave;
  if (t >= p.tokens) return;
  const int64_t slot = p.slots[t];
  uint8_t* dst = p.out + (int64_t)t * p.o_st;
  i32x4 v = {0, 0, 0, 0}, r = v;
  if (slot >= 0 && slot < p.cache.tokens) {  // uniform
    const int64_t page = slot / kPage;
    const int row = (int)(slot % kPage);
    const uint8_t* src = p.cache.nope + page * p.cache.sp + row * p.cache.st;
    if (lane < 8) r = *(const i32x4*)(p.cache.rope + page * p.cache.rp + row * p.cache.rt + 16 * lane);
    if constexpr (FMT == MLA_KV_NATIVE) {
      v = *(const i32x4*)(src + 16 * lane);
    } else if constexpr (FMT == MLA_KV_FP4_E2M1) {
      const int w = *(const int*)(src + 4 * lane);
      const float sc = __uint_as_float((uint32_t)p.cache.scale[page * p.cache.cp + row * p.cache.ct + (lane >> 2)] << 23);
      v = i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3))};
    } else {
      const i32x2 w = *(const i32x2*)(src + 8 * lane);
      const float sc = *(const float*)(p.cache.scale + page * p.cache.cp + (lane >> 4) * p.cache.ct + 4 * row);
      const int a = w[0], b = w[1];
      v = i32x4{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, false)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, true)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, false)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, true))};
    }
  }
  *(i32x4*)(dst + 16 * lane) = v;
  if (lane < 8) *(i32x4*)(dst + 2 * kDV + 16 * lane) = r;
}

// ---------------------------------------------------------------------------------------
// pages, block tables and slot maps
// ---------------------------------------------------------------------------------------
// The pool is a stack: free[0 .. count) are the free pages, taken from the top.  Request b needs the pages
// between ceil(L / 64) and ceil((L + n) / 64); requests are served in order, from prefix sums of the rows
// and pages asked for, so which page goes where depends on nothing but the inputs.
constexpr int kChunk = 1024;

__device__ __forceinline__ int pages_up(int64_t t) { return (int)((t + kPage - 1) / kPage); }

// inclusive prefix sum over the workgroup's 1024 threads; `wsum`: 16 words
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* wsum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up((long long)v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();  // the words' last readers are done
  if (lane == 63) wsum[wave] = v;
  __syncthreads();
  int64_t before = 0;
#pragma unroll
  for (int w = 0; w < kChunk / 64; ++w) before += w < wave ? wsum[w] : 0;
  return v + before;
}

struct ReserveParams {
  const int32_t* free;
  int32_t* count;
  int32_t num_blocks;
  int32_t* block_table;
  int32_t bt_stride, width, batch, tokens;
  int32_t* seqlens;
  const int32_t* new_lens;
  int32_t* slots;
  int32_t* positions;
  int32_t* cu_new;   // [batch + 1]
  int32_t* granted;  // [batch]
  int32_t* first;    // [batch + 1]: rank of the request's first new page; the count before the call
};

// Row t of the map: request b, its length before the call, rank of its first new page.
__device__ __forceinline__ void place_row(const ReserveParams& p, int t, int b, int start, int L, int on, int first, int count) {
  int slot = -1, pos = -1;
  if (on) {
    pos = L + (t - start);
    const int col = pos / kPage;
    int* cell = p.block_table + (int64_t)b * p.bt_stride + col;
    int page;
    if (col < pages_up(L)) {
      page = *cell;
    } else {
      page = p.free[count - 1 - (first + col - pages_up(L))];
      if ((pos & (kPage - 1)) == 0) *cell = page;  // every new page starts with a new row
    }
    if (page >= 0 && page < p.num_blocks) slot = page * kPage + (pos & (kPage - 1));  // else no row, and no overflow
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

// One workgroup: the prefix sums, grants, lengths and the pool's count, chunk by chunk; ROWS: the map too
// (with many rows mla_slot_rows_kernel fills it from what is left in cu_new, granted and first).  A grant depends on
// every earlier request, so the work is three prefix sums of a chunk of 1024 requests, and what bounds it is their
// latency: 5 to 6 us of kernel for up to 1024 requests, most of it the dependent loads and barriers.
template <bool ROWS>
__global__ __launch_bounds__(kChunk) void mla_reserve_kernel(ReserveParams p) {
  __shared__ int64_t wsum[kChunk / 64];
  __shared__ int start_sh[kChunk + 1], len_sh[kChunk], first_sh[kChunk];
  __shared__ int on_sh[kChunk];
  __shared__ int64_t carry_sh[2];
  const int tid = threadIdx.x;
  int count = *p.count;
  count = count < 0 ? 0 : (count > p.num_blocks ? p.num_blocks : count);
  int64_t rows = 0, asked = 0, used = 0;  // before this chunk
  for (int base = 0; base < p.batch; base += kChunk) {
    const int b = base + tid;
    int n = 0, L = -1;
    if (b < p.batch) {
      n = p.new_lens[b];
      n = n > 0 ? n : 0;
      L = p.seqlens[b];
    }
    const int64_t end = rows + block_scan(n, wsum);
    bool fits = L >= 0 && (int64_t)L + n <= (int64_t)p.width * kPage && end <= p.tokens;
    if (fits && (L & (kPage - 1)) != 0 && n > 0) {  // its new rows start in a page it holds
      const int page = p.block_table[(int64_t)b * p.bt_stride + L / kPage];
      fits = page >= 0 && page < p.num_blocks;
    }
    const int need = fits ? pages_up((int64_t)L + n) - pages_up(L) : 0;
    const int64_t upto = asked + block_scan(need, wsum);
    const bool on = fits && (need == 0 || upto <= count);
    const int64_t spent = used + block_scan(on ? need : 0, wsum);
    const int64_t begin = end - n;
    const int begin32 = (int)(begin < INT32_MAX ? begin : INT32_MAX);
    const int first = (int)(on ? upto - need : 0);
    start_sh[tid] = begin32;
    len_sh[tid] = L;
    first_sh[tid] = first;
    on_sh[tid] = on;
    if (b < p.batch) {
      p.cu_new[b] = begin32;
      p.granted[b] = on;
      p.first[b] = first;
      if (on && n > 0) p.seqlens[b] = L + n;
    }
    if (tid == kChunk - 1) {
      start_sh[kChunk] = (int)(end < INT32_MAX ? end : INT32_MAX);
      carry_sh[0] = upto;
      carry_sh[1] = spent;
    }
    __syncthreads();
    if constexpr (ROWS) {
      const int lo = start_sh[0], hi = start_sh[kChunk] < p.tokens ? start_sh[kChunk] : p.tokens;
      for (int t = lo + tid; t < hi; t += kChunk) {
        int i = 0, j = kChunk;  // the last request that starts at or before t
        while (j - i > 1) {
          const int m = (i + j) >> 1;
          if (start_sh[m] <= t) i = m; else j = m;
        }
        place_row(p, t, base + i, start_sh[i], len_sh[i], on_sh[i], first_sh[i], count);
      }
    }
    rows = start_sh[kChunk];
    asked = carry_sh[0];
    used = carry_sh[1];
    __syncthreads();
  }
  if (tid == 0) {
    p.cu_new[p.batch] = (int)rows;
    p.first[p.batch] = count;
    *p.count = count - (int)used;
  }
  if constexpr (ROWS) {
    for (int64_t t = rows + tid; t < p.tokens; t += kChunk) p.slots[t] = p.positions[t] = -1;
  }
}

__global__ __launch_bounds__(256) void mla_slot_rows_kernel(ReserveParams p) {
  const uint32_t row = blockIdx.x * 256 + threadIdx.x;  // past 2^31 in the last workgroup of the longest map
  if (row >= (uint32_t)p.tokens) return;
  const int t = (int)row;
  const int count = p.first[p.batch];
  if (t >= p.cu_new[p.batch]) {
    p.slots[t] = p.positions[t] = -1;
    return;
  }
  int i = 0, j = p.batch;
  while (j - i > 1) {
    const int m = (i + j) >> 1;
    if (p.cu_new[m] <= t) i = m; else j = m;
  }
  const int on = p.granted[i], start = p.cu_new[i];
  place_row(p, t, i, start, p.seqlens[i] - (on ? p.cu_new[i + 1] - start : 0), on, p.first[i], count);
}

struct ReleaseParams {
  int32_t* free;
  int32_t* count;
  int32_t num_blocks;
  const int32_t* block_table;
  int32_t bt_stride, width, batch;
  int32_t* seqlens;
  const int32_t* keep;
};

// Sequence b keeps its first min(L, keep) tokens; the pages behind them go back so that the last page taken
// comes off first again: releasing what a reservation took leaves the stack as it was.  A table entry that is no page of
// the pool is not put back: the first pass counts those that are, and where some are not (rare) the second
// closes the gaps with a prefix sum over the entries.
__global__ __launch_bounds__(kChunk) void mla_release_kernel(ReleaseParams p) {
  __shared__ int64_t wsum[kChunk / 64];
  __shared__ int64_t sum_sh;
  __shared__ int64_t start_sh[kChunk + 1];
  __shared__ int from_sh[kChunk];
  __shared__ int gaps_sh;
  const int tid = threadIdx.x;
  int count = *p.count;
  count = count < 0 ? 0 : (count > p.num_blocks ? p.num_blocks : count);
  auto is_page = [&](int page) { return page >= 0 && page < p.num_blocks; };
  // table entry r of those that the chunk's requests drop
  auto entry = [&](int base, int64_t r) __attribute__((always_inline)) {
    int i = 0, j = kChunk;
    while (j - i > 1) {
      const int m = (i + j) >> 1;
      if (start_sh[m] <= r) i = m; else j = m;
    }
    return p.block_table[(int64_t)(base + i) * p.bt_stride + from_sh[i] + (r - start_sh[i])];
  };
  if (tid == 0) gaps_sh = 0;  // ordered by the scan's barriers
  int keep = 0, held[2] = {-1, -1};  // held: this thread's first entries of a single chunk
  bool cut = false, gaps = false;
  int64_t dropped = 0, missing = 0, total = 0, before = 0;  // missing: of this thread's entries; before: pages put back
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
    for (int base = 0; base < p.batch; base += kChunk) {
      if (pass == 0 || p.batch > kChunk) {  // uniform: a single chunk is kept from the first pass
        const int b = base + tid;
        int64_t from = 0, n = 0;
        cut = false;
        if (b < p.batch) {
          const int64_t most = (int64_t)p.width * kPage;
          const int L = p.seqlens[b];
          keep = p.keep[b];
          keep = keep > 0 ? keep : 0;
          cut = L > keep;
          from = pages_up(keep);
          n = cut ? pages_up(L < most ? L : most) - from : 0;
          n = n > 0 ? n : 0;
        }
        const int64_t end = block_scan(n, wsum);
        start_sh[tid] = end - n;
        from_sh[tid] = (int)from;
        if (tid == kChunk - 1) start_sh[kChunk] = end;
        __syncthreads();
      }
      const int64_t here = start_sh[kChunk];
      if (pass == 0) {
        dropped += here;
        // the first two requested together
        if (tid < here) held[0] = entry(base, tid);
        if (tid + kChunk < here) held[1] = entry(base, tid + kChunk);
        missing += (tid < here && !is_page(held[0])) + (tid + kChunk < here && !is_page(held[1]));
        for (int64_t r = tid + 2 * kChunk; r < here; r += kChunk) missing += !is_page(entry(base, r));
      } else {
        for (int64_t r0 = 0; r0 < here; r0 += kChunk) {  // uniform
          const bool again = p.batch <= kChunk && r0 < 2 * kChunk;  // uniform
          const int page = r0 + tid >= here ? -1 : again ? held[r0 >= kChunk] : entry(base, r0 + tid);
          int64_t rank = before + tid;
          if (gaps) {  // uniform
            rank = before + block_scan(is_page(page) ? 1 : 0, wsum) - 1;
            if (tid == kChunk - 1) sum_sh = rank + 1;
            __syncthreads();
            before = sum_sh;
            __syncthreads();
          } else {
            before += here - r0 < kChunk ? here - r0 : kChunk;
          }
          const int64_t at = count + total - 1 - rank;
          if (is_page(page) && at >= 0 && at < p.num_blocks) p.free[at] = page;
        }
        if (cut) p.seqlens[base + tid] = keep;
      }
      if (p.batch > kChunk) __syncthreads();  // read before the next chunk's
    }
    if (pass == 0) {
      if (missing != 0) gaps_sh = 1;
      __syncthreads();
      gaps = gaps_sh != 0;
      total = dropped;
      if (gaps) {  // uniform
        const int64_t all = block_scan(missing, wsum);
        if (tid == kChunk - 1) sum_sh = all;
        __syncthreads();
        total -= sum_sh;
        __syncthreads();
      }
    }
  }
  if (tid == 0) {
    const int64_t now = count + total;
    *p.count = (int)(now < p.num_blocks ? now : p.num_blocks);
  }
}

// ---------------------------------------------------------------------------------------
// argument checks and launches
// ---------------------------------------------------------------------------------------
static bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

static int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLA_ERR_HIP, std::string(what) + " launch failed: " + hipGetErrorString(e));
  return MLA_OK;
}

// Workgroups of `per` tokens each; 0, with the error left, where they are more than a launch takes (2^32 threads).
static uint32_t groups_of(int64_t tokens, int per) {
  const int64_t n = (tokens + per - 1) / per;
  if (n < (int64_t(1) << 24)) return (uint32_t)n;
  set_error(MLA_ERR_UNSUPPORTED, "too many tokens for one call");
  return 0;
}

// Checks a cache descriptor and fills the kernels' form of it (strides in bytes).
static int check_cache(const mla_kv_cache* c, Cache* k) {
  if (c->format != MLA_KV_NATIVE && c->format != MLA_KV_FP8_E4M3 && c->format != MLA_KV_FP4_E2M1)
    return set_error(MLA_ERR_INVALID, "kv_format must be MLA_KV_NATIVE, MLA_KV_FP8_E4M3 or MLA_KV_FP4_E2M1");
  if (c->dtype != MLA_DTYPE_BF16 && c->dtype != MLA_DTYPE_F16)
    return set_error(MLA_ERR_INVALID, "dtype must be MLA_DTYPE_BF16 or MLA_DTYPE_F16");
  if (c->format != MLA_KV_NATIVE && c->dtype != MLA_DTYPE_BF16)
    return set_error(MLA_ERR_UNSUPPORTED, "the fp8 and fp4 caches hold bf16 tokens");
  if (c->reserved != 0) return set_error(MLA_ERR_INVALID, "reserved must be 0");
  if (c->num_blocks < 1 || c->num_blocks > INT32_MAX / kPage)
    return set_error(MLA_ERR_INVALID, "num_blocks must be in [1, 2^25): a slot is a 32-bit number");
  if (!c->nope || !c->rope || !aligned(c->nope, 16) || !aligned(c->rope, 16))
    return set_error(MLA_ERR_INVALID, "cache pointers must be 16-byte aligned");
  const int64_t s[] = {c->stride_page, c->stride_tok, c->rope_stride_page, c->rope_stride_tok};
  for (int64_t v : s)
    if (v < 0 || v % 8) return set_error(MLA_ERR_INVALID, "strides must be non-negative multiples of 8 elements");
  const int e = c->format == MLA_KV_NATIVE ? 2 : 1;
  k->format = c->format;
  k->f16 = c->dtype == MLA_DTYPE_F16;
  k->tokens = (int64_t)c->num_blocks * kPage;
  k->nope = (uint8_t*)c->nope;
  k->rope = (uint8_t*)c->rope;
  k->scale = (uint8_t*)c->scale;
  k->sp = c->stride_page * e;
  k->st = c->stride_tok * e;
  k->rp = c->rope_stride_page * 2;
  k->rt = c->rope_stride_tok * 2;
  k->cp = c->scale_stride_page;
  k->ct = c->scale_stride_blk;
  if (c->format != MLA_KV_NATIVE) {
    if (c->stride_page % 16 || c->stride_tok % 16)
      return set_error(MLA_ERR_INVALID, "fp8 and fp4 latent strides must be multiples of 16 bytes");
    const int unit = c->format == MLA_KV_FP4_E2M1 ? 16 : 4;
    if (!c->scale || !aligned(c->scale, 16) || c->scale_stride_page < 0 || c->scale_stride_blk < 0 ||
        c->scale_stride_page % unit || c->scale_stride_blk % unit)
      return set_error(MLA_ERR_INVALID, "kv_scale must be 16-byte aligned with non-negative strides of whole 16 bytes");
    if (c->format == MLA_KV_FP8_E4M3) k->cp *= 4, k->ct *= 4;
  }
  return MLA_OK;
}

static int check_rope(const mla_rope* r, int dim) {
  if (!r->freqs || !aligned(r->freqs, 8)) return set_error(MLA_ERR_INVALID, "rope: freqs must be 8-byte aligned and not NULL");
  if (r->layout != MLA_ROPE_INTERLEAVED && r->layout != MLA_ROPE_HALF)
    return set_error(MLA_ERR_INVALID, "rope: layout must be MLA_ROPE_INTERLEAVED or MLA_ROPE_HALF");
  if (r->dim < 2 || r->dim % 2 || r->dim > 2 * kPairs || (dim && r->dim != dim))
    return set_error(MLA_ERR_INVALID, dim ? "rope: dim must be 64 here" : "rope: dim must be even, in [2, 1024]");
  if (!isfinite(r->amp)) return set_error(MLA_ERR_INVALID, "rope: amp must be finite");
  return MLA_OK;
}

template <class E>
static void launch_rope(const RopeParams& k, bool vec, uint32_t grid, hipStream_t st) {
  if (vec)
    hipLaunchKernelGGL((mla_rope_kernel<E, true>), dim3(grid), dim3(256), 0, st, k);
  else
    hipLaunchKernelGGL((mla_rope_kernel<E, false>), dim3(grid), dim3(256), 0, st, k);
}

int append_fp4(const mla_kv_append_args* a, hipStream_t st) {
  SeqAppendParams k{};
  const mla_kv_cache c = {a->kv_format, a->dtype, a->num_blocks, 0, a->kv_nope, a->kv_rope, a->kv_scale,
                          a->kv_stride_page, a->kv_stride_tok, a->kv_rope_stride_page, a->kv_rope_stride_tok,
                          a->kv_scale_stride_page, a->kv_scale_stride_blk};
  const int rc = check_cache(&c, &k.cache);
  if (rc != MLA_OK) return rc;
  k.kv_new = (const uint8_t*)a->kv_new;
  k.n_sb = a->new_stride_b * 2;
  k.n_st = a->new_stride_t * 2;
  k.block_table = a->block_table;
  k.bt_stride = a->block_table_stride;
  k.max_pages = a->max_pages;
  k.n_new = a->n_new;
  k.seqlens = a->cache_seqlens;
  k.status = a->status;
  const int waves = a->n_new < 16 ? a->n_new : 16;
  hipLaunchKernelGGL(mla_append_fp4_kernel, dim3(a->batch), dim3(64 * waves), 0, st, k);
  return launched("kv append");
}

}  // namespace mla_srv

using namespace mla_srv;

extern "C" {

int mla_apply_rope(const mla_rope* rope, const mla_rope_args* a, void* stream) {
  if (!rope || !a) return set_error(MLA_ERR_INVALID, "args is NULL");
  const int rc = check_rope(rope, 0);
  if (rc != MLA_OK) return rc;
  if (a->dtype != MLA_DTYPE_BF16 && a->dtype != MLA_DTYPE_F16 && a->dtype != MLA_DTYPE_F32)
    return set_error(MLA_ERR_INVALID, "dtype must be MLA_DTYPE_BF16, MLA_DTYPE_F16 or MLA_DTYPE_F32");
  if (a->tokens < 0 || a->heads < 0 || a->dim < 1 || a->reserved != 0)
    return set_error(MLA_ERR_INVALID, "tokens and heads must be >= 0, dim >= 1, reserved 0");
  if (a->first < 0 || a->first > a->dim - rope->dim)
    return set_error(MLA_ERR_INVALID, "the rotated dims [first, first + rope.dim) must lie in the head");
  if (a->tokens == 0 || a->heads == 0) return MLA_OK;
  if (!a->x || !a->out || !a->positions) return set_error(MLA_ERR_INVALID, "a required pointer is NULL");
  const int es = a->dtype == MLA_DTYPE_F32 ? 4 : 2;
  if (!aligned(a->x, es) || !aligned(a->out, es) || !aligned(a->positions, 4))
    return set_error(MLA_ERR_INVALID, "x, out and positions must be aligned to their elements");
  if (a->x_stride_t < 0 || a->x_stride_h < 0 || a->o_stride_t < 0 || a->o_stride_h < 0)
    return set_error(MLA_ERR_INVALID, "strides must be non-negative");
  if (a->x == a->out && (a->x_stride_t != a->o_stride_t || a->x_stride_h != a->o_stride_h))
    return set_error(MLA_ERR_INVALID, "in place, the strides of x and out must agree");
  if ((int64_t)a->heads * a->dim > INT32_MAX / 512)
    return set_error(MLA_ERR_UNSUPPORTED, "heads * dim must be below 2^22");
  RopeParams k{};
  k.x = (const uint8_t*)a->x;
  k.out = (uint8_t*)a->out;
  k.x_st = a->x_stride_t * es; k.x_sh = a->x_stride_h * es;
  k.o_st = a->o_stride_t * es; k.o_sh = a->o_stride_h * es;
  k.positions = a->positions;
  k.freqs = rope->freqs;
  k.tokens = a->tokens; k.heads = a->heads; k.dim = a->dim; k.rot = rope->dim; k.first = a->first;
  k.half = rope->layout == MLA_ROPE_HALF;
  k.amp = rope->amp;
  // 16-byte chunks where they fall on whole pairs and every row starts on one
  const int w = 16 / es;
  const bool vec = aligned(a->x, 16) && aligned(a->out, 16) && k.x_st % 16 == 0 && k.x_sh % 16 == 0 && k.o_st % 16 == 0 &&
                   k.o_sh % 16 == 0 && a->dim % w == 0 && a->first % w == 0 && (k.half ? rope->dim / 2 : rope->dim) % w == 0;
  const int pairs = rope->dim / 2;
  // Several tokens a workgroup where there are many (the fewer workgroups wait for positions and frequencies), but
  // 1024 workgroups at least: 4096 tokens x 32 heads 12.7 us; 13.5 with 256 at least, 13.3 with 4096.  With few
  // tokens their heads are split, up to 512 workgroups: 128 tokens x 128 heads 4.8 us (7.3 without, 5.3 with 2048),
  // 16 x 128 3.3 (4.2 with 2048).
  int tile = kPairs / pairs;
  tile = tile < kRopeTile ? tile : kRopeTile;
  while (tile > 1 && ((int64_t)a->tokens + tile - 1) / tile < 1024) tile >>= 1;
  const uint32_t groups = groups_of(a->tokens, tile);
  if (groups == 0) return MLA_ERR_UNSUPPORTED;
  uint32_t split = 1;
  while (groups * split < 512 && 2 * split <= (uint32_t)a->heads) split *= 2;
  k.tile = tile;
  k.split = (int)split;
  const uint32_t grid = groups * split;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == MLA_DTYPE_BF16) launch_rope<Bf16>(k, vec, grid, st);
  else if (a->dtype == MLA_DTYPE_F16) launch_rope<F16>(k, vec, grid, st);
  else launch_rope<F32>(k, vec, grid, st);
  return launched("rope");
}

int mla_kv_append_slots(const mla_kv_cache* cache, const mla_rope* rope, const mla_append_slots_args* a, void* stream) {
  if (!cache || !a) return set_error(MLA_ERR_INVALID, "args is NULL");
  AppendParams k{};
  int rc = check_cache(cache, &k.cache);
  if (rc != MLA_OK) return rc;
  if (rope && (rc = check_rope(rope, kRope)) != MLA_OK) return rc;
  if (a->tokens < 0 || a->heads < 0) return set_error(MLA_ERR_INVALID, "tokens and heads must be >= 0");
  if (a->tokens == 0) return MLA_OK;
  if (!a->kv_new || !a->slots || (rope && !a->positions)) return set_error(MLA_ERR_INVALID, "a required pointer is NULL");
  if (!aligned(a->kv_new, 16) || a->new_stride < 0 || a->new_stride % 8)
    return set_error(MLA_ERR_INVALID, "kv_new must be 16-byte aligned with a stride that is a multiple of 8 elements");
  k.kv_new = (const uint8_t*)a->kv_new;
  k.n_st = a->new_stride * 2;
  k.slots = a->slots;
  k.positions = a->positions;
  if (rope) {
    k.freqs = rope->freqs;
    k.half = rope->layout == MLA_ROPE_HALF;
    k.amp = rope->amp;
  }
  k.tokens = a->tokens;
  if (a->q_pe && a->heads > 0) {
    if (!rope) return set_error(MLA_ERR_INVALID, "q_pe is rotated: it needs a rope");
    const int64_t s[] = {a->pe_stride_t, a->pe_stride_h, a->q_stride_t, a->q_stride_h};
    if (!a->q_rope || !aligned(a->q_pe, 16) || !aligned(a->q_rope, 16))
      return set_error(MLA_ERR_INVALID, "q_pe and q_rope must be 16-byte aligned");
    for (int64_t v : s)
      if (v < 0 || v % 8) return set_error(MLA_ERR_INVALID, "query strides must be non-negative multiples of 8 elements");
    if (a->heads > 65536) return set_error(MLA_ERR_UNSUPPORTED, "heads must be at most 65536");
    k.q_pe = (const uint8_t*)a->q_pe;
    k.q = (uint8_t*)a->q_rope;
    k.pe_st = a->pe_stride_t * 2; k.pe_sh = a->pe_stride_h * 2;
    k.q_st = a->q_stride_t * 2; k.q_sh = a->q_stride_h * 2;
    k.heads = a->heads;
  }
  // 1024 workgroups at least: 1024 tokens x 128 heads 8.2 us, 4096 x 16 6.3 (11.7 and 7.0 with 256 at least, 8.1
  // and 8.6 with 4096)
  int tile = kAppendTile;
  while (tile > 1 && ((int64_t)a->tokens + tile - 1) / tile < 1024) tile >>= 1;
  k.tile = tile;
  const uint32_t groups = groups_of(a->tokens, tile);
  if (groups == 0) return MLA_ERR_UNSUPPORTED;
  const dim3 grid(groups);
  if (k.cache.f16)
    hipLaunchKernelGGL(mla_append_slots_kernel<F16>, grid, dim3(256), 0, (hipStream_t)stream, k);
  else
    hipLaunchKernelGGL(mla_append_slots_kernel<Bf16>, grid, dim3(256), 0, (hipStream_t)stream, k);
  return launched("append by slots");
}

int mla_kv_gather(const mla_kv_cache* cache, const int32_t* slots, int32_t tokens, void* out, int64_t out_stride, void* stream) {
  if (!cache) return set_error(MLA_ERR_INVALID, "args is NULL");
  GatherParams k{};
  const int rc = check_cache(cache, &k.cache);
  if (rc != MLA_OK) return rc;
  if (tokens < 0) return set_error(MLA_ERR_INVALID, "tokens must be >= 0");
  if (tokens == 0) return MLA_OK;
  if (!slots || !out) return set_error(MLA_ERR_INVALID, "a required pointer is NULL");
  if (!aligned(out, 16) || out_stride < MLA_DIM_QK || out_stride % 8)
    return set_error(MLA_ERR_INVALID, "out must be 16-byte aligned with a stride >= 576 that is a multiple of 8 elements");
  k.slots = slots;
  k.out = (uint8_t*)out;
  k.o_st = out_stride * 2;
  k.tokens = tokens;
  const uint32_t groups = groups_of(tokens, 4);
  if (groups == 0) return MLA_ERR_UNSUPPORTED;
  const dim3 grid(groups);
  const hipStream_t st = (hipStream_t)stream;
  if (cache->format == MLA_KV_NATIVE)
    hipLaunchKernelGGL(mla_gather_kernel<MLA_KV_NATIVE>, grid, dim3(256), 0, st, k);
  else if (cache->format == MLA_KV_FP8_E4M3)
    hipLaunchKernelGGL(mla_gather_kernel<MLA_KV_FP8_E4M3>, grid, dim3(256), 0, st, k);
  else
    hipLaunchKernelGGL(mla_gather_kernel<MLA_KV_FP4_E2M1>, grid, dim3(256), 0, st, k);
  return launched("gather");
}

static int check_pool(const mla_page_pool* p) {
  if (!p->free_pages || !p->count || p->num_blocks < 1 || p->num_blocks > INT32_MAX / kPage)
    return set_error(MLA_ERR_INVALID, "pool: free_pages and count must not be NULL, num_blocks in [1, 2^25)");
  if (!p->block_table || !p->cache_seqlens || p->block_table_width < 1 || p->block_table_stride < p->block_table_width ||
      p->block_table_width > (1 << 24))
    return set_error(MLA_ERR_INVALID, "block_table and cache_seqlens must not be NULL, the table's width in [1, min(stride, 2^24)]");
  if (p->batch < 1 || p->batch > 16384) return set_error(MLA_ERR_INVALID, "batch must be in [1, 16384]");
  return MLA_OK;
}

int mla_reserve_pages(const mla_page_pool* pool, const int32_t* new_lens, int32_t tokens, int32_t* slots, int32_t* positions,
                      int32_t* cu_new, int32_t* granted, int32_t* scratch, void* stream) {
  if (!pool) return set_error(MLA_ERR_INVALID, "args is NULL");
  const int rc = check_pool(pool);
  if (rc != MLA_OK) return rc;
  if (tokens < 0) return set_error(MLA_ERR_INVALID, "tokens must be >= 0");
  if (!new_lens || !cu_new || !granted || !scratch || (tokens > 0 && (!slots || !positions)))
    return set_error(MLA_ERR_INVALID, "a required pointer is NULL");
  ReserveParams k{};
  k.free = pool->free_pages;
  k.count = pool->count;
  k.num_blocks = pool->num_blocks;
  k.block_table = pool->block_table;
  k.bt_stride = pool->block_table_stride;
  k.width = pool->block_table_width;
  k.batch = pool->batch;
  k.seqlens = pool->cache_seqlens;
  k.new_lens = new_lens;
  k.tokens = tokens;
  k.slots = slots;
  k.positions = positions;
  k.cu_new = cu_new;
  k.granted = granted;
  k.first = scratch;
  const hipStream_t st = (hipStream_t)stream;
  if (tokens <= kFusedRows) {
    hipLaunchKernelGGL(mla_reserve_kernel<true>, dim3(1), dim3(kChunk), 0, st, k);
  } else {
    hipLaunchKernelGGL(mla_reserve_kernel<false>, dim3(1), dim3(kChunk), 0, st, k);
    hipLaunchKernelGGL(mla_slot_rows_kernel, dim3(((uint32_t)tokens + 255) / 256), dim3(256), 0, st, k);
  }
  return launched("reserve pages");
}

int mla_release_pages(const mla_page_pool* pool, const int32_t* keep_lens, void* stream) {
  if (!pool) return set_error(MLA_ERR_INVALID, "args is NULL");
  const int rc = check_pool(pool);
  if (rc != MLA_OK) return rc;
  if (!keep_lens) return set_error(MLA_ERR_INVALID, "a required pointer is NULL");
  ReleaseParams k{};
  k.free = pool->free_pages;
  k.count = pool->count;
  k.num_blocks = pool->num_blocks;
  k.block_table = pool->block_table;
  k.bt_stride = pool->block_table_stride;
  k.width = pool->block_table_width;
  k.batch = pool->batch;
  k.seqlens = pool->cache_seqlens;
  k.keep = keep_lens;
  hipLaunchKernelGGL(mla_release_kernel, dim3(1), dim3(kChunk), 0, (hipStream_t)stream, k);
  return launched("release pages");
}

}  // extern "C"
