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
// Bound by memory for many rows, by latency for few: row, sum, two barriers.
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

// One row by T threads; 256 / T rows a workgroup where T < 256.
template <class E, int V, int T, int P>
__global__ __launch_bounds__(T < 256 ? 256 : T) void mla_rms_norm_kernel(NormParams p) {
  constexpr int kRows = T < 256 ? 256 / T : 1;
  constexpr int kWaves = T / 64;
  __shared__ float sum_sh[kRows][kWaves];
  const int sub = kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : 0;
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
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if constexpr (kWaves > 1) {
    if ((t & 63) == 0) sum_sh[sub][t >> 6] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum += sum_sh[sub][i];
  }
  if (!on) return;  // a wave belongs to one row
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
  if (pieces <= 64) return launch_norm_as<E, V, 64, 1>(p, st);
  if (pieces <= 128) return launch_norm_as<E, V, 64, 2>(p, st);
  if (pieces <= 256) return launch_norm_as<E, V, 256, 1>(p, st);
  if (pieces <= 512) return launch_norm_as<E, V, 256, 2>(p, st);
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
  if (a->dtype == MLA_DTYPE_BF16) launch_norm_type<Bf16>(k, vec, cus, st);
  else if (a->dtype == MLA_DTYPE_F16) launch_norm_type<F16>(k, vec, cus, st);
  else launch_norm_type<F32>(k, vec, cus, st);
  return launched("rms norm");
}

}  // extern "C"
