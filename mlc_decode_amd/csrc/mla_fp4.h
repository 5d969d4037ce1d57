// mla_fp4.h -- the split-KV decode over the 4-bit latent cache, as mla_decode.hip launches it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mla4 {

struct DecodeParams {
  const uint16_t* q_nope;
  const uint16_t* q_rope;
  int64_t q_sb, q_ss, q_sh;
  int64_t qr_sb, qr_ss, qr_sh;
  const uint8_t* codes;  // [page][token][256] (strides in bytes)
  const uint8_t* scale;  // [page][token][16] (strides in bytes)
  const uint16_t* rope;  // [page][token][64] bf16
  int64_t c_sp, c_st, s_sp, s_st, r_sp, r_st;
  const int32_t* block_table;
  int32_t bt_stride, bt_width, num_blocks;
  int32_t* status;
  const int32_t* seqlens;
  const int32_t* splits;
  const int32_t* indices;  // sparse decode, as in mla_decode_args
  int32_t idx_stride, topk;
  int64_t pool_tokens;
  uint16_t* out;
  int64_t o_sb, o_ss, o_sh;
  float* lse;
  float* ws_lse;
  float* ws_scale;
  uint16_t* ws_o;
  int32_t batch, s_q, heads, rows, causal;
  float scale_log2;
};

// Query rows of a workgroup for `rows` = s_q * heads rows, and workgroups of R rows per compute unit.
int rows_per_workgroup(int64_t rows);
int workgroups_per_cu(int R);
// Row tiles of 16 times pages up to which workgroups of 16 rows are the faster ones for any row count.
constexpr int64_t kFewPages = 6144;

hipError_t launch_decode(const DecodeParams& p, const int32_t* sched, int num_parts, int cus, hipStream_t st);

}  // namespace mla4
