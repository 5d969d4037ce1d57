// mla_tree.h -- the drafted tokens' part of a tree decode, as mla_decode.hip launches it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mla_tree {

constexpr int kMaxNodes = 64;  // a row's mask is one 64-bit word

struct TreeParams {
  const uint16_t* q_nope;
  const uint16_t* q_rope;
  int64_t q_sb, q_ss, q_sh;  // elements
  int64_t qr_sb, qr_ss, qr_sh;
  const uint8_t* nope;
  const uint8_t* rope;
  const uint8_t* scale;
  int64_t sp, st, rp, rt, cp, ct;  // page and token (fp8 scale: block) strides in bytes
  const int32_t* block_table;
  int32_t bt_stride, bt_width, num_blocks;
  int32_t* status;
  const int32_t* prefix;  // [batch] cached tokens that every row sees
  const uint64_t* mask;   // [batch, s_q] bit j: the row sees drafted token j
  const int32_t* splits;  // the schedule's prefix sums over the splits of the prefixes
  int32_t* splits_out;    // the same with one more split a sequence, its last: the drafted tokens
  float* ws_lse;
  float* ws_scale;
  uint16_t* ws_o;
  int32_t batch, s_q, heads, rows;
  int32_t format, f16;
  int32_t pages;     // nonzero: the prefixes' pages too, each a split (splits is not read)
  float scale_log2;
};

bool takes_pages(int64_t batch, int64_t rows, int format, int64_t bt_width, int64_t slots, int cus);
hipError_t launch_tiles(const TreeParams& p, int cus, hipStream_t st);

}  // namespace mla_tree
