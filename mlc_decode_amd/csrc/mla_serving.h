// mla_serving.h -- what mla_decode.hip and mla_serving.hip share (host code).
#pragma once
#include <hip/hip_runtime.h>
#include <string>

#include "mla_decode_amd.h"

namespace mla_srv {

// Leaves `msg` for mla_last_error() on this thread and returns `code`.
int set_error(int code, const std::string& msg);

// mla_kv_append into the 4-bit cache, its other arguments checked.
int append_fp4(const mla_kv_append_args* a, hipStream_t st);

// Slot rows up to which one workgroup reserves pages and fills the map in one launch.  With the release after it, in
// one launch and in two: 128 rows 10.5, 11.9 us; 2048 rows 11.8, 13.7; 4096 rows 14.0, 13.7; 8192 rows 18.4, 13.8.
constexpr int kFusedRows = 4096;

}  // namespace mla_srv
