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

// Slot rows up to which one workgroup reserves pages and fills the map in one launch.
constexpr int kFusedRows = 4096;

}  // namespace mla_srv
