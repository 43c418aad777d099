// The window form of bmx_prefill for few rows (prefill_rows.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "bmx_prefill.h"

namespace bmx {

// query rows (positions times heads of a KV head) the form takes: a lane keeps
// 8 channels of every row's query and sum
constexpr int kRowsMax = 8;

size_t rows_workspace_bytes(const bmx_prefill_args* a);
hipError_t rows_launch(const bmx_prefill_args* a, hipStream_t st);

}  // namespace bmx
