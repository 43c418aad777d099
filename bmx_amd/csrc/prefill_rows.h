// The window form of bmx_prefill for few rows (prefill_rows.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "bmx_prefill.h"

namespace bmx {

// query rows (positions times heads of a KV head) the form takes: the columns
// of one 16x16 matrix product
constexpr int kRowsMax = 16;

size_t rows_workspace_bytes(const bmx_prefill_args* a);
hipError_t rows_launch(const bmx_prefill_args* a, hipStream_t st);

}  // namespace bmx
