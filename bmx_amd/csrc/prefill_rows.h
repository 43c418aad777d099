// The window form of bmx_prefill for few rows (prefill_rows.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "bmx_prefill.h"

namespace bmx {

// query rows (positions times heads of a KV head) the form takes, 16 a workgroup: a
// window of 4,096 bf16 keys, 8 heads, takes 20 rows 12.1 us (in the row tiles' form
// 24.1) and 64 rows 16.9 (26.7), one of 300 keys 8.7 and 8.8 (16.5, 17.3); only
// blocks that all walk a long window lose (64 rows over 32,000 keys 79 and 74)
constexpr int kRowsMax = 64;

size_t rows_workspace_bytes(const bmx_prefill_args* a);
hipError_t rows_launch(const bmx_prefill_args* a, hipStream_t st);

}  // namespace bmx
