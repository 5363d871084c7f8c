// Host helpers shared by the translation units behind the C ABI (defined in pa_api.cu).
#pragma once
#include <cuda.h>
#include <cstdint>

namespace pa_host {

// Records a message for pa_last_error() and returns `code`.
int fail(int code, const char* fmt, ...);
// Streaming multiprocessors of the current device.
int sm_count();
// Tensor map over [chunk][batch][head][row][head_dim], element strides, boxes of box_rows x box_cols elements
// (64: 128-byte swizzle, 32: 64-byte swizzle).
int make_map(CUtensorMap* map, const void* base, int dtype, int head_dim, int rows, int heads, int batch, int chunks,
             int64_t s_row, int64_t s_head, int64_t s_batch, int64_t s_chunk, const char* what, int box_rows = 128, int box_cols = 64);

}  // namespace pa_host
