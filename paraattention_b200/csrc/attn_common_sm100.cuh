// What the attention kernels share: tile sizes, TMEM columns, when O is rescaled.
#pragma once
#include <cuda.h>
#include <cstdint>

#include "../../include/pa_b200.h"
#include "pa_ptx.cuh"

namespace pa {

// head_dim is a template parameter of the kernel (kD = 64 or 128). Shared-memory slots keep
// the 128-wide size for both: a 64-wide tile is one swizzle atom and fills the first half.
constexpr int kTileM = 128;
constexpr int kTileN = 128;
constexpr int kHalfBytes = 128 * 128;       // 128 rows x 64 elements x 2 B (one swizzle atom wide)
constexpr int kTileBytes = 2 * kHalfBytes;  // 128 x 128 x 2 B
constexpr int kTmemCols = 512;
constexpr uint32_t kColS0 = 0, kColO0 = 256;
// log2-domain growth of the running row maximum that is tolerated before O is rescaled
constexpr float kRescaleThreshold = 8.0f;

}  // namespace pa
