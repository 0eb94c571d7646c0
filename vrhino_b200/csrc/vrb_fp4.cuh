// Shared pieces of the microscaled 4-bit formats (layout: include/vrb.h).
#pragma once

#include "vrb_common.cuh"

namespace vrb {

inline int fp4_block(int format) { return format == VRB_NVFP4 ? 16 : 32; }
inline int64_t fp4_row_bytes(int64_t k) { return (k + 31) / 32 * 16; }
// 512-byte scale tiles along k
inline int64_t fp4_block_tiles(int format, int64_t k) {
    const int64_t per_tile = 4 * fp4_block(format);
    return (k + per_tile - 1) / per_tile;
}
// bounded waits of vrb_fp4_linear that ran out on the current device (0 / 1); a synchronising copy
cudaError_t fp4_wait_failures(int* failures);

}  // namespace vrb
