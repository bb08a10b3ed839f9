// Dense states gathered by their parents (fie_reorder_states).
#pragma once

#include "copy.h"
#include "fie_decode.h"

namespace fie {

struct StateBlocks {
    int32_t end[FIE_MAX_STATES];        // workgroups up to and with each tensor
    int32_t chunks[FIE_MAX_STATES];     // of a row
};

// A workgroup a chunk of a row of one tensor.  512 rows of 16 tensors of 131074 bytes, at odd addresses,
// 313 us (5.5 TB/s written and read from each kept row), 4 rows of 8 tensors of 8 KB 3.3.
__global__ __launch_bounds__(kCopyThreads) void k_reorder(const fie_states_args a, const StateBlocks b)
{
    const int block = blockIdx.x;
    int t = 0;
    while (block >= b.end[t]) ++t;
    const int in = block - (t ? b.end[t - 1] : 0);
    const int row = in / b.chunks[t], chunk = in - row * b.chunks[t];
    const fie_state s = a.state[t];
    int64_t from = a.parents[row];
    if (from < 0 || from >= s.rows) from = row;
    copy_chunk((uint8_t*)s.dst + (int64_t)row * s.dst_stride, (const uint8_t*)s.src + from * s.src_stride, s.row_bytes, chunk);
}

}  // namespace fie
