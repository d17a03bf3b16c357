// Windowed prefill: what its launches take.
#pragma once

#include "prefill_common.h"

namespace hipattn {

struct WindowParams : PrefillParams {
  int block_rows;             // rows of a row block
  int n_parts, part_tiles;    // pieces of a row block's keys at most, and 64-key tiles in each
  float *part_acc, *part_ml;  // of piece i of row r and head h, at (i * total_q + r) * Hq + h: d sums; maximum and sum
};

// Block images of the cache, in workgroups of `waves` wavefronts (4 or 8): prefill_window_{8,16,32}.hip.
void launch_window_images_8(const WindowParams &p, int waves, int dtype, hipStream_t stream);
void launch_window_images_16(const WindowParams &p, int waves, int dtype, hipStream_t stream);
void launch_window_images_32(const WindowParams &p, int waves, int dtype, hipStream_t stream);

}  // namespace hipattn
