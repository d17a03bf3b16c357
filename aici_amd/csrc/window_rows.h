// Few new tokens of a sequence over a window of its paged cache, by the kernel of decode rows (window_rows.hip).
#pragma once

#include "prefill_common.h"

namespace hipattn {

// Whether that kernel covers the launch in p (head sizes, lengths) in at most that many parts, the form it would take and about how long that takes.
struct RowsPlan {
  int waves;       // wavefronts of a workgroup, 4 or 8
  int part_pairs;  // block pairs (32 tokens) of a part
  int num_parts;   // 1: no merge, no scratch memory; else fp32 of that many parts x rows x query heads x (head size + 2)
  double us;
};
bool plan_window_rows(const PrefillParams &p, int most_parts, RowsPlan &plan);
void launch_window_rows(const PrefillParams &p, const RowsPlan &plan, int dtype, void *scratch, hipStream_t stream);

}  // namespace hipattn
