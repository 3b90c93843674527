// Column folds shared by the row operators (norm.hip).
#pragma once
#include "common.h"

// out[col] = sum_p part[p][cols] in a fixed order; columns below `split` go to out0, the others to out1 (either may be
// null).  Outputs are rounded once to `dtype`.
int vg_fold_cols(const float* part, int parts, int64_t cols, void* out0, int64_t split, void* out1, int dtype, hipStream_t st);
