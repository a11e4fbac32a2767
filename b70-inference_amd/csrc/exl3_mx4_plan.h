// Host-side choices of the MX4 kernels: row blocks and their number. Plain C++ without device code. They follow from the shape
// alone: a call gives the same bits eager and captured.
#pragma once

#include <stdint.h>

#include "exl3_moe.h"

namespace exl3 {

// How an expert's rows are cut: blocks of `rows`, the last one short (whole: a remainder is never cut smaller).
inline BlockCut mx4_cut(int rows) { return {rows, 0, 1}; }

// Blocks of a call of npairs rows over E experts, at most.
inline int64_t mx4_max_blocks(int64_t npairs, int64_t E, int rows) { return npairs / rows + (E < npairs ? E : npairs); }

}  // namespace exl3
