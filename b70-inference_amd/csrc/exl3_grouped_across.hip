// Products grouped by expert whose weights lie across the contraction: the rows' gradient.
#include "exl3_grouped_tile.h"

namespace exl3 {

int grouped_rows_across(const GroupedArgs& g, int dtype, int tile, hipStream_t st) {
    return dtype == EXL3_F16 ? launch_grouped_rows<kRowF16, true>(g, tile, st) : launch_grouped_rows<kRowBF16, true>(g, tile, st);
}

}  // namespace exl3
