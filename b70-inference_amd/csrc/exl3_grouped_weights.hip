// The weights' gradient of products grouped by expert: both operands lie across the contraction.
#include "exl3_grouped_tile.h"

namespace exl3 {

template <int XT>
static int launch(const GroupedArgs& g, int tile, hipStream_t st) {
    const char* name = "grouped_weights";
    switch (tile) {
        case kTile256: return launch_grouped<XT, kGroupWeights, true, 256, 256, 2, 4, 2, 2, true>(name, g, st);
        case kTile128: return launch_grouped<XT, kGroupWeights, true, 128, 128, 2, 2, 2, 2, true>(name, g, st);
        default: return launch_grouped<XT, kGroupWeights, true, 128, 128, 2, 2, 2, 2, false>(name, g, st);
    }
}

int grouped_weights(const GroupedArgs& g, int dtype, int tile, hipStream_t st) {
    return dtype == EXL3_F16 ? launch<kRowF16>(g, tile, st) : launch<kRowBF16>(g, tile, st);
}

}  // namespace exl3
