// Products of fp16 rows with 4-bit weights and group scales.
#include "exl3_g4_kernels.h"

namespace exl3 {

int g4_run_f16(const G4Args& g, int group, int tile, hipStream_t st) { return launch_g4<kRowF16>(g, group, tile, st); }

}  // namespace exl3
