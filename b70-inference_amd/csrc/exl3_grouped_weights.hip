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

// The splits' sums in order, added to what is there where that is wanted, one rounding. A thread has four neighbours of a row.
__global__ __launch_bounds__(256) void grouped_reduce_kernel(GroupedArgs g, const float* part, int64_t n4, int64_t stride) {
    const int64_t q4 = n4 / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / q4;
    if (row >= (int64_t)g.E * g.m) return;
    const int n = 4 * (int)(i - row * q4);
    const float* p = part + row * n4 + n;
    f4_t v = ldg(reinterpret_cast<const f4_t*>(p));
    for (int s0 = 1; s0 < g.splits; s0 += 4) {                 // four loads under way
        f4_t t[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) t[s] = ldg(reinterpret_cast<const f4_t*>(p + (s0 + s < g.splits ? s0 + s : s0) * stride));
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] += s0 + s < g.splits ? t[s][q] : 0.f;
    }
    const int64_t e = row / g.m, o = e * g.out_es + (row - e * g.m) * g.out_ld + n;
    for (int q = 0; q < 4 && n + q < g.n; ++q)
        store_as(g.out, o + q, v[q] + (g.accumulate ? load_as(g.out, o + q, g.out_dtype) : 0.f), g.out_dtype);
}

int grouped_reduce(const GroupedArgs& g, const float* part, int64_t n4, int64_t stride, hipStream_t st) {
    const int64_t wgs = ((int64_t)g.E * g.m * (n4 / 4) + 255) / 256;
    EXL3_CHECK_ARG(wgs <= kMx4Grid, "grouped_reduce: grid too large");
    GROUPED_LAUNCH("grouped_reduce", grouped_reduce_kernel, dim3((unsigned)wgs), dim3(256), g.accumulate, st, g, part, n4, stride);
    return EXL3_OK;
}

int grouped_weights(const GroupedArgs& g, int dtype, int tile, hipStream_t st) {
    return dtype == EXL3_F16 ? launch<kRowF16>(g, tile, st) : launch<kRowBF16>(g, tile, st);
}

}  // namespace exl3
