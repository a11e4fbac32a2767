// Products grouped by expert for few rows, weights along the contraction: blocks of up to 16 rows, whose inputs stay in registers. A wave
// has SLICE inputs of the block's rows and of one tile of 16 outputs after another; the waves of a workgroup share the inputs and
// are added in order through LDS. A load takes 64 neighbouring bytes of 16 weight rows, eight of them are under way per wave, those of
// the next tile behind the last of this one. Bound by the weights' bytes, of a few experts by the chain of ends, weights, sum and
// store: ten rows of 512 experts of 2048 -> 1024, 42 MB, in 11.4 us as one of a graph's nodes.
#include "exl3_grouped.h"
#include "exl3_grouped_tile.h"

namespace exl3 {

template <int XT, int SLICE>
__global__ __launch_bounds__(1024, 4) void grouped_few_kernel(GroupedArgs g, int split) {
    constexpr int kParts = SLICE / 32, kRing = 8;
    extern __shared__ f4_t red[];
    const int lane = threadIdx.x & 63, l = lane & 15, q4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
              waves = blockDim.x >> 6;
    const unsigned slot = blockIdx.x / (unsigned)split, first = blockIdx.x - slot * (unsigned)split;
    const GroupSlot s = group_slot<16>(g.ends, g.E, g.T, slot);
    if (s.rows == 0 || (s.e == g.E && !g.rest)) return;
    const int tiles = (g.n + 15) / 16, k0 = wave * SLICE + 8 * q4, parts = s.e == g.E ? 0 : kParts;
    const uint16_t* wp = g.b + (s.e < g.E ? s.e : 0) * g.b_es;
    const uint32_t off = (uint32_t)l * (uint32_t)(2 * g.b_ld) + 2 * k0;
    const auto rsrc = [&](int tile) {
        const int left = g.n - tile * 16 < 16 ? g.n - tile * 16 : 16;
        return mx4_rsrc(reinterpret_cast<const uint8_t*>(wp + (int64_t)tile * 16 * g.b_ld), ((left - 1) * g.b_ld + g.c) * 2);
    };
    const auto load = [&](__amdgpu_buffer_rsrc_t r, int u) { return mx4_buffer16(r, u < parts && k0 + 32 * u < g.c ? off + 64 * u : kMx4Out); };
    u32x4_t w[kRing], x[kParts];
    {
        const __amdgpu_buffer_rsrc_t r = rsrc(first);
#pragma unroll
        for (int u = 0; u < kRing; ++u) w[u] = load(r, u);
        const __amdgpu_buffer_rsrc_t xr = mx4_rsrc(reinterpret_cast<const uint8_t*>(g.a + s.row * g.a_ld), 0xE0000000LL);
        const uint32_t at = (uint32_t)(l < s.rows ? l : 0) * (uint32_t)(2 * g.a_ld) + 2 * k0;
#pragma unroll
        for (int u = 0; u < kParts; ++u) x[u] = mx4_buffer16(xr, u < parts && k0 + 32 * u < g.c ? at + 64 * u : kMx4Out);
    }
    int buf = 0;
#pragma unroll 1
    for (int tile = first; tile < tiles; tile += split, buf ^= 1) {
        const __amdgpu_buffer_rsrc_t r = rsrc(tile), rn = rsrc(tile + split < tiles ? tile + split : tile);   // (the last: not used)
        f4_t acc = {};
#pragma unroll
        for (int u = 0; u < kParts; ++u) {
            acc = mfma16<XT>(w[u % kRing], x[u], acc);
            w[u % kRing] = u + kRing < kParts ? load(r, u + kRing) : load(rn, u + kRing - kParts);
        }
        if (waves > 1) {
            f4_t* o = red + buf * waves * 64;                  // two, so that one barrier a tile is enough
            o[wave * 64 + lane] = acc;
            __syncthreads();
            if (wave != 0) continue;
            for (int w0 = 1; w0 < waves; w0 += 5) {            // five reads under way
                f4_t v[5];
#pragma unroll
                for (int i = 0; i < 5; ++i) v[i] = o[(w0 + i < waves ? w0 + i : w0) * 64 + lane];
#pragma unroll
                for (int i = 0; i < 5; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] += w0 + i < waves ? v[i][e] : 0.f;
            }
        }
        int m = l, n = 16 * tile + 4 * q4;
        asm volatile("" : "+v"(m), "+v"(n));                   // (addresses are worked out here, not kept)
        if (m >= s.rows || n >= g.n) continue;
        const int64_t at = (s.row + m) * g.out_ld + n;
        if (g.vec) {
            store4_as(g.out, at, acc, g.out_dtype);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < g.n) store_as(g.out, at + e, acc[e], g.out_dtype);
    }
}

template <int XT, int SLICE>
static int launch(const GroupedArgs& g, hipStream_t st) {
    const int waves = (g.c + SLICE - 1) / SLICE;
    const int64_t slots = group_slots(g.T, g.E, 16, g.rest), tiles = (g.n + 15) / 16;
    const int64_t split = group_split(g.T, g.E, tiles, waves, 16 / waves > 4 ? 4 : 16 / waves, 6, (double)g.c * 32 / 19.5e3);
    EXL3_CHECK_ARG(slots * split <= kMx4Grid / 4, "grouped_few: grid too large");
    EXL3_LAUNCH("grouped_few", (grouped_few_kernel<XT, SLICE>), dim3((unsigned)(slots * split)), dim3(64 * waves),
                (size_t)(waves > 1 ? 2 * waves * 1024 : 0), st, g, (int)split);
    return EXL3_OK;
}

int grouped_rows_few(const GroupedArgs& g, int dtype, hipStream_t st) {
    if (g.c <= 16 * 256) return dtype == EXL3_F16 ? launch<kRowF16, 256>(g, st) : launch<kRowBF16, 256>(g, st);
    return dtype == EXL3_F16 ? launch<kRowF16, 512>(g, st) : launch<kRowBF16, 512>(g, st);
}

}  // namespace exl3
