// Kernels of the products with 4-bit weights and group scales, for one type of rows (XT). SG: scales of a chunk of 128 inputs (4
// with groups of 32, 2 with 64, else 1); Z: zeros are given.
#pragma once

#include "exl3_g4.h"

namespace exl3 {

// A weight row's scales (and zeros) of chunks that a load brings at once: four scales.
template <int XT, int SG, bool Z>
struct G4Scales {
    static constexpr int kChunks = 4 / SG;
    uint64_t s;
    uint32_t z;
    __device__ __forceinline__ void load(const G4Args& g, int64_t row, int64_t rows, int chunk) {
        const int64_t at = row * g.groups, left = (rows - row) * g.groups;
        if (SG > 1 || g.per == 1) {    // uniform
            s = g4_scales4(g.scales + at, SG * chunk, g.groups, left);
            if constexpr (Z) z = g4_zeros4(g.zeros + at, SG * chunk, g.groups, left);
        } else {                       // groups of several chunks: each chunk's own
            s = 0;
            z = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int G = (chunk + i) / g.per;
                if (G < g.groups) {
                    s |= (uint64_t)ldg(g.scales + at + G) << (16 * i);
                    if constexpr (Z) z |= (uint32_t)ldg(g.zeros + at + G) << (8 * i);
                }
            }
        }
    }
    // scale i of the four
    __device__ __forceinline__ float scale(int i, int bf16) const { return g4_scale((uint32_t)(s >> (16 * i)), bf16) * kG4Scale<XT, Z>; }
    __device__ __forceinline__ uint32_t zero(int i) const { return g4_zero<XT, Z>(Z ? z >> (8 * i) & 255 : 8); }
};

// ------------------------------------------------------------------------------------------------ few rows
// Blocks of up to 16 rows. A wave takes 512 inputs (four chunks) of the block's rows, which stay in its registers, and of one tile of
// 16 weight rows after another; the waves of a workgroup share the inputs and are added in order through LDS. Bound by the
// weights' bytes, for small matrices by the chain of load, sum and store.
constexpr int kG4Waves = 16, kG4Slice = 512;

template <int XT, int SG, bool Z>
__global__ __launch_bounds__(1024, 4) void g4_decode_kernel(G4Args g, int split) {
    extern __shared__ f4_t red[];
    const int lane = threadIdx.x & 63, l = lane & 15, q4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
              waves = blockDim.x >> 6;
    const unsigned slot = blockIdx.x / (unsigned)split, first = blockIdx.x - slot * (unsigned)split;
    const GroupSlot s = g4_slot<16>(g, slot);
    if (s.rows == 0 || (s.e == g.E && !g.rest)) return;
    const int tiles = (g.n + 15) / 16, kb = g.k / 32, c0 = 4 * wave;
    if (s.e == g.E) {                                          // rows of no expert
        for (int tile = first; tile < tiles; tile += split)
            if (wave == 0)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (4 * q4 + q < s.rows && 16 * tile + l < g.n)
                        store_as(g.out, (s.row + 4 * q4 + q) * g.out_ld + 16 * tile + l, 0.f, g.out_dtype);
        return;
    }
    const int64_t row0 = (int64_t)s.e * g.n, rows = (int64_t)g.E * g.n;
    const uint8_t* codes = g.codes + row0 * (kb * 16);
    const uint32_t off = (uint32_t)l * (uint32_t)(kb * 16) + 64 * c0 + 16 * q4;
    struct Group {
        u32x4_t w[4];
        G4Scales<XT, SG, Z> sc[SG];
    };
    const auto load = [&](int tile, Group& d) {
        const int64_t n0 = (int64_t)tile * 16, left = g.n - n0 < 16 ? g.n - n0 : 16;
        const __amdgpu_buffer_rsrc_t r = mx4_rsrc(codes + n0 * kb * 16, left * kb * 16);
#pragma unroll
        for (int u = 0; u < 4; ++u) d.w[u] = mx4_buffer16(r, 4 * (c0 + u) + q4 < kb ? off + 64 * u : kMx4Out);
        const int64_t n = n0 + l < g.n ? n0 + l : g.n - 1;
#pragma unroll
        for (int u = 0; u < SG; ++u) d.sc[u].load(g, row0 + n, rows, c0 + u * (4 / SG));
    };
    Group q, nx;
    load(first, q);
    // x: of lane l the row l, inputs 32 v + 8 (lane >> 4) of each chunk; 0 behind the row's end
    u32x4_t x[4][4];
    {
        const __amdgpu_buffer_rsrc_t r = mx4_rsrc(reinterpret_cast<const uint8_t*>(g.x + s.row * g.x_ld), 0xE0000000LL);
        const uint32_t at = (uint32_t)(l < s.rows ? l : 0) * (uint32_t)(2 * g.x_ld) + 256 * c0 + 16 * q4;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int v = 0; v < 4; ++v) x[u][v] = mx4_buffer16(r, 4 * (c0 + u) + v < kb ? at + 256 * u + 64 * v : kMx4Out);
    }
    int buf = 0;
    for (int tile = first; tile < tiles; tile += split, buf ^= 1) {
        if (tile + split < tiles) load(tile + split, nx);
        f4_t acc = {};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (4 * (c0 + u) >= kb) break;                     // uniform
            u32x4_t w = q.w[u];
            g4_turn(w);
#pragma unroll
            for (int i = 0; i < SG; ++i) {
                const int at = u * SG + i;                     // of the sixteen or fewer scales
                const uint32_t zero = q.sc[at / 4].zero(at & 3);
                f4_t part = {};
#pragma unroll
                for (int v = i * (4 / SG); v < (i + 1) * (4 / SG); ++v)
                    part = mfma16<XT>(x[u][v], g4_frag<XT, Z>(w[v], zero), part);
                const float sc = q.sc[at / 4].scale(at & 3, g.scale_bf16);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(sc, part[e], acc[e]);
            }
        }
        q = nx;
        if (waves > 1) {
            f4_t* o = red + buf * waves * 64;                  // two, so that one barrier a tile is enough
            o[wave * 64 + lane] = acc;
            __syncthreads();
            if (wave != 0) continue;
            for (int w = 1; w < waves; ++w) {
                const f4_t t = o[w * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += t[e];
            }
        }
        const int n = 16 * tile + l;
        if (n >= g.n) continue;
        const float b = g.bias ? ldg(g.bias + n) : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * q4 + e < s.rows) store_as(g.out, (s.row + 4 * q4 + e) * g.out_ld + n, acc[e] + b, g.out_dtype);
    }
}

template <int XT, int SG, bool Z>
static int launch_g4_decode(G4Args g, hipStream_t st) {
    const int waves = (g.k + kG4Slice - 1) / kG4Slice;
    g.slots = (int)(g.ends ? group_slots(g.T, g.E, 16, g.rest) : (g.T + 15) / 16);
    // row blocks that have work: no more than there are rows, nor than slots
    const int64_t tiles = (g.n + 15) / 16, room = 256 * (16 / waves > 4 ? 4 : 16 / waves), live = g.slots;
    const int64_t rounds = (tiles * live + room - 1) / room, split = (tiles + rounds - 1) / rounds;
    EXL3_CHECK_ARG(g.slots * split <= kMx4Grid / 4, "g4: grid too large");
    EXL3_LAUNCH("g4_decode", (g4_decode_kernel<XT, SG, Z>), dim3((unsigned)(g.slots * split)), dim3(64 * waves),
                (size_t)(waves > 1 ? 2 * waves * 1024 : 0), st, g, (int)split);
    return EXL3_OK;
}

// ------------------------------------------------------------------------------------------------ many rows
// Tiles of BM rows x 256 outputs, 64 of them per wave, in steps of a chunk. x goes to one of two LDS buffers by direct loads (eight
// values a unit, permuted as in the 16-bit products), the weights straight to the registers of the one wave that converts
// them, both a step ahead. Tile j of a wave has outputs 4 (lane & 15) + j, so that a lane stores four neighbours.
template <int XT, int SG, bool Z, int BM, int OCC>
__global__ __launch_bounds__(256, OCC) void g4_wide_kernel(G4Args g) {
    constexpr int kUnits = BM * 16, kLoads = kUnits / 256, RT = BM / 16;
    __shared__ u32x4_t lds[2 * kUnits];
    const int t = threadIdx.x, lane = t & 63, l = lane & 15, q4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    unsigned mt, nt, sp;
    if (!mx4_tile_of((unsigned)g.slots, (unsigned)((g.n + 255) / 256), 1, mt, nt, sp)) return;
    const GroupSlot s = g4_slot<BM>(g, mt);
    if (s.rows == 0 || (s.e == g.E && !g.rest)) return;
    const int kb = g.k / 32, steps = s.e == g.E ? 0 : (kb + 3) / 4;
    const int64_t n0 = (int64_t)nt * 256 + 64 * wave, row0 = (int64_t)(s.e < g.E ? s.e : 0) * g.n, rows = (int64_t)g.E * g.n;
    f4_t acc[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f4_t{};
    if (steps > 0) {
        // x: unit u of a row lies at u ^ (row & 15)
        const __amdgpu_buffer_rsrc_t xr = mx4_rsrc(reinterpret_cast<const uint8_t*>(g.x + s.row * g.x_ld), 0xE0000000LL);
        uint32_t xo[kLoads];
        const int xu = t & 15;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (t >> 4) + 16 * i;
            xo[i] = r < s.rows ? (uint32_t)r * (uint32_t)(2 * g.x_ld) + 16 * (xu ^ (r & 15)) : kMx4Out;
        }
        const int block = (xu ^ (t >> 4 & 15)) >> 2;           // of the chunk, that this thread's units lie in (alike for all i)
        const auto load_x = [&](int c) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (__attribute__((address_space(3))) void*)(lds + (c & 1) * kUnits + wave * 64 + i * 256),
                                                         16, (int)(4 * c + block < kb && xo[i] != kMx4Out ? xo[i] + 256 * c : kMx4Out), 0, 0, 0);
        };
        const int64_t left = g.n - n0 < 64 ? (g.n > n0 ? g.n - n0 : 0) : 64;
        const __amdgpu_buffer_rsrc_t wr = mx4_rsrc(g.codes + (row0 + (left > 0 ? n0 : 0)) * (kb * 16), left * kb * 16);
        const uint32_t wo = (uint32_t)(4 * l) * (uint32_t)(kb * 16) + 16 * q4;
        const auto load_w = [&](int c, u32x4_t (&w)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = mx4_buffer16(wr, 4 * c + q4 < kb ? wo + j * kb * 16 + 64 * c : kMx4Out);
        };
        G4Scales<XT, SG, Z> sc[4];
        const auto load_s = [&](int c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t n = n0 + 4 * l + j;
                sc[j].load(g, row0 + (n < g.n ? n : g.n - 1), rows, c);
            }
        };
        u32x4_t nx[4];
        load_x(0);
        load_w(0, nx);
        for (int c = 0; c < steps; ++c) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            u32x4_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = nx[j];
            const int at = c % (4 / SG) * SG;
            if (at == 0) load_s(c);
            load_x(c + 1);                                     // (past the last: zeros)
            load_w(c + 1, nx);
#pragma unroll
            for (int j = 0; j < 4; ++j) g4_turn(w[j]);
            const u32x4_t* xb = lds + (c & 1) * kUnits;
#pragma unroll
            for (int i = 0; i < SG; ++i) {
                constexpr int V = 4 / SG;
                u32x4_t f[4][V];
                float scale[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t zero = sc[j].zero(at + i);
#pragma unroll
                    for (int v = 0; v < V; ++v) f[j][v] = g4_frag<XT, Z>(w[j][i * V + v], zero);
                    scale[j] = sc[j].scale(at + i, g.scale_bf16);
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    f4_t part[4] = {};
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const u32x4_t xv = xb[(16 * r + l) * 16 + ((4 * (i * V + v) + q4) ^ l)];
#pragma unroll
                        for (int j = 0; j < 4; ++j) part[j] = mfma16<XT>(xv, f[j][v], part[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[r][j][e] = __builtin_fmaf(scale[j], part[j][e], acc[r][j][e]);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // the LDS is the next workgroup's behind the end
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = 16 * r + 4 * q4 + e;
            if (m < s.rows) g4_store4(g, s.row + m, n0 + 4 * l, f4_t{acc[r][0][e], acc[r][1][e], acc[r][2][e], acc[r][3][e]});
        }
}

template <int XT, int SG, bool Z, int BM, int OCC>
static int launch_g4_wide(G4Args g, hipStream_t st) {
    g.slots = (int)(g.ends ? group_slots(g.T, g.E, BM, g.rest) : (g.T + BM - 1) / BM);
    const int64_t tiles = (int64_t)g.slots * ((g.n + 255) / 256);
    EXL3_CHECK_ARG(tiles <= kMx4Grid - 7, "g4: grid too large");
    EXL3_LAUNCH("g4_wide", (g4_wide_kernel<XT, SG, Z, BM, OCC>), dim3((unsigned)((tiles + 7) & ~7)), dim3(256), 0, st, g);
    return EXL3_OK;
}

template <int XT, int SG, bool Z>
static int launch_g4(const G4Args& g, int tile, hipStream_t st) {
    return tile == 0 ? launch_g4_decode<XT, SG, Z>(g, st) : tile == 1 ? launch_g4_wide<XT, SG, Z, 32, 4>(g, st)
         : tile == 2 ? launch_g4_wide<XT, SG, Z, 64, 3>(g, st) : launch_g4_wide<XT, SG, Z, 128, 2>(g, st);
}

// tile: 0 few rows, 1, 2, 3 blocks of 32, 64, 128 rows
template <int XT>
static int launch_g4(const G4Args& g, int group, int tile, hipStream_t st) {
    if (g.zeros)
        return group == 32 ? launch_g4<XT, 4, true>(g, tile, st) : group == 64 ? launch_g4<XT, 2, true>(g, tile, st)
                                                                              : launch_g4<XT, 1, true>(g, tile, st);
    return group == 32 ? launch_g4<XT, 4, false>(g, tile, st) : group == 64 ? launch_g4<XT, 2, false>(g, tile, st)
                                                                           : launch_g4<XT, 1, false>(g, tile, st);
}

}  // namespace exl3
