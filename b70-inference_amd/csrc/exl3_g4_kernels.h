// Kernels of the products with 4-bit weights and group scales, for one type of rows (XT). SG: scales of a chunk of 128 inputs (4
// with groups of 32, 2 with 64, else 1); Z: zeros are given.
#pragma once

#include "exl3_g4.h"

namespace exl3 {

// Where a wave's scales and zeros begin, and how many lie from there to the tensor's end.
struct G4Base {
    const uint16_t* s;
    const uint8_t* z;
    int left;
    __device__ __forceinline__ G4Base(const G4Args& g, int64_t row, int64_t rows)
        : s(g.scales + row * g.groups), z(g.zeros ? g.zeros + row * g.groups : nullptr) {
        const int64_t n = (rows - row) * g.groups;
        left = (int)(n < 0x40000000 ? n : 0x40000000);
    }
};

// Four scales (and zeros) of a weight row from a chunk's first on: those of 4 / SG chunks. Kept as the loads bring them, so that nothing
// waits where they are asked for; where a load would pass the tensor's end (which has four or more) it begins earlier.
template <int XT, int SG, bool Z>
struct G4Scales {
    uint64_t s;
    uint32_t z;
    __device__ __forceinline__ static int first(const G4Args& g, int chunk) { return SG > 1 || g.per == 1 ? SG * chunk : chunk / g.per; }
    // `row`: where the row's begin, from the base
    __device__ __forceinline__ static int back(const G4Base& b, int at) { return at + 4 > b.left ? at + 4 - b.left : 0; }
    __device__ __forceinline__ void load(const G4Args& g, const G4Base& b, int row, int chunk) {
        typedef uint64_t any8_t __attribute__((aligned(2)));
        typedef uint32_t any4_t __attribute__((aligned(1)));
        const int f = first(g, chunk), at = row + (f < g.groups ? f : 0), from = at - back(b, at);   // (behind the row: not used)
        s = *(const __attribute__((address_space(1))) any8_t*)(b.s + from);
        if constexpr (Z) z = *(const __attribute__((address_space(1))) any4_t*)(b.z + from);
    }
    // behind a load with the same arguments, where they are used: the first scale first
    __device__ __forceinline__ void fix(const G4Args& g, const G4Base& b, int row, int chunk) {
        const int d = back(b, row + first(g, chunk));
        s >>= 16 * (d & 3);
        if constexpr (Z) z >>= 8 * (d & 3);
    }
    // which of them is that of place i of chunk c (of 4 / SG from `chunk`)
    __device__ __forceinline__ static int index(const G4Args& g, int chunk, int c, int i) {
        return SG > 1 || g.per == 1 ? SG * (c - chunk) + i : c / g.per - chunk / g.per;
    }
    // scale i of the four; `in`: 0 for those that are not there, beside x that is 0
    __device__ __forceinline__ float scale(int i, bool in, int bf16) const {
        return in ? g4_scale((uint32_t)(s >> (16 * i)), bf16) * kG4Scale<XT, Z> : 0.f;
    }
    __device__ __forceinline__ uint32_t zero(int i) const { return g4_zero<XT, Z>(Z ? z >> (8 * i) & 15 : 8); }
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
    typedef G4Scales<XT, SG, Z> S;
    const auto load = [&](int tile, Group& d) {
        const int64_t n0 = (int64_t)tile * 16, left = g.n - n0 < 16 ? g.n - n0 : 16;
        const __amdgpu_buffer_rsrc_t r = mx4_rsrc(codes + n0 * kb * 16, left * kb * 16);
#pragma unroll
        for (int u = 0; u < 4; ++u) d.w[u] = mx4_buffer16(r, 4 * (c0 + u) + q4 < kb ? off + 64 * u : kMx4Out);
        const G4Base b(g, row0 + n0, rows);
#pragma unroll
        for (int u = 0; u < SG; ++u) d.sc[u].load(g, b, (l < left ? l : (int)left - 1) * g.groups, c0 + u * (4 / SG));
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
        {
            const int64_t n0 = (int64_t)tile * 16, left = g.n - n0 < 16 ? g.n - n0 : 16;
            const G4Base b(g, row0 + n0, rows);
#pragma unroll
            for (int u = 0; u < SG; ++u) q.sc[u].fix(g, b, (l < left ? l : (int)left - 1) * g.groups, c0 + u * (4 / SG));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (4 * (c0 + u) >= kb) break;                     // uniform
            u32x4_t w = q.w[u];
            g4_turn(w);
#pragma unroll
            for (int i = 0; i < SG; ++i) {
                const int set = u * SG / 4, cf = c0 + set * (4 / SG), at = S::index(g, cf, c0 + u, i);
                const uint32_t zero = q.sc[set].zero(at);
                f4_t part = {};
#pragma unroll
                for (int v = i * (4 / SG); v < (i + 1) * (4 / SG); ++v)
                    part = mfma16<XT>(x[u][v], g4_frag<XT, Z>(w[v], zero), part);
                const float sc = q.sc[set].scale(at, S::first(g, cf) + at < g.groups, g.scale_bf16);
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

// ------------------------------------------------------------------------------------------------ some rows
// Tiles of 16 RT rows x 64 outputs whose chunks go round the waves of a workgroup, which are added in order through LDS: more
// workgroups, and fewer steps for each, than the tiles below have where those leave CUs idle or each wave one step after
// another to wait for. A wave has its own chunks of x, so x comes straight into registers, half a chunk (64 inputs) ahead; the
// weights and scales a chunk ahead. Output j of a wave's four is 4 (lane & 15) + j.
template <int XT, int SG, bool Z, int RT>
__global__ __launch_bounds__(512, 2) void g4_split_kernel(G4Args g) {
    extern __shared__ f4_t red[];
    const int lane = threadIdx.x & 63, l = lane & 15, q4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
              waves = blockDim.x >> 6;
    const unsigned nnt = (unsigned)((g.n + 63) / 64), id = grouped_place(kChunk);
    if (id >= g.slots * nnt) return;
    unsigned mt, nt;
    grouped_tile(id, (unsigned)g.slots, nnt, mt, nt);
    const GroupSlot s = g4_slot<16 * RT>(g, mt);
    if (s.rows == 0 || (s.e == g.E && !g.rest)) return;
    const int kb = g.k / 32, steps = s.e == g.E ? 0 : (kb + 3) / 4;
    const int64_t n0 = (int64_t)nt * 64, row0 = (int64_t)(s.e < g.E ? s.e : 0) * g.n, rows = (int64_t)g.E * g.n;
    const int left = (int)(g.n - n0 < 64 ? g.n - n0 : 64);
    f4_t acc[RT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[r][j] = f4_t{};
    if (wave < steps) {
        const __amdgpu_buffer_rsrc_t wr = mx4_rsrc(g.codes + (row0 + n0) * (kb * 16), (int64_t)left * kb * 16);
        const uint32_t wo = (uint32_t)(4 * l) * (uint32_t)(kb * 16) + 16 * q4;
        const auto load_w = [&](int c, u32x4_t (&w)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = mx4_buffer16(wr, 4 * c + q4 < kb ? wo + j * kb * 16 + 64 * c : kMx4Out);
        };
        const uint8_t* xp = reinterpret_cast<const uint8_t*>(g.x + s.row * g.x_ld);
        uint32_t xo[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int m = 16 * r + l;
            xo[r] = m < s.rows ? (uint32_t)m * (uint32_t)(2 * g.x_ld) + 16 * q4 : kMx4Out;
        }
        const auto load_x = [&](int c, int h, u32x4_t (&x)[RT][2]) {
            const __amdgpu_buffer_rsrc_t xr = mx4_rsrc(xp + (c < steps ? (int64_t)c * 256 : 0), 0xE0000000LL);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int v = 0; v < 2; ++v)
                    x[r][v] = mx4_buffer16(xr, 4 * c + 2 * h + v < kb && xo[r] != kMx4Out ? xo[r] + 128 * h + 64 * v : kMx4Out);
        };
        const G4Base sb(g, row0 + n0, rows);
        typedef G4Scales<XT, SG, Z> S;
        S sc[4], sn[4];
        const auto srow = [&](int j) { return (4 * l + j < left ? 4 * l + j : left - 1) * g.groups; };
        const auto load_s = [&](int c, G4Scales<XT, SG, Z> (&d)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j].load(g, sb, srow(j), c);
        };
        u32x4_t w[4], nw[4], x[RT][2], nx[RT][2];
        load_w(wave, nw);
        load_s(wave, sn);
        load_x(wave, 0, nx);
#pragma unroll 1
        for (int c = wave; c < steps; c += waves) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = nw[j];
                sc[j] = sn[j];
                sc[j].fix(g, sb, srow(j), c);
            }
            const int there = g.groups - S::first(g, c);       // scales from the chunk's first on
            load_w(c + waves, nw);                             // (past the last: zeros)
            load_s(c + waves, sn);
#pragma unroll
            for (int j = 0; j < 4; ++j) g4_turn(w[j]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int v = 0; v < 2; ++v) x[r][v] = nx[r][v];
                load_x(h == 0 ? c : c + waves, 1 - h, nx);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // with groups of 64 and more one scale and zero for both products
                    const int i0 = SG == 4 ? 2 * h : SG == 2 ? h : 0, i1 = SG == 4 ? i0 + 1 : i0;
                    const u32x4_t f0 = g4_frag<XT, Z>(w[j][2 * h], sc[j].zero(i0)), f1 = g4_frag<XT, Z>(w[j][2 * h + 1], sc[j].zero(i1));
                    const float s0 = sc[j].scale(i0, i0 < there, g.scale_bf16), s1 = SG == 4 ? sc[j].scale(i1, i1 < there, g.scale_bf16) : s0;
                    f4_t p[RT];
#pragma unroll
                    for (int r = 0; r < RT; ++r) p[r] = mfma16<XT>(x[r][0], f0, f4_t{});
                    if constexpr (SG == 4) {
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[r][j][e] = __builtin_fmaf(s0, p[r][e], acc[r][j][e]);
                            p[r] = f4_t{};
                        }
                    }
#pragma unroll
                    for (int r = 0; r < RT; ++r) p[r] = mfma16<XT>(x[r][1], f1, p[r]);
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[r][j][e] = __builtin_fmaf(s1, p[r][e], acc[r][j][e]);
                }
            }
        }
    }
    // row 16 r + 4 q4 + e, outputs 4 l ..: piece 4 r + e of a wave; the pieces go round the waves
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            red[(wave * 4 * RT + 4 * r + e) * 64 + lane] = f4_t{acc[r][0][e], acc[r][1][e], acc[r][2][e], acc[r][3][e]};
    __syncthreads();
    for (int p = wave; p < 4 * RT; p += waves) {
        const int m = 16 * (p >> 2) + 4 * q4 + (p & 3);
        f4_t v = red[p * 64 + lane];
        for (int u = 1; u < waves; ++u) {
            const f4_t o = red[(u * 4 * RT + p) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += o[e];
        }
        if (m < s.rows) g4_store4(g, s.row + m, n0 + 4 * l, v);
    }
}

template <int XT, int SG, bool Z, int RT>
static int launch_g4_split(G4Args g, hipStream_t st) {
    g.slots = (int)(g.ends ? group_slots(g.T, g.E, 16 * RT, g.rest) : (g.T + 16 * RT - 1) / (16 * RT));
    const int64_t tiles = (int64_t)g.slots * ((g.n + 63) / 64), steps = (g.k + 127) / 128;
    const int waves = steps < 8 ? (int)steps : 8;
    constexpr int64_t kRound = 8 * kChunk;
    EXL3_CHECK_ARG(tiles <= kMx4Grid / 2 - kRound, "g4: grid too large");
    EXL3_LAUNCH("g4_split", (g4_split_kernel<XT, SG, Z, RT>), dim3((unsigned)((tiles + kRound - 1) / kRound * kRound)), dim3(64 * waves),
                (size_t)waves * 4 * RT * 1024, st, g);
    return EXL3_OK;
}

// ------------------------------------------------------------------------------------------------ many rows
// Tiles of BM rows x 256 outputs, 64 of them per wave, in steps of a chunk. x goes to one of two LDS buffers by direct loads (eight
// values a unit, permuted as in the 16-bit products), the weights straight to the registers of the one wave that converts
// them, both a step ahead, the scales four at a time. Tile j of a wave has outputs 4 (lane & 15) + j, so that a lane stores four
// neighbours. Two of the four are converted and multiplied at a time, over pairs of 16 rows: four chains of MFMAs, whose sums are
// scaled behind the next four.
template <int XT, int SG, bool Z, int BM, int OCC>
__global__ __launch_bounds__(256, OCC) void g4_wide_kernel(G4Args g) {
    constexpr int kUnits = BM * 16, kLoads = kUnits / 256, RT = BM / 16;
    __shared__ u32x4_t lds[2 * kUnits + 4 * (Z ? 128 : 64)];   // x, and the waves' scales and zeros
    const int t = threadIdx.x, lane = t & 63, l = lane & 15, q4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const unsigned nnt = (unsigned)((g.n + 255) / 256), id = grouped_place(kChunk);
    if (id >= g.slots * nnt) return;
    unsigned mt, nt;
    grouped_tile(id, (unsigned)g.slots, nnt, mt, nt);
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
        const uint8_t* xp = reinterpret_cast<const uint8_t*>(g.x + s.row * g.x_ld);
        uint32_t xo[kLoads];
        const int xu = (t & 15) ^ (t >> 4 & 15);               // this thread's unit, alike in all its rows
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (t >> 4) + 16 * i;
            xo[i] = r < s.rows ? (uint32_t)r * (uint32_t)(2 * g.x_ld) + 16 * xu : kMx4Out;
        }
        const auto load_x = [&](int c) {
            const __amdgpu_buffer_rsrc_t xr = mx4_rsrc(xp + (c < steps ? (int64_t)c * 256 : 0), 0xE0000000LL);
            const bool in = 4 * c + (xu >> 2) < kb;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) lds_load16(xr, in ? xo[i] : kMx4Out, lds + (c & 1) * kUnits + wave * 64 + i * 256);
        };
        const int64_t left = g.n - n0 < 64 ? (g.n > n0 ? g.n - n0 : 0) : 64;
        const __amdgpu_buffer_rsrc_t wr = mx4_rsrc(g.codes + (row0 + (left > 0 ? n0 : 0)) * (kb * 16), left * kb * 16);
        const uint32_t wo = (uint32_t)(4 * l) * (uint32_t)(kb * 16) + 16 * q4;
        const auto next_w = [&](int c, int j) {
            return mx4_buffer16(wr, 4 * c + q4 < kb ? wo + j * kb * 16 + 64 * c : kMx4Out);
        };
        // Scales and zeros: lane r brings four of the wave's row r and lays them out in LDS as they are used, [four][64 rows].
        const G4Base sb(g, row0 + (left > 0 ? n0 : 0), rows);
        const int srow = (lane < left ? lane : left > 0 ? (int)left - 1 : 0) * g.groups;
        typedef G4Scales<XT, SG, Z> S;
        S raw;
        float* const ls = reinterpret_cast<float*>(lds + 2 * kUnits) + wave * (Z ? 512 : 256);
        uint32_t* const lz = reinterpret_cast<uint32_t*>(ls + 256);
        u32x4_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = next_w(0, j);
        raw.load(g, sb, srow, 0);
        load_x(0);
        for (int c = 0; c < steps; ++c) {
            __builtin_amdgcn_s_waitcnt(0x0070);                // vmcnt(0) lgkmcnt(0)
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            const int at = c % (4 / SG) * SG;
            if (SG == 4 || at == 0) {                          // uniform
                raw.fix(g, sb, srow, c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = S::index(g, c, c + i / SG, i % SG);
                    ls[64 * i + lane] = raw.scale(k, S::first(g, c) + k < g.groups, g.scale_bf16);
                    if constexpr (Z) lz[64 * i + lane] = raw.zero(k);
                }
                raw.load(g, sb, srow, c + 4 / SG);             // (past the last: not used)
            }
            load_x(c + 1);
            const u32x4_t* xb = lds + (c & 1) * kUnits;
            const auto read_x = [&](int r, u32x4_t (&x)[4]) {
#pragma unroll
                for (int v = 0; v < 4; ++v) x[v] = xb[(16 * r + l) * 16 + ((4 * v + q4) ^ l)];
            };
#pragma unroll
            for (int jp = 0; jp < 4; jp += 2) {
                u32x4_t f[2][4], x[2][4];
                read_x(0, x[0]);
                f2_t scale[SG];
                uint2 zero[SG];
#pragma unroll
                for (int i = 0; i < SG; ++i) {
                    scale[i] = *reinterpret_cast<const f2_t*>(ls + 64 * (at + i) + 4 * l + jp);
                    if constexpr (Z) zero[i] = *reinterpret_cast<const uint2*>(lz + 64 * (at + i) + 4 * l + jp);
                    else zero[i] = make_uint2(g4_zero<XT, Z>(8), g4_zero<XT, Z>(8));
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    g4_turn(w[jp + j]);
#pragma unroll
                    for (int v = 0; v < 4; ++v) f[j][v] = g4_frag<XT, Z>(w[jp + j][v], j ? zero[v / (4 / SG)].y : zero[v / (4 / SG)].x);
                    w[jp + j] = next_w(c + 1, jp + j);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if (r + 1 < RT) read_x(r + 1, x[(r + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < SG; ++i) {
                        constexpr int V = 4 / SG;
                        f4_t part[2] = {};
#pragma unroll
                        for (int v = i * V; v < (i + 1) * V; ++v)
#pragma unroll
                            for (int j = 0; j < 2; ++j) part[j] = mfma16<XT>(x[r & 1][v], f[j][v], part[j]);
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[r][jp + j][e] = __builtin_fmaf(scale[i][j], part[j][e], acc[r][jp + j][e]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_waitcnt(0x0070);                    // the LDS is the next workgroup's behind the end
        asm volatile("" ::: "memory");
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
    constexpr int64_t kRound = 8 * kChunk;
    EXL3_CHECK_ARG(tiles <= kMx4Grid - kRound, "g4: grid too large");
    EXL3_LAUNCH("g4_wide", (g4_wide_kernel<XT, SG, Z, BM, OCC>), dim3((unsigned)((tiles + kRound - 1) / kRound * kRound)), dim3(256), 0,
                st, g);
    return EXL3_OK;
}

template <int XT, int SG, bool Z>
static int launch_g4(const G4Args& g, int tile, hipStream_t st) {
    return tile == 0 ? launch_g4_decode<XT, SG, Z>(g, st) : tile == 1 ? launch_g4_wide<XT, SG, Z, 32, 3>(g, st)
         : tile == 2 ? launch_g4_wide<XT, SG, Z, 64, 2>(g, st) : tile == 3 ? launch_g4_wide<XT, SG, Z, 128, 2>(g, st)
         : tile == 4 ? launch_g4_split<XT, SG, Z, 2>(g, st) : launch_g4_split<XT, SG, Z, 4>(g, st);
}

// tile: 0 few rows, 1, 2, 3 blocks of 32, 64, 128 rows, 4, 5 of 32, 64 rows with split chunks
template <int XT>
static int launch_g4(const G4Args& g, int group, int tile, hipStream_t st) {
    if (g.zeros)
        return group == 32 ? launch_g4<XT, 4, true>(g, tile, st) : group == 64 ? launch_g4<XT, 2, true>(g, tile, st)
                                                                              : launch_g4<XT, 1, true>(g, tile, st);
    return group == 32 ? launch_g4<XT, 4, false>(g, tile, st) : group == 64 ? launch_g4<XT, 2, false>(g, tile, st)
                                                                           : launch_g4<XT, 1, false>(g, tile, st);
}

}  // namespace exl3
