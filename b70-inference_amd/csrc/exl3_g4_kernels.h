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
        return g4_scale((uint32_t)(s >> (16 * i)) & 0xFFFFu, bf16, in);
    }
    __device__ __forceinline__ uint32_t zero(int i) const { return g4_zero<XT, Z>(Z ? z >> (8 * i) & 15 : 8); }
};

// ------------------------------------------------------------------------------------------------ few rows
// Blocks of up to 16 rows; tiles of 16 weight rows whose inputs the waves of a workgroup share, groups of 512 (four chunks) in turn,
// added in order through LDS. A group's weights and scales are asked for as soon as those of the one before are used, the next tile's
// behind the last.
//   XL: x lies in LDS, and eight waves go round a tile's groups: two workgroups to a CU, one of which works while the other waits
//   for its barrier (replayed from a graph, with and without: ten rows of 512 experts of 2048 -> 1024 7.6 and 7.9 us, six rows of
//   4096 -> 4096 7.7 and 7.9, one row of it 5.9 and 5.6).
//   Not XL, where x leaves room for one workgroup: a wave has one group of every tile, whose x stays in its registers.
// Bound by the weights' bytes (6 rows of 5376 -> 21504, fp16 with zeros: 61 MB in 20.7 us, 3.0 TB/s) and by the instructions that take
// the codes apart (9 us of each SIMD), for small matrices by the chain of launch, load, sum and store.
constexpr int kG4Waves = 16, kG4Slice = 512;
// Tiles between two barriers, each added by another wave: where all waves of a CU wait for one barrier (6 rows of 5376 -> 21504 with one
// tile 23.8 us, with two 21.1, with three 21.2; 6 rows of 4096 -> 21504 19.8 and 19.4).
__host__ __device__ constexpr int g4_tiles_held(bool xl) { return xl ? 1 : 3; }
constexpr int kG4Lds = 163840;         // of a CU

// Bytes from row to row of x in LDS: whole chunks, and 16 bytes to spread the rows over the banks.
__host__ __device__ constexpr int64_t g4_x_stride(int64_t k) { return (k + 127) / 128 * 256 + 16; }

template <int XT, int SG, bool Z, bool XL>
__global__ __launch_bounds__(XL ? 512 : 1024, 4) void g4_decode_kernel(G4Args g, int split) {
    extern __shared__ f4_t red[];
    constexpr int kTiles = g4_tiles_held(XL);
    const int lane = threadIdx.x & 63, l = lane & 15, q4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
              waves = blockDim.x >> 6;
    const unsigned slot = blockIdx.x / (unsigned)split, first = blockIdx.x - slot * (unsigned)split;
    const GroupSlot s = g4_slot<16>(g, slot);
    if (s.rows == 0 || (s.e == g.E && !g.rest)) return;
    const int tiles = (g.n + 15) / 16, kb = g.k / 32, groups = (kb + 15) / 16;
    if (s.e == g.E) {                                          // rows of no expert
        for (int tile = first; tile < tiles; tile += split)
            if (wave == 0)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (4 * q4 + q < s.rows && 16 * tile + l < g.n)
                        store_as(g.out, (s.row + 4 * q4 + q) * g.out_ld + 16 * tile + l, 0.f, g.out_dtype);
        return;
    }
    // a tile's weights and scales; a chunk's are asked for anew for the next tile as soon as they are used
    const int64_t row0 = (int64_t)s.e * g.n, rows = (int64_t)g.E * g.n;
    const uint32_t off = (uint32_t)l * (uint32_t)(kb * 16) + 16 * q4;
    typedef G4Scales<XT, SG, Z> S;
    struct Tile {
        __amdgpu_buffer_rsrc_t w;
        G4Base b;
        int srow;
        __device__ __forceinline__ Tile(const G4Args& g, int64_t row0, int64_t rows, int n0, int kb, int l)
            : b(g, row0 + n0, rows) {
            const int left = g.n - n0 < 16 ? g.n - n0 : 16;
            w = mx4_rsrc(g.codes + (row0 + n0) * (kb * 16), (int64_t)left * kb * 16);
            srow = (l < left ? l : left - 1) * g.groups;
        }
    };
    const auto load_w = [&](const Tile& d, int c) { return mx4_buffer16(d.w, 4 * c + q4 < kb ? off + 64 * c : kMx4Out); };
    // Scales: lane group u brings the four of chunks 4 / SG u .. of its row and lays them out in LDS as they are used, [16][16 rows].
    u32x4_t w[4];
    S raw;
    const int set = q4 < SG ? q4 : SG - 1, cs = set * (4 / SG);
    float* const ls = reinterpret_cast<float*>(red + (waves > 1 ? 2 * kTiles * waves * 64 : 0)) + wave * (Z ? 512 : 256) + l;
    uint32_t* const lz = reinterpret_cast<uint32_t*>(ls + 256);
    {
        const Tile d(g, row0, rows, first * 16, kb, l);
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = load_w(d, 4 * wave + u);
        raw.load(g, d.b, d.srow, 4 * wave + cs);
    }
    // x: of lane l the row l, inputs 32 v + 8 (lane >> 4) of each chunk; 0 behind the row's end
    u32x4_t x[XL ? 1 : 4][4];
    const int stride = (int)g4_x_stride(g.k);
    char* const xl = reinterpret_cast<char*>(red + (waves > 1 ? 2 * kTiles * waves * 64 : 0)) + waves * (Z ? 2048 : 1024);
    const __amdgpu_buffer_rsrc_t xr = mx4_rsrc(reinterpret_cast<const uint8_t*>(g.x + s.row * g.x_ld), 0xE0000000LL);
    if constexpr (XL) {
        // all rows' units in one run over the threads, eight loads under way
        const unsigned units = (unsigned)(kb + 3) / 4 * 16, all = units * s.rows, T = blockDim.x;
        const unsigned dr = T / units, dc = T - dr * units;
        unsigned r = threadIdx.x / units, c = threadIdx.x - r * units;
        for (unsigned u0 = threadIdx.x; u0 < all; u0 += 8 * T) {
            u32x4_t v[8];
            unsigned to[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = mx4_buffer16(xr, u0 + i * T < all && c < (unsigned)kb * 4 ? r * (uint32_t)(2 * g.x_ld) + 16 * c : kMx4Out);
                to[i] = r * stride + 16 * c;
                r += dr;
                c += dc;
                if (c >= units) {
                    c -= units;
                    ++r;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (u0 + i * T < all) *reinterpret_cast<u32x4_t*>(xl + to[i]) = v[i];
        }
        __syncthreads();
    } else {
        const uint32_t at = (uint32_t)(l < s.rows ? l : 0) * (uint32_t)(2 * g.x_ld) + 1024 * wave + 16 * q4;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int v = 0; v < 4; ++v) x[u][v] = mx4_buffer16(xr, 4 * (4 * wave + u) + v < kb ? at + 256 * u + 64 * v : kMx4Out);
    }
    const char* const xrow = xl + (l < s.rows ? l : s.rows - 1) * stride + 16 * q4;
    int buf = 0, held = 0;                                     // tiles in LDS behind the last barrier
#pragma unroll 1
    for (int tile = first; tile < tiles; tile += split) {
        f4_t acc = {};
        int n0 = 16 * tile;
#pragma unroll 1
        for (int gi = wave; gi < groups; gi += waves) {        // (waves <= groups: every wave has a group of every tile)
            // the next group: this tile's, or the next tile's first (the last tile's is read again and not used)
            const bool on = gi + waves < groups;
            const int c0 = 4 * gi, cn = 4 * (on ? gi + waves : wave), tn = on || tile + split >= tiles ? tile : tile + split;
            const Tile next(g, row0, rows, 16 * tn, kb, l);
            {
                const Tile d(g, row0, rows, 16 * tile, kb, l);
                raw.fix(g, d.b, d.srow, c0 + cs);
            }
            g4_wave_sync();                                    // the group before is read
            if (q4 < SG)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const int k = S::index(g, c0 + cs, c0 + cs + p / SG, p % SG);
                    ls[(4 * set + p) * 16] = raw.scale(k, S::first(g, c0 + cs) + k < g.groups, g.scale_bf16);
                    if constexpr (Z) lz[(4 * set + p) * 16] = raw.zero(k);
                }
            raw.load(g, next.b, next.srow, cn + cs);
            g4_wave_sync();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (4 * (c0 + u) < kb) {                       // uniform
                    if constexpr (XL)
#pragma unroll
                        for (int v = 0; v < 4; ++v) x[0][v] = *reinterpret_cast<const u32x4_t*>(xrow + 256 * (c0 + u) + 64 * v);
                    g4_turn(w[u]);
#pragma unroll
                    for (int i = 0; i < SG; ++i) {
                        const float f = ls[(u * SG + i) * 16];
                        const uint32_t zero = Z ? lz[(u * SG + i) * 16] : g4_zero<XT, Z>(8);
                        f4_t part = {};
#pragma unroll
                        for (int v = i * (4 / SG); v < (i + 1) * (4 / SG); ++v)
                            part = mfma16<XT>(x[XL ? 0 : u][v], g4_frag<XT, Z>(w[u][v], zero), part);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(f, part[e], acc[e]);
                    }
                }
                w[u] = load_w(next, cn + u);
            }
        }
        if (waves > 1) {
            red[((buf * kTiles + held) * waves + wave) * 64 + lane] = acc;
            if (held + 1 < kTiles && tile + split < tiles) {
                ++held;
                continue;
            }
            __syncthreads();
            const int back = held - wave;                      // each of these tiles is a wave's
            const f4_t* o = red + (buf * kTiles + wave) * waves * 64;
            held = 0;
            buf ^= 1;                                          // two, so that one barrier is enough
            if (back < 0) continue;
            n0 -= 16 * back * split;
            acc = o[lane];
            for (int w0 = 1; w0 < waves; w0 += 5) {            // five reads under way
                f4_t t[5];
#pragma unroll
                for (int i = 0; i < 5; ++i) t[i] = o[(w0 + i < waves ? w0 + i : w0) * 64 + lane];
#pragma unroll
                for (int i = 0; i < 5; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] += w0 + i < waves ? t[i][e] : 0.f;
            }
        }
        const int n = n0 + l;
        if (n >= g.n) continue;
        const float b = g.bias ? ldg(g.bias + n) : 0.f;
        int m = 4 * q4;
        asm volatile("" : "+v"(m));                            // (the rows' addresses are worked out here, not kept)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (m + e < s.rows) store_as(g.out, (s.row + m + e) * g.out_ld + n, __builtin_fmaf(kG4Factor<XT, Z>, acc[e], b), g.out_dtype);
    }
}

template <int XT, int SG, bool Z>
static int launch_g4_decode(G4Args g, hipStream_t st) {
    const int groups = (g.k + kG4Slice - 1) / kG4Slice, few = g.T < 16 ? g.T : 16;
    const int64_t own = Z ? 2048 : 1024, xb = few * g4_x_stride(g.k);
    // x in LDS where two workgroups of eight waves fit a CU: as few rounds of groups as eight waves take, with as few waves as do them
    int waves = (groups + 7) / 8;
    waves = (groups + waves - 1) / waves;
    const bool xl = 2 * (xb + waves * (2048 + own)) <= kG4Lds;
    if (!xl) waves = groups;
    EXL3_CHECK_ARG(waves <= kG4Waves, "g4: too many inputs");
    const int64_t lds = (waves > 1 ? 2 * g4_tiles_held(xl) * waves * 1024 : 0) + waves * own + (xl ? xb : 0);
    g.slots = (int)(g.ends ? group_slots(g.T, g.E, 16, g.rest) : (g.T + 15) / 16);
    const int64_t by_lds = kG4Lds / lds, by_waves = 16 / waves, fit = by_lds < by_waves ? by_lds : by_waves;
    const int64_t split = group_split(g.T, g.E, (g.n + 15) / 16, waves, fit > 4 ? 4 : fit, 8, (double)g.k * 8 / 12e3);
    EXL3_CHECK_ARG(g.slots * split <= kMx4Grid / 4, "g4: grid too large");
    if (xl)
        EXL3_LAUNCH("g4_decode", (g4_decode_kernel<XT, SG, Z, true>), dim3((unsigned)(g.slots * split)), dim3(64 * waves), (size_t)lds, st,
                    g, (int)split);
    else
        EXL3_LAUNCH("g4_decode", (g4_decode_kernel<XT, SG, Z, false>), dim3((unsigned)(g.slots * split)), dim3(64 * waves), (size_t)lds,
                    st, g, (int)split);
    return EXL3_OK;
}

// ------------------------------------------------------------------------------------------------ many rows
// Tiles of BM rows x 256 outputs, 64 of them per wave, in steps of a chunk; the steps of the last tiles, or of all, may be split over
// workgroups, whose sums g4_reduce_kernel adds. x goes to LDS by direct loads (eight values a unit, permuted as in the 16-bit products), the weights
// straight to the registers of the one wave that converts them, the scales four at a time. Tile j of a wave has outputs
// 4 (lane & 15) + j, so that a lane stores four neighbours. JN of the four are converted and multiplied at a time, and
// their registers take the next step's weights: two, or one for smaller tiles of experts, whose tiles are many and of few steps, so
// that one workgroup more fits a CU and hides their starts (10240 rows over 512 experts of 640 -> 2560 168 -> 150 us, 40000 rows 333 ->
// 289; of 2560 -> 640 151 -> 154; a linear's splits are slower by it, and so are groups of 32 and 64, whose products are short then).
template <int XT, int SG, bool Z, int BM, int OCC, int JN>
__global__ __launch_bounds__(256, OCC) void g4_wide_kernel(G4Args g) {
    constexpr int kUnits = BM * 16, kLoads = kUnits / 256, RT = BM / 16;
    __shared__ u32x4_t lds[2 * kUnits + 4 * (Z ? 128 : 64)];   // x, and the waves' scales and zeros
    const int t = threadIdx.x, lane = t & 63, l = lane & 15, q4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const unsigned nnt = (unsigned)((g.n + 255) / 256), whole = (unsigned)g.whole, tail = g.slots * nnt - whole,
                   id = grouped_place(kChunk, blockIdx.x);
    if (id >= whole + tail * g.splits) return;
    const bool parted = id >= whole;                           // uniform
    const unsigned sp = parted ? (id - whole) / tail : 0, tile = parted ? id - sp * tail : id;
    unsigned mt, nt;
    grouped_tile(tile, (unsigned)g.slots, nnt, mt, nt);
    const GroupSlot s = g4_slot<BM>(g, mt);
    if (s.rows == 0 || (s.e == g.E && !g.rest)) return;
    const int kb = g.k / 32, c0 = (int)sp * g.spc, end = !parted || (kb + 3) / 4 - c0 < g.spc ? (kb + 3) / 4 : c0 + g.spc,
              steps = s.e == g.E ? 0 : end - c0;
    const int64_t n0 = (int64_t)nt * 256 + 64 * wave, row0 = (int64_t)(s.e < g.E ? s.e : 0) * g.n, rows = (int64_t)g.E * g.n;
    f4_t acc[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f4_t{};
    if (steps > 0) {
        // x: unit u of a row lies at u ^ (row & 15)
        const uint8_t* xp = reinterpret_cast<const uint8_t*>(g.x + s.row * g.x_ld);
        const int xu = (t & 15) ^ (t >> 4 & 15);               // this thread's unit, alike in all its rows (t >> 4) + 16 i
        const uint32_t xo = (uint32_t)(t >> 4) * (uint32_t)(2 * g.x_ld) + 16 * xu, xs = 32 * (uint32_t)g.x_ld;
        const auto load_x = [&](int c) {                       // (past the last: zeros)
            const __amdgpu_buffer_rsrc_t xr = mx4_rsrc(xp + (c < end ? (int64_t)c * 256 : 0), 0xE0000000LL);
            const int have = c < end && 4 * c + (xu >> 2) < kb ? s.rows - (t >> 4) : 0;
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                lds_load16(xr, 16 * i < have ? xo + i * xs : kMx4Out, lds + ((c - c0) & 1) * kUnits + wave * 64 + i * 256);
        };
        const int64_t left = g.n - n0 < 64 ? (g.n > n0 ? g.n - n0 : 0) : 64;
        const __amdgpu_buffer_rsrc_t wr = mx4_rsrc(g.codes + (row0 + (left > 0 ? n0 : 0)) * (kb * 16), left * kb * 16);
        const uint32_t wo = (uint32_t)(4 * l) * (uint32_t)(kb * 16) + 16 * q4;
        const auto next_w = [&](int c, int j) {
            return mx4_buffer16(wr, c < end && 4 * c + q4 < kb ? wo + j * kb * 16 + 64 * c : kMx4Out);
        };
        // Scales and zeros: lane r brings four of the wave's row r and lays them out in LDS as they are used, [four][64 rows].
        const G4Base sb(g, row0 + (left > 0 ? n0 : 0), rows);
        const int srow = (lane < left ? lane : left > 0 ? (int)left - 1 : 0) * g.groups;
        typedef G4Scales<XT, SG, Z> S;
        S raw;
        float* const ls = reinterpret_cast<float*>(lds + 2 * kUnits) + wave * (Z ? 512 : 256);
        uint32_t* const lz = reinterpret_cast<uint32_t*>(ls + 256);
        u32x4_t w[4];
        raw.load(g, sb, srow, c0);
        load_x(c0);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = next_w(c0, j);
        for (int c = c0; c < end; ++c) {
            __builtin_amdgcn_s_waitcnt(0x0070);                // vmcnt(0) lgkmcnt(0)
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            const int at = (c - c0) % (4 / SG) * SG;
            if (SG == 4 || at == 0) {                          // uniform
                raw.fix(g, sb, srow, c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = S::index(g, c, c + i / SG, i % SG);
                    ls[64 * i + lane] = raw.scale(k, S::first(g, c) + k < g.groups, g.scale_bf16);
                    if constexpr (Z) lz[64 * i + lane] = raw.zero(k);
                }
                raw.load(g, sb, srow, c + 4 / SG);             // (past the last: not used)
                g4_wave_sync();
            }
            load_x(c + 1);
            const u32x4_t* xb = lds + ((c - c0) & 1) * kUnits;
            const auto read_x = [&](int r, u32x4_t (&x)[4]) {
#pragma unroll
                for (int v = 0; v < 4; ++v) x[v] = xb[(16 * r + l) * 16 + ((4 * v + q4) ^ l)];
            };
#pragma unroll
            for (int jp = 0; jp < 4; jp += JN) {
                u32x4_t f[JN][4], x[2][4];
                read_x(0, x[0]);
                float scale[SG][JN];
                uint32_t zero[SG][JN];
#pragma unroll
                for (int i = 0; i < SG; ++i)
#pragma unroll
                    for (int j = 0; j < JN; ++j) {
                        scale[i][j] = ls[64 * (at + i) + 4 * l + jp + j];
                        zero[i][j] = Z ? lz[64 * (at + i) + 4 * l + jp + j] : g4_zero<XT, Z>(8);
                    }
#pragma unroll
                for (int j = 0; j < JN; ++j) {
                    g4_turn(w[jp + j]);
#pragma unroll
                    for (int v = 0; v < 4; ++v) f[j][v] = g4_frag<XT, Z>(w[jp + j][v], zero[v / (4 / SG)][j]);
                    w[jp + j] = next_w(c + 1, jp + j);
                }
                __builtin_amdgcn_s_setprio(1);                 // the other waves convert meanwhile
                __builtin_amdgcn_sched_barrier(0);
                // a product's sums are scaled behind the next one's MFMAs, where there are registers for it
                constexpr bool kLate = SG == 1 || BM < 128;
                f4_t part[kLate ? 2 : 1][JN];
                const auto scaled = [&](int q) {
#pragma unroll
                    for (int j = 0; j < JN; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[q / SG][jp + j][e] = __builtin_fmaf(scale[q % SG][j], part[kLate ? q & 1 : 0][j][e], acc[q / SG][jp + j][e]);
                };
#pragma unroll
                for (int q = 0; q < RT * SG; ++q) {
                    constexpr int V = 4 / SG;
                    const int r = q / SG;
                    if (q % SG == 0 && r + 1 < RT) read_x(r + 1, x[(r + 1) & 1]);
#pragma unroll
                    for (int v = q % SG * V; v < (q % SG + 1) * V; ++v)
#pragma unroll
                        for (int j = 0; j < JN; ++j)
                            part[kLate ? q & 1 : 0][j] = mfma16<XT>(x[r & 1][v], f[j][v], v == q % SG * V ? f4_t{} : part[kLate ? q & 1 : 0][j]);
                    if (!kLate) scaled(q);
                    else if (q > 0) scaled(q - 1);
                    if (kLate || q % SG == SG - 1) __builtin_amdgcn_sched_barrier(0);
                }
                if (kLate) scaled(RT * SG - 1);
                __builtin_amdgcn_s_setprio(0);
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
            constexpr float k = kG4Factor<XT, Z>;
            if (m >= s.rows) continue;
            const f4_t v = {k * acc[r][0][e], k * acc[r][1][e], k * acc[r][2][e], k * acc[r][3][e]};
            if (parted && g.splits > 1) *reinterpret_cast<f4_t*>(g.part + ((int64_t)(sp * tail + tile - whole) * g.part_rows + m) * 256 + 64 * wave + 4 * l) = v;
            else g4_store4(g, s.row + m, n0 + 4 * l, v);
        }
}

template <int XT, int SG, bool Z, int BM, int OCC, int JN>
static int launch_g4_wide(G4Args g, hipStream_t st) {
    g.slots = (int)(g.ends ? group_slots(g.T, g.E, BM, g.rest) : (g.T + BM - 1) / BM);
    const int64_t all = (int64_t)g.slots * ((g.n + 255) / 256), tiles = g.whole + (all - g.whole) * g.splits;
    constexpr int64_t kRound = 8 * kChunk;
    EXL3_CHECK_ARG(tiles <= kMx4Grid - kRound, "g4: grid too large");
    EXL3_LAUNCH("g4_wide", (g4_wide_kernel<XT, SG, Z, BM, OCC, JN>), dim3((unsigned)((tiles + kRound - 1) / kRound * kRound)), dim3(256), 0,
                st, g);
    return EXL3_OK;
}

template <int XT, int SG, bool Z>
static int launch_g4(const G4Args& g, int tile, hipStream_t st) {
    if (tile == 0) return launch_g4_decode<XT, SG, Z>(g, st);
    if constexpr (SG == 1)
        if (g.ends && tile < 3) return tile == 1 ? launch_g4_wide<XT, SG, Z, 32, 4, 1>(g, st) : launch_g4_wide<XT, SG, Z, 64, 3, 1>(g, st);
    return tile == 1 ? launch_g4_wide<XT, SG, Z, 32, 3, 2>(g, st) : tile == 2 ? launch_g4_wide<XT, SG, Z, 64, 2, 2>(g, st)
                                                                              : launch_g4_wide<XT, SG, Z, 128, 2, 2>(g, st);
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
