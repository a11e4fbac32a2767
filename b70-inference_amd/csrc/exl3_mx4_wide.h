// Products of many 16-bit rows with MX4 weights: a workgroup of four waves takes 32 RG rows of x and 64 weight rows (outputs)
// per wave, in steps of 128 k (four blocks). Bound by the MFMAs at 128 rows (RG 4: 2048 cycles of them per wave and step
// against 64 conversions and 32 LDS reads), by the weights' bytes at 32. 1021 rows of 5376 -> 21504 (RG 4) 238 us, 0.99
// PFLOP/s, MFMAs busy 55 % of the time (672 tiles over 512 slots are half of what is missing); 512 experts of 2560 -> 640
// with 20 rows each (RG 1) gate and up 239 us, 3.7 TB/s of weights, down 138 us, 3.2 beside 0.8 of outputs.
//
// x goes through one of two LDS buffers, staged through registers while the step before is multiplied. Weights are read
// straight into the lanes that convert them, each by one wave of the workgroup only; every word of a block, converted with
// the block's scale, is one fragment.
//   RG 1, 2: 16 x 16 x 32 MFMAs, four tiles per wave. Lane l holds weight row l & 15 of each and block l >> 4 of the step, so a
//     load takes 64 neighbouring bytes of 16 rows: whole sectors, each asked for once (with 32 x 32 tiles 32 bytes of 32
//     rows, and the rest of the sector has left the L1 when its turn comes: 1.2 times the time for 20 rows per expert).
//     Weights and x are on their way for a whole step.
//   RG 4: 32 x 32 x 16 MFMAs, two tiles per wave, half the fragments in registers (the 16 x 16 form spills). Lane l holds row
//     l & 31 and blocks 2 (l >> 5) and 2 (l >> 5) + 1; weights and x are on their way for half a step.
// Scales: a step needs four bytes of a row, a cache line holds those of 32 steps, and the lines of all the rows under way do
// not stay in the L2; so a wave takes the words of 16 steps (RG 4: 8, for want of LDS) of each of its 64 rows at a time
// into LDS of its own.
#pragma once

#include <type_traits>

#include "exl3_mx4.h"

namespace exl3 {

template <int XT>
__device__ __forceinline__ f16_t mfma32(u32x4_t a, u32x4_t b, f16_t c) {
    if constexpr (XT == kRowF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

// MID: x rows are fp16 intermediates with an exponent per step of 128 (mid_exponent); staging brings a row's steps to the largest
// of them (er), by which the caller scales the sums.
template <int XT, int RG, bool MID = false>
struct Mx4Wide {
    static constexpr int kBuf = 32 * RG * 16;                      // units of 16 bytes of an x buffer
    static constexpr int kScaleSteps = RG == 4 ? 8 : 16;
    static constexpr int kScaleRow = kScaleSteps + 1;              // words per row (odd: 32 rows at one word touch every bank once)
    static constexpr int kScales = 4 * 64 * kScaleRow / 4;         // units of the four waves' scales
    static constexpr int kLds = 2 * kBuf + kScales;
    static constexpr int kTiles = RG == 4 ? 2 : 4, kRowTiles = RG == 4 ? RG : 2 * RG;
    typedef std::conditional_t<RG == 4, f16_t, f4_t> Tile;
    typedef Tile Acc[kRowTiles][kTiles];
    const uint8_t* xp[RG];             // this thread's staged rows (t >> 3) + 32 i
    __amdgpu_buffer_rsrc_t wr;         // codes of the wave's 64 weight rows, 0 past the matrix
    const uint8_t* wsc;                // scales of weight row l of the wave's 64
    int64_t sleft;                     // bytes from there to the end of the matrix's scales
    int base;
    int kb;
    u32x4_t* lds;                      // two x buffers, the waves' scales
    const int8_t* xe;                  // MID: exponents of the block's rows
    int ev[RG];                        // those of the staged rows' step on its way
    int* er;                           // LDS: a row's largest [32 RG], where its exponents begin [32 RG]

    // The staged rows' largest exponents: the eight lanes that stage a row share its steps.
    __device__ __forceinline__ void row_exponents(int t) const {
        const int n = (kb + 3) / 4;
#pragma unroll
        for (int i = 0; i < RG; ++i) {
            const int8_t* p = xe + (unsigned)er[32 * RG + (t >> 3) + 32 * i];
            int top = -126;
            for (int c = t & 7; c < n; c += 8) {
                const int e = ldg(p + c);
                top = top > e ? top : e;
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                const int e = __shfl_xor(top, o);
                top = top > e ? top : e;
            }
            er[(t >> 3) + 32 * i] = top;                       // (the wave's own rows: no barrier)
        }
    }

    // The wave's weight rows n0 .. n0 + 63 of `rows` (n0 below it or not), 32 kb wide.
    __device__ __forceinline__ void weights(const uint8_t* codes, const uint8_t* scales, int64_t n0, int64_t rows, int lane) {
        const int64_t left = rows - n0 < 64 ? (rows > n0 ? rows - n0 : 0) : 64, n = n0 + lane < rows ? n0 + lane : rows - 1;
        wr = mx4_rsrc(codes + (left > 0 ? n0 * kb * 16 : 0), left * kb * 16);
        wsc = scales + n * kb;
        sleft = (rows - n) * kb;
    }
    __device__ __forceinline__ static void zero(Acc& acc) {
#pragma unroll
        for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
            for (int i = 0; i < kTiles; ++i) acc[j][i] = Tile{};
    }
    // fn(row of the 32, weight row of the wave's 64, its four neighbouring outputs' values) over the row group j of acc
    template <typename F>
    __device__ __forceinline__ static void each(const Acc& acc, int j, int lane, F fn) {
        if constexpr (RG == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    fn(lane & 31, 32 * i + 8 * q + 4 * (lane >> 5),
                       f4_t{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]});
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) fn(16 * q + (lane & 15), 16 * i + 4 * (lane >> 4), acc[2 * j + q][i]);
        }
    }

    // RG 4: fn(row of the 32, first of sixteen weight rows, this lane's four at 4 (lane >> 5) of them, those at 8 + 4 (lane >> 5))
    template <typename F>
    __device__ __forceinline__ static void each16(const Acc& acc, int j, int lane, F fn) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; q += 2)
                fn(lane & 31, 32 * i + 8 * q,
                   f4_t{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]},
                   f4_t{acc[j][i][4 * q + 4], acc[j][i][4 * q + 5], acc[j][i][4 * q + 6], acc[j][i][4 * q + 7]});
    }

    // unit u (eight k) of row r of a buffer; the row number permutes its sixteen units, so that eight lanes reading eight
    // rows or writing half of one touch every bank once (with RG 1 the counters show conflicts for a third of the LDS cycles)
    __device__ __forceinline__ static int unit(int r, int u) { return r * 16 + (u ^ (r & 15)); }

    // blocks 2 h and 2 h + 1 of step c
    __device__ __forceinline__ void load_x(int c, int h, int t, u32x4_t (&st)[RG]) {
        if constexpr (MID) {
            if (h == 0)
#pragma unroll
                for (int i = 0; i < RG; ++i) ev[i] = ldg(xe + (unsigned)er[32 * RG + (t >> 3) + 32 * i] + c);
        }
        const int b = 4 * c + 2 * h + ((t & 7) >> 2), bc = b < kb ? b : kb - 1;
#pragma unroll
        for (int i = 0; i < RG; ++i) st[i] = ldg(reinterpret_cast<const u32x4_t*>(xp[i] + (int64_t)bc * 64) + (t & 3));
    }
    __device__ __forceinline__ void store_x(int c, int h, int t, u32x4_t (&st)[RG]) const {
        if constexpr (MID) {
#pragma unroll
            for (int i = 0; i < RG; ++i) {
                const int d = ev[i] - er[(t >> 3) + 32 * i];
                if (__ballot(d != 0)) st[i] = half_shift(st[i], d);   // uniform
            }
        }
        if (4 * c + 4 > kb) {                                  // uniform: blocks past the row are 0
            const uint32_t keep = 4 * c + 2 * h + ((t & 7) >> 2) < kb ? ~0u : 0u;
#pragma unroll
            for (int i = 0; i < RG; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) st[i][q] &= keep;
        }
        u32x4_t* o = lds + (c & 1) * kBuf;
#pragma unroll
        for (int i = 0; i < RG; ++i) o[unit((t >> 3) + 32 * i, 8 * h + (t & 7))] = st[i];
    }
    // this lane's block of step c of the tiles (RG 4: block j of its two); past the row's end the next row's, beside x that is 0
    __device__ __forceinline__ void load_w(int c, int j, uint32_t off, u32x4_t (&w)[kTiles]) const {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) w[i] = mx4_buffer16(wr, off + ((64 / kTiles) * i * kb * 16 + 64 * c + 16 * j));
    }
    __device__ __forceinline__ uint32_t* scale_words(int t) const {
        return reinterpret_cast<uint32_t*>(lds + 2 * kBuf) + (t >> 6) * (64 * kScaleRow);
    }
    // the wave's scales of kScaleSteps steps from c: bytes past the row's end (the next row's) become 0
    __device__ __forceinline__ void fetch_scales(int c, int t) const {
        uint32_t* o = scale_words(t) + (t & 63) * kScaleRow;
#pragma unroll 1
        for (int q = 0; q < kScaleSteps; q += 4) {
            const u32x4_t v = mx4_scales16(wsc, 4 * (c + q), sleft);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int left = kb - 4 * (c + q + e);
                o[q + e] = v[e] & (left >= 4 ? ~0u : left > 0 ? (1u << (8 * left)) - 1 : 0u);
            }
        }
    }
    // the scales of block b (of a step's four) of this lane's weight rows, from the step's words
    __device__ __forceinline__ void tile_scales(const uint32_t* sw, int b, float (&sc)[kTiles]) const {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) sc[i] = mx4_scale(sw[64 / kTiles * i * kScaleRow] >> (8 * b) & 255, base);
    }
    // products of words v0 .. v1 - 1 of the lane's block b of step c: acc += W rows x rows of x
    __device__ __forceinline__ void part(int c, int b, int v0, int v1, int r, const u32x4_t (&w)[kTiles], const float (&sc)[kTiles],
                                         Acc& acc) const {
        const u32x4_t* x = lds + (c & 1) * kBuf;
#pragma unroll
        for (int v = v0; v < v1; ++v) {
            u32x4_t f[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) f[i] = mx4_frag<XT>(w[i][v], sc[i]);
#pragma unroll
            for (int j = 0; j < kRowTiles; ++j) {
                const u32x4_t xv = x[unit(r + 32 * RG / kRowTiles * j, 4 * b + v)];
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    if constexpr (RG == 4) acc[j][i] = mfma32<XT>(f[i], xv, acc[j][i]);
                    else acc[j][i] = mfma16<XT>(f[i], xv, acc[j][i]);
                }
            }
        }
    }
    // acc += the products of steps c0 .. c0 + steps - 1 (those there are)
    __device__ __forceinline__ void run(int t, int c0, int steps, Acc& acc) {
        const int lane = t & 63, r = RG == 4 ? lane & 31 : lane & 15, g = RG == 4 ? lane >> 5 : lane >> 4;
        const int end = (kb + 3) / 4 - c0 < steps ? (kb + 3) / 4 : c0 + steps;
        const uint32_t off = (uint32_t)r * (uint32_t)(kb * 16) + (RG == 4 ? 32 : 16) * g;
        u32x4_t st[RG], su[RG], w[kTiles], n[kTiles];
        load_x(c0, 0, t, st);
        load_x(c0, 1, t, su);
        load_w(c0, 0, off, w);
        if constexpr (MID) row_exponents(t);
        store_x(c0, 0, t, st);
        store_x(c0, 1, t, su);
        __syncthreads();
        for (int c = c0; c < end; ++c) {
            const int cn = c + 1 < end ? c + 1 : c;            // (past the last: read again, stored into the idle buffer)
            const uint32_t* sw = scale_words(t) + r * kScaleRow + (c - c0) % kScaleSteps;
            float sc[kTiles];
            if ((c - c0) % kScaleSteps == 0) fetch_scales(c, t);
            load_x(cn, 0, t, st);
            if constexpr (RG == 4) {
                load_w(c, 1, off, n);
                tile_scales(sw, 2 * g, sc);
                __builtin_amdgcn_sched_barrier(0);
                part(c, 2 * g, 0, 4, r, w, sc, acc);
                __builtin_amdgcn_sched_barrier(0);
                store_x(c + 1, 0, t, st);
                load_x(cn, 1, t, st);
                load_w(cn, 0, off, w);
                tile_scales(sw, 2 * g + 1, sc);
                __builtin_amdgcn_sched_barrier(0);
                part(c, 2 * g + 1, 0, 4, r, n, sc, acc);
                __builtin_amdgcn_sched_barrier(0);
                store_x(c + 1, 1, t, st);
            } else {
                load_x(cn, 1, t, su);
                load_w(cn, 0, off, n);
                tile_scales(sw, g, sc);
                __builtin_amdgcn_sched_barrier(0);
                part(c, g, 0, 4, r, w, sc, acc);
                __builtin_amdgcn_sched_barrier(0);
                store_x(c + 1, 0, t, st);
                store_x(c + 1, 1, t, su);
#pragma unroll
                for (int i = 0; i < kTiles; ++i) w[i] = n[i];
            }
            __syncthreads();
        }
    }
};

// Waves per SIMD that the kernels with 32 RG rows are compiled for.
constexpr int mx4_wide_occ(int RG) { return RG == 4 ? 2 : RG == 2 ? 3 : 4; }

}  // namespace exl3
