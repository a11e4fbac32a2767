// Products of many 16-bit rows with MX4 weights on 32 x 32 x 16 MFMAs: a workgroup of four waves takes 32 RG rows of x and
// 64 weight rows (outputs) per wave. Bound by the MFMAs from about 64 rows (RG 4: 64 MFMAs of 32 cycles per wave and step
// against 64 conversions and 32 LDS reads), below by the conversions and the weights' bytes.
//
// Steps of 128 k (four blocks). Lane l holds weight row l & 31 and blocks 2 g and 2 g + 1, g = l >> 5, of the step: 32
// neighbouring bytes of codes, read straight from memory (each weight is read and converted by one wave of the workgroup
// only); every word of a block, converted with the block's scale, is one fragment. x goes through one of two LDS buffers,
// staged through registers while the step before is multiplied (RG 4: in halves of 64 k, for want of registers); a block
// of weights is on its way for a whole step before its products.
#pragma once

#include "exl3_mx4.h"

namespace exl3 {

template <int XT>
__device__ __forceinline__ f16_t mfma32(u32x4_t a, u32x4_t b, f16_t c) {
    if constexpr (XT == kRowF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

// Scales: a step needs four bytes of a row, a cache line holds those of 32 steps, and the lines of all the rows under way do
// not stay in the L2; so a wave takes the words of 16 steps (RG 4: 8, for want of LDS) of each of its 64 rows at a time
// into LDS of its own.

template <int XT, int RG>
struct Mx4Wide {
    static constexpr int kBuf = 32 * RG * 16;                      // units of 16 bytes of an x buffer
    static constexpr int kScaleSteps = RG == 4 ? 8 : 16;
    static constexpr int kScaleRow = kScaleSteps + 1;              // words per row (odd: 32 rows at one word touch every bank once)
    static constexpr int kScales = 4 * 64 * kScaleRow / 4;         // units of the four waves' scales
    static constexpr int kLds = 2 * kBuf + kScales;
    const uint8_t* xp[RG];             // this thread's staged rows (t >> 3) + 32 i
    const uint8_t* wq[2];              // codes of this lane's weight rows, l & 31 of the wave's two tiles
    const uint8_t* wsc;                // scales of weight row l of the wave's 64
    int64_t sleft;                     // bytes from there to the end of the matrix's scales
    int base[2];
    int kb;
    u32x4_t* lds;                      // two x buffers, the waves' scales

    // unit u (eight k) of row r of a buffer; the row number permutes its sixteen units, so that eight lanes reading eight
    // rows or writing half of one touch every bank once
    __device__ __forceinline__ static int unit(int r, int u) { return r * 16 + (u ^ (r & 15)); }

    __device__ __forceinline__ void load_x(int c, int h, int t, u32x4_t (&st)[RG]) const {
        const int b = 4 * c + 2 * h + ((t & 7) >> 2), bc = b < kb ? b : kb - 1;
#pragma unroll
        for (int i = 0; i < RG; ++i) st[i] = ldg(reinterpret_cast<const u32x4_t*>(xp[i] + (int64_t)bc * 64) + (t & 3));
    }
    __device__ __forceinline__ void store_x(int c, int h, int t, u32x4_t (&st)[RG]) const {
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
    __device__ __forceinline__ void load_w(int c, int j, int g, u32x4_t (&w)[2]) const {
        const int b = 4 * c + 2 * g + j, bc = b < kb ? b : kb - 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = ldg(reinterpret_cast<const u32x4_t*>(wq[i] + (int64_t)bc * 16));
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
    // products of one block: acc += W rows (lane l & 31) x rows of x
    __device__ __forceinline__ void block(int c, int j, int r, int g, const u32x4_t (&w)[2], const uint32_t (&s)[2],
                                          f16_t (&acc)[RG][2]) const {
        const u32x4_t* x = lds + (c & 1) * kBuf;
        const float s0 = mx4_scale(s[0] >> (16 * g + 8 * j) & 255, base[0]), s1 = mx4_scale(s[1] >> (16 * g + 8 * j) & 255, base[1]);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const u32x4_t f0 = mx4_frag<XT>(w[0][v], s0), f1 = mx4_frag<XT>(w[1][v], s1);
#pragma unroll
            for (int i = 0; i < RG; ++i) {
                const u32x4_t xv = x[unit(r + 32 * i, 4 * (2 * g + j) + v)];
                acc[i][0] = mfma32<XT>(f0, xv, acc[i][0]);
                acc[i][1] = mfma32<XT>(f1, xv, acc[i][1]);
            }
        }
    }
    __device__ __forceinline__ void run(int t, f16_t (&acc)[RG][2]) const {
        const int lane = t & 63, r = lane & 31, g = lane >> 5, nch = (kb + 3) / 4;
        u32x4_t st[RG], su[RG], w0[2], w1[2], n0[2], n1[2];
        load_x(0, 0, t, st);
        load_x(0, 1, t, su);
        load_w(0, 0, g, w0);
        load_w(0, 1, g, w1);
        store_x(0, 0, t, st);
        store_x(0, 1, t, su);
        __syncthreads();
        for (int c = 0; c < nch; ++c) {
            const int cn = c + 1 < nch ? c + 1 : c;            // (past the last: read again, stored into the idle buffer)
            if (c % kScaleSteps == 0) fetch_scales(c, t);
            load_x(cn, 0, t, st);
            if constexpr (RG < 4) {
                load_x(cn, 1, t, su);
                load_w(cn, 0, g, n0);
                load_w(cn, 1, g, n1);
            } else if (c > 0) {
                load_w(c, 1, g, w1);
            }
            const uint32_t* sw = scale_words(t) + r * kScaleRow + c % kScaleSteps;
            const uint32_t s[2] = {sw[0], sw[32 * kScaleRow]};
            __builtin_amdgcn_sched_barrier(0);
            block(c, 0, r, g, w0, s, acc);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (RG == 4) {
                store_x(c + 1, 0, t, st);
                load_x(cn, 1, t, st);
                load_w(cn, 0, g, w0);
                __builtin_amdgcn_sched_barrier(0);
            }
            block(c, 1, r, g, w1, s, acc);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (RG < 4) {
                store_x(c + 1, 0, t, st);
                store_x(c + 1, 1, t, su);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    w0[i] = n0[i];
                    w1[i] = n1[i];
                }
            } else {
                store_x(c + 1, 1, t, st);
            }
            __syncthreads();
        }
    }
};

// Waves per SIMD that the kernels with 32 RG rows are compiled for.
constexpr int mx4_wide_occ(int RG) { return RG == 4 ? 2 : RG == 2 ? 3 : 4; }

}  // namespace exl3
