// Products of many 16-bit rows with MX4 weights on 32 x 32 x 16 MFMAs: a workgroup of four waves takes 32 RG rows of x and
// 64 weight rows (outputs) per wave. Bound by the MFMAs from about 64 rows (RG 4: 64 MFMAs of 32 cycles per wave and step
// against 64 conversions and 32 LDS reads), below by the conversions and the weights' bytes.
//
// Steps of 128 k (four blocks). Lane l holds weight row l & 31 and blocks 2 g and 2 g + 1, g = l >> 5, of the step: 32
// neighbouring bytes of codes, read straight from memory (each weight is read and converted by one wave of the workgroup
// only); every word of a block, converted with the block's scale, is one fragment. x goes through one of two LDS buffers,
// staged through registers in halves of 64 k: the first half of the next step's rows arrives during block 0 and is stored
// before block 1, the second during block 1. Weights likewise: block 1 of a step arrives during its block 0, block 0 of
// the next during block 1.
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

template <int XT, int RG>
struct Mx4Wide {
    static constexpr int kBuf = 32 * RG * 16, kLdsBytes = 2 * kBuf * 16;
    const uint8_t* xp[RG];             // this thread's staged rows (t >> 3) + 32 i
    const uint8_t *wq[2], *wsc[2];     // this lane's weight rows l & 31 of the wave's two tiles: codes, scales
    int base[2];
    int kb;
    u32x4_t* lds;                      // two buffers

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
    __device__ __forceinline__ void load_w(int c, int j, int g, u32x4_t (&w)[2], int (&s)[2]) const {
        const int b = 4 * c + 2 * g + j, bc = b < kb ? b : kb - 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[i] = ldg(reinterpret_cast<const u32x4_t*>(wq[i] + (int64_t)bc * 16));
            s[i] = ldg(wsc[i] + bc);
        }
    }
    // products of one block: acc += W rows (lane l & 31) x rows of x
    __device__ __forceinline__ void block(int c, int j, int r, int g, const u32x4_t (&w)[2], const int (&s)[2],
                                          f16_t (&acc)[RG][2]) const {
        const u32x4_t* x = lds + (c & 1) * kBuf;
        // a block past the row multiplies zeros: any scale but 255 does
        const bool in = 4 * c + 2 * g + j < kb;
        const float s0 = mx4_scale(in ? s[0] : 0, base[0]), s1 = mx4_scale(in ? s[1] : 0, base[1]);
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
        u32x4_t st[RG], w0[2], w1[2];
        int s0[2], s1[2];
        load_x(0, 0, t, st);
        load_w(0, 0, g, w0, s0);
        store_x(0, 0, t, st);
        load_x(0, 1, t, st);
        store_x(0, 1, t, st);
        __syncthreads();
        for (int c = 0; c < nch; ++c) {
            const int cn = c + 1 < nch ? c + 1 : c;            // (past the last: read again, stored into the idle buffer)
            load_w(c, 1, g, w1, s1);
            load_x(cn, 0, t, st);
            __builtin_amdgcn_sched_barrier(0);
            block(c, 0, r, g, w0, s0, acc);
            __builtin_amdgcn_sched_barrier(0);
            if (c + 1 < nch) store_x(cn, 0, t, st);
            load_w(cn, 0, g, w0, s0);
            load_x(cn, 1, t, st);
            __builtin_amdgcn_sched_barrier(0);
            block(c, 1, r, g, w1, s1, acc);
            __builtin_amdgcn_sched_barrier(0);
            if (c + 1 < nch) store_x(cn, 1, t, st);
            __syncthreads();
        }
    }
};

// Waves per SIMD that the kernels with 32 RG rows are compiled for.
constexpr int mx4_wide_occ(int RG) { return RG == 4 ? 2 : RG == 2 ? 3 : 4; }

}  // namespace exl3
