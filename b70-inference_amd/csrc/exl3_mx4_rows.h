// Products of a few rows with MX4 weights: D[n][m] tiles of 16 x 16 on MFMAs with the weights as the first operand, k
// split over the waves of a workgroup, every operand read from memory straight into the lanes that multiply it.
// A decode call is bound by the weights' bytes: each weight is read once, by one wave, with no barrier before the end;
// the rows come from the L2. One 16 x 16 x 32 MFMA takes a wave as long as the four v_dot2 that it replaces at one row, and
// serves up to 16 rows for it.
#pragma once

#include "exl3_mx4.h"

namespace exl3 {

// Accumulates the chunks c0, c0 + cstep, ... < nch of 128 k (4 blocks of 32; block 4 c + (lane >> 4) is this lane's).
// wq / wsc: this lane's weight row (lane & 15) of each n tile, its codes and scales; xq / xsc: this lane's x row of each m
// tile. kb: blocks in a row. U chunks are loaded before the first is used. Blocks past the row are read at its last
// block and zeroed in both operands.
template <int XT, int NT, int MT, int U>
__device__ __forceinline__ void mx4_rows_loop(const uint8_t* const (&wq)[NT], const uint8_t* const (&wsc)[NT],
                                              const int (&base)[NT], const uint8_t* const (&xq)[MT],
                                              const uint8_t* const (&xsc)[MT], int kb, int c0, int cstep, int nch, int g,
                                              f4_t (&acc)[NT][MT]) {
    constexpr int XV = XT == kRowMX4 ? 1 : 4;
    for (int c = c0; c < nch; c += U * cstep) {
        u32x4_t w[U][NT], x[U][MT][XV];
        int ws[U][NT], xs[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = 4 * (c + u * cstep) + g, bc = b < kb ? b : kb - 1;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                w[u][i] = ldg(reinterpret_cast<const u32x4_t*>(wq[i] + (int64_t)bc * 16));
                ws[u][i] = ldg(wsc[i] + bc);
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
#pragma unroll
                for (int v = 0; v < XV; ++v)
                    x[u][j][v] = ldg(reinterpret_cast<const u32x4_t*>(xq[j] + (int64_t)bc * (16 * XV)) + v);
                if constexpr (XT == kRowMX4) xs[u][j] = ldg(xsc[j] + bc);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int cc = c + u * cstep;
            if (cc >= nch) break;                              // uniform
            if (4 * cc + 4 > kb) {                             // uniform: a row's last chunk, partly past it
                const uint32_t keep = 4 * cc + g < kb ? ~0u : 0u;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) w[u][i][q] &= keep;
#pragma unroll
                for (int j = 0; j < MT; ++j)
#pragma unroll
                    for (int v = 0; v < XV; ++v)
#pragma unroll
                        for (int q = 0; q < 4; ++q) x[u][j][v][q] &= keep;
            }
            if constexpr (XT == kRowMX4) {
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < MT; ++j)
                        acc[i][j] = mfma16_mx4(w[u][i], ws[u][i], x[u][j][0], xs[u][j], acc[i][j]);
            } else {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const float s = mx4_scale(ws[u][i], base[i]);
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const u32x4_t f = mx4_frag<XT>(w[u][i][v], s);
#pragma unroll
                        for (int j = 0; j < MT; ++j) acc[i][j] = mfma16<XT>(f, x[u][j][v], acc[i][j]);
                    }
                }
            }
        }
    }
}

// Sum of the waves' tiles in wave order, through LDS (`red`: waves x NT x MT x 64 f4_t). The caller reads tile (i, j) of
// lane l with mx4_rows_sum after this.
template <int NT, int MT>
__device__ __forceinline__ void mx4_rows_put(f4_t* red, int wave, int lane, const f4_t (&acc)[NT][MT]) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) red[((wave * NT + i) * MT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
}
template <int NT, int MT>
__device__ __forceinline__ f4_t mx4_rows_sum(const f4_t* red, int waves, int i, int j, int l) {
    f4_t s = red[(i * MT + j) * 64 + l];
    for (int w = 1; w < waves; ++w) {
        const f4_t t = red[((w * NT + i) * MT + j) * 64 + l];
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += t[q];
    }
    return s;
}

// Waves of a workgroup over nch chunks of 128 k.
inline int mx4_rows_waves(int nch) { return nch < 8 ? (nch < 1 ? 1 : nch) : 8; }

}  // namespace exl3
