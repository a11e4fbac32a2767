// Host-side choices of the MX4 kernels: tiles, k-splits, row blocks and their number. Plain C++ without device code. They follow
// from the shape alone: a call gives the same bits eager and captured.
#pragma once

#include <stdint.h>

#include "exl3_moe.h"

namespace exl3 {

// How an expert's rows are cut: blocks of `rows`, the last one short (whole: a remainder is never cut smaller).
inline BlockCut mx4_cut(int rows) { return {rows, 0, 1}; }

// Blocks of a call of npairs rows over E experts, at most.
inline int64_t mx4_max_blocks(int64_t npairs, int64_t E, int rows) { return npairs / rows + (E < npairs ? E : npairs); }

// Rows of a block (32, 64 or 128) by the mean load: a block costs its whole rows' MFMAs, a second block of an expert its weights
// again. us at 32 / 64 / 128 rows: 20 rows per expert (512 of 2560 -> 640) 434 / 485 / 703; 32 (32 of 7168 -> 2048) 281 / 239 / 340;
// 64 (64 of 4096 -> 1408) 355 / 282 / 314, (32 of 7168 -> 2048) 399 / 328 / 354.
inline int mx4_moe_rows(int64_t npairs, int64_t E) { return npairs <= 26 * E ? 32 : npairs <= 96 * E ? 64 : 128; }

// Tile (index into the candidates) and k-splits of a dense product by estimated time.
struct Mx4Plan {
    int tile, P, bps;                  // splits, steps of 128 k in each
};

// A candidate: rows and columns of a tile, workgroups per CU; microseconds per step of a CU with 1 .. occ of them, per round, and
// per MB of partials.
struct Mx4Cand {
    int bm, bn, occ;
    float step[4], edge, mb;
};

// The workgroups spread over the CUs in rounds of occ each; several splits add their partials and the reduce kernel (`red`
// us). Fitted to measured points (4096 x 1024 .. 21504 x 5376, 8 .. 2048 rows, 1 .. 16 splits): 16-bit rows 578 points, the one
// picked within 2.3 % of the best on average, 18 % at worst; MX4 rows 350 points, 0.8 % and 11 %.
inline Mx4Plan mx4_plan(const Mx4Cand* cand, int ncand, float red, int64_t m, int64_t n, int64_t k, int cus) {
    const int nst = (int)((k + 127) / 128);
    Mx4Plan best = {0, 1, nst};
    float tb = 1e30f;
    for (int c = 0; c < ncand; ++c) {
        const int64_t tiles = (m + cand[c].bm - 1) / cand[c].bm * ((n + cand[c].bn - 1) / cand[c].bn);
        for (int p = 1; p <= 16 && p <= nst; ++p) {
            const int bps = (nst + p - 1) / p;
            if ((nst + bps - 1) / bps != p) continue;          // the same splits as with fewer
            const int64_t w = (tiles * p + cus - 1) / cus, full = w / cand[c].occ, rem = w % cand[c].occ;
            float t = (float)(full + (rem > 0)) * cand[c].edge +
                      (float)bps * ((float)full * cand[c].step[cand[c].occ - 1] + (rem ? cand[c].step[rem - 1] : 0.f));
            if (p > 1) t += red + cand[c].mb * (float)p * (float)m * (float)n * 4e-6f;
            if (t < tb) {
                tb = t;
                best = {c, p, bps};
            }
        }
    }
    return best;
}

// 16-bit rows: blocks of 32, 64, 128 rows x 256 outputs
inline Mx4Plan mx4_linear_plan(int64_t m, int64_t n, int64_t k, int cus) {
    static const Mx4Cand kCand[3] = {{32, 256, 4, {0.86f, 1.19f, 1.68f, 2.09f}, 3.9f, 0.37f},
                                     {64, 256, 3, {1.10f, 1.66f, 2.47f, 0.f}, 6.3f, 0.21f},
                                     {128, 256, 2, {1.71f, 3.14f, 0.f, 0.f}, 6.4f, 0.24f}};
    return mx4_plan(kCand, 3, 5.9f, m, n, k, cus);
}

// MX4 rows: tiles of 64 x 128, 128 x 128, 256 x 256
inline Mx4Plan mx4_gemm_plan(int64_t m, int64_t n, int64_t k, int cus) {
    static const Mx4Cand kCand[3] = {{64, 128, 4, {0.39f, 0.56f, 0.75f, 0.76f}, 5.7f, 0.36f},
                                     {128, 128, 3, {0.47f, 0.70f, 1.09f, 0.f}, 6.0f, 0.29f},
                                     {256, 256, 1, {1.00f, 0.f, 0.f, 0.f}, 11.7f, 0.25f}};
    return mx4_plan(kCand, 3, 2.8f, m, n, k, cus);
}

}  // namespace exl3
