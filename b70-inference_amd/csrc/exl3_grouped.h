// Rows grouped by expert: rows ends[e - 1] .. ends[e] - 1 of a matrix (from 0 for e = 0) belong to expert e, rows behind the last end
// to none. The ends lie on the GPU, so the grid holds as many blocks of BM rows as T rows over E experts can need, and a workgroup
// finds the expert of its block in a running sum of the experts' blocks, 64 experts at a time.
#pragma once

#include <cmath>

#include "exl3_mx4.h"

namespace exl3 {

struct GroupSlot {
    int e;                             // expert; E: the rows of none
    int64_t row;                       // first row of the block
    int rows;                          // of the block; 0: nothing to do
};

// Ends outside [0, T] count as 0 and T, an expert that ends before it begins has no rows: no value of `ends` leads out of range.
__device__ __forceinline__ int group_end(const int32_t* ends, int e, int T) {
    const int v = ldg(ends + e);
    return v < 0 ? 0 : v > T ? T : v;
}

// Most blocks of BM rows that T rows over E experts have, with `rest` the rows of none among them.
inline int64_t group_slots(int64_t T, int64_t E, int64_t BM, bool rest) {
    const int64_t n = T / BM + E + (rest ? 1 : 0);
    return T < n ? T : n;
}

// Experts that have rows, if all are as likely.
inline double group_live(int64_t T, int64_t E) { return E == 1 ? 1.0 : (double)E * (1.0 - std::pow(1.0 - 1.0 / (double)E, (double)T)); }

// Workgroups to a block of rows for kernels of few rows, whose workgroups go round the block's tiles: as many as fill the CUs by the
// estimate that is least for the CU with most tiles. `us`: what a tile's weights take a CU without a pause, which takes `need` waves (16-bit
// weights six; 4-bit ones, which are converted, eight); a workgroup that waits for another's end starts late. As many as need no more
// rounds, without regard to the tiles of a CU, were slower: ten rows of 512 experts of 2048 -> 1024, 16-bit weights, 14.2 against 11.8 us;
// 4-bit, 16 rows of 4096 -> 6144 15.5 and 11.1.
inline int64_t group_split(int64_t T, int64_t E, int64_t tiles, int64_t waves, int64_t fit, int64_t need, double us) {
    const int64_t slots = E == 1 ? (T + 15) / 16 : T / 16 + (int64_t)std::ceil(group_live(T, E));   // blocks of 16 rows
    int64_t best = 1;
    double least = 1e30;
    const int64_t mean = slots * tiles / 256 + 1;
    for (int64_t q = 1; q <= (tiles < 32 ? tiles : 32); ++q) {
        const int64_t n = (slots * ((tiles + q - 1) / q) + 255) / 256, rounds = (n + fit - 1) / fit, busy = (n < fit ? n : fit) * waves;
        const double t = (double)(n * q) * us * (busy < need ? (double)need / (double)busy : 1.0) + 4.0 * (double)(rounds - 1);
        if (t > least) continue;
        least = t;
        best = n * 256 / slots;
    }
    // (as few as fill the CUs where a workgroup has more tiles than that)
    if (mean > 16 * fit) best = 256 * fit / slots;
    return best < 1 ? 1 : best < tiles ? best : tiles;
}

// Sum over the lanes up to and with this one: shifts by 1, 2, 4, 8 inside the 16 lanes of a row, then the rows' sums on.
__device__ __forceinline__ int wave_running_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast:31 into rows 2, 3
    return v;
}

// fn(first expert of 64, this lane's begin and end) for the experts and the rows of none as the last of all, until it returns true.
// Nine loads of either kind are under way: one after another they are a microsecond for every 64 experts and more.
template <typename F>
__device__ __forceinline__ void group_each(const int32_t* ends, int E, int T, F fn) {
    constexpr int kBatch = 9;
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 <= E; i0 += 64 * kBatch) {
        int lo[kBatch], hi[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (i0 + 64 * i > E) break;                        // uniform
            const int e = i0 + 64 * i + lane;
            lo[i] = ldg(ends + (e < 1 ? 0 : e <= E ? e - 1 : E - 1));
            hi[i] = ldg(ends + (e < E ? e : E - 1));
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (i0 + 64 * i > E) break;
            const int e = i0 + 64 * i + lane;
            const int l = e < 1 ? 0 : lo[i] < 0 ? 0 : lo[i] > T ? T : lo[i], h = e < E ? hi[i] < 0 ? 0 : hi[i] > T ? T : hi[i] : e == E ? T : l;
            if (fn(i0 + 64 * i, l, h)) return;
        }
    }
}

// The same value in every lane (wave-uniform). Blocks behind the last one have no rows.
template <int BM>
__device__ __forceinline__ GroupSlot group_slot(const int32_t* ends, int E, int T, unsigned slot) {
    GroupSlot s = {E, 0, 0};
    unsigned first = 0;                // blocks of the experts before
    group_each(ends, E, T, [&](int i, int lo, int hi) {
        const int blocks = hi > lo ? (hi - lo + BM - 1) / BM : 0, sum = wave_running_sum(blocks);
        const uint64_t in = __ballot(first + (unsigned)sum > slot);
        first += (unsigned)__builtin_amdgcn_readlane(sum, 63);
        if (!in) return false;         // uniform
        const int l = __builtin_ctzll(in), before = (int)first - __builtin_amdgcn_readlane(sum, 63);
        const int block = (int)slot - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(blocks, l));
        const int row = __builtin_amdgcn_readlane(lo, l) + block * BM, left = __builtin_amdgcn_readlane(hi, l) - row;
        s.e = i + l;
        s.row = row;
        s.rows = left < BM ? left : BM;
        return true;
    });
    return s;
}

// The blocks there are, with `rest` those of the rows of none (wave-uniform).
template <int BM>
__device__ __forceinline__ unsigned group_blocks(const int32_t* ends, int E, int T, bool rest) {
    int n = 0;
    group_each(ends, E, T, [&](int i, int lo, int hi) {
        const bool in = hi > lo && (rest || i + (int)(threadIdx.x & 63) < E);
        n += __builtin_amdgcn_readlane(wave_running_sum(in ? (hi - lo + BM - 1) / BM : 0), 63);
        return false;
    });
    return (unsigned)n;
}

// A workgroup's place in a grid that takes `chunk` tiles after one another on an XCD, the XCDs in turn (workgroups go round robin over
// them): what runs together on one shares operands in its L2, and tiles of little work (experts of few rows) spread over all.
__device__ __forceinline__ unsigned grouped_place(unsigned chunk, unsigned block) {
    const unsigned j = block >> 3, c = j / chunk;
    return (c * 8 + (block & 7)) * chunk + j - c * chunk;
}
// Tile `in` of nmt x nnt: eight rows of tiles after one another for each column.
__device__ __forceinline__ void grouped_tile(unsigned in, unsigned nmt, unsigned nnt, unsigned& mt, unsigned& nt) {
    const unsigned band = in / (8 * nnt), i = in - band * 8 * nnt, h = nmt - 8 * band < 8 ? nmt - 8 * band : 8;
    nt = i / h;
    mt = 8 * band + i - nt * h;
}
constexpr unsigned kChunk = 32;        // the CUs of an XCD

// 16 bytes per lane from `at` bytes on to LDS (address `lds` and 16 bytes a lane from there on). Inline assembly: behind the builtin
// the compiler waits for the load before every transposing read, whatever it reads. What it brings is waited for by wait_step.
__device__ __forceinline__ void lds_load16(__amdgpu_buffer_rsrc_t r, uint32_t at, const void* lds) {
    const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(r));
}

}  // namespace exl3
