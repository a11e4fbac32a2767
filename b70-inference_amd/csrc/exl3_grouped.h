// Rows grouped by expert: rows ends[e - 1] .. ends[e] - 1 of a matrix (from 0 for e = 0) belong to expert e, rows behind the last end
// to none. The ends lie on the GPU, so the grid holds as many blocks of BM rows as T rows over E experts can need, and a workgroup
// finds the expert of its block in a running sum of the experts' blocks, 576 experts at a time.
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

// Where the K experts of a lane end, from `e0` on: v[i] .. v[i + 1] the rows of expert e0 + i; expert E has the rows of none, those
// behind it no rows. The loads are under way together.
template <int K>
__device__ __forceinline__ void group_ends(const int32_t* ends, int E, int T, int e0, int (&v)[K + 1]) {
#pragma unroll
    for (int i = 0; i <= K; ++i) {
        const int e = e0 + i - 1;
        v[i] = ldg(ends + (e < 0 ? 0 : e < E ? e : E - 1));
    }
#pragma unroll
    for (int i = 0; i <= K; ++i) {
        const int e = e0 + i - 1, c = v[i] < 0 ? 0 : v[i] > T ? T : v[i];
        v[i] = e < 0 ? 0 : e < E ? c : T;
    }
}
template <int BM>
__device__ __forceinline__ int group_blocks_of(int lo, int hi) {
    return hi > lo ? (hi - lo + BM - 1) / BM : 0;
}

// The same value in every lane (wave-uniform). Blocks behind the last one have no rows.
template <int BM, int K>
__device__ __forceinline__ GroupSlot group_slot_of(const int32_t* ends, int E, int T, unsigned slot) {
    const int lane = threadIdx.x & 63;
    unsigned first = 0;                // blocks of the experts before
    for (int i0 = 0; i0 <= E; i0 += 64 * K) {
        const int e0 = i0 + lane * K;
        int v[K + 1], upto[K], sum = 0;
        group_ends<K>(ends, E, T, e0, v);
#pragma unroll
        for (int i = 0; i < K; ++i) upto[i] = sum += group_blocks_of<BM>(v[i], v[i + 1]);
        const int run = wave_running_sum(sum);
        const uint64_t in = __ballot(first + (unsigned)run > slot);
        if (!in) {                     // uniform
            first += (unsigned)__builtin_amdgcn_readlane(run, 63);
            continue;
        }
        // every lane looks as if the block were its own, the one that has it is right
        const int l = __builtin_ctzll(in), at = (int)(slot - first) - (run - sum);
        int e = e0, row = 0, left = 0;
#pragma unroll
        for (int i = K - 1; i >= 0; --i)
            if (upto[i] > at) {
                e = e0 + i;
                row = v[i] + (at - (i ? upto[i - 1] : 0)) * BM;
                left = v[i + 1] - row;
            }
        GroupSlot s;
        s.e = __builtin_amdgcn_readlane(e, l);
        s.row = __builtin_amdgcn_readlane(row, l);
        left = __builtin_amdgcn_readlane(left, l);
        s.rows = left < BM ? left : BM;
        return s;
    }
    return GroupSlot{E, 0, 0};
}

// Nine experts to a lane, one of fewer than 64 (64 rows over 512 experts of 512 -> 512 7.1 us; with one expert to a lane, and the lanes' sums
// for each, 8.7. One row of one matrix of 4096 -> 4096 10.5; with nine 11.2).
constexpr int kLaneExperts = 9;
template <int BM>
__device__ __forceinline__ GroupSlot group_slot(const int32_t* ends, int E, int T, unsigned slot) {
    return E < 64 ? group_slot_of<BM, 1>(ends, E, T, slot) : group_slot_of<BM, kLaneExperts>(ends, E, T, slot);
}

// The blocks there are, with `rest` those of the rows of none (wave-uniform).
template <int BM>
__device__ __forceinline__ unsigned group_blocks(const int32_t* ends, int E, int T, bool rest) {
    unsigned n = 0;
    for (int i0 = 0; i0 <= E; i0 += 64 * kLaneExperts) {
        const int e0 = i0 + (int)(threadIdx.x & 63) * kLaneExperts;
        int v[kLaneExperts + 1], sum = 0;
        group_ends<kLaneExperts>(ends, E, T, e0, v);
#pragma unroll
        for (int i = 0; i < kLaneExperts; ++i) sum += rest || e0 + i < E ? group_blocks_of<BM>(v[i], v[i + 1]) : 0;
        n += (unsigned)__builtin_amdgcn_readlane(wave_running_sum(sum), 63);
    }
    return n;
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
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(r) : "m0", "memory");
}

}  // namespace exl3
