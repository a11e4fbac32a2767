// Rows grouped by expert: rows ends[e - 1] .. ends[e] - 1 of a matrix (from 0 for e = 0) belong to expert e, rows behind the last end
// to none. The ends lie on the GPU; the grid follows from the sizes alone: expert e's blocks of BM rows take the slots from
// floor(ends[e - 1] / BM) + e on, which are enough for them (ceil((b - a) / BM) <= floor(b / BM) - floor(a / BM) + 1) and
// disjoint, so a workgroup finds its expert by counting the experts whose first slot is not behind its own, one load per 64 of them.
#pragma once

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

// Slots of T rows over E experts, and with `rest` of the rows of none: of blocks of BM rows, or where that is fewer one for every
// row, of which a block's first does the block's work (few rows over many experts: an empty slot costs a workgroup's launch).
inline int64_t group_slots(int64_t T, int64_t E, int64_t BM, bool rest) {
    const int64_t n = T / BM + E + (rest ? 1 : 0);
    return T < n ? T : n;
}

// The same value in every lane (wave-uniform). `slots`: group_slots.
template <int BM>
__device__ __forceinline__ GroupSlot group_slot(const int32_t* ends, int E, int T, unsigned slot, int slots) {
    const int lane = threadIdx.x & 63;
    const bool by_row = slots == T;    // (every block's first row is a slot's then too if T = T / BM + E)
    int e = 0;
    for (int i = 0; i < E; i += 64) {
        const int at = i + lane, end = group_end(ends, at < E ? at : E - 1, T);
        const bool in = at < E && (by_row ? (unsigned)end : (unsigned)(end / BM + at + 1)) <= slot;
        e += __popcll(__ballot(in));
    }
    e = __builtin_amdgcn_readfirstlane(e);
    const int lo = __builtin_amdgcn_readfirstlane(e > 0 ? group_end(ends, e - 1, T) : 0);
    const int hi = __builtin_amdgcn_readfirstlane(e < E ? group_end(ends, e, T) : T);
    GroupSlot s;
    s.e = e;
    if (by_row) {
        s.row = slot;
        s.rows = (int)slot < lo || (int)slot >= hi || ((int)slot - lo) % BM != 0 ? 0 : hi - (int)slot < BM ? hi - (int)slot : BM;
        return s;
    }
    const int64_t block = (int64_t)slot - (lo / BM + e);
    s.row = lo + block * BM;
    s.rows = block < 0 || s.row >= hi ? 0 : hi - s.row < BM ? (int)(hi - s.row) : BM;
    return s;
}

}  // namespace exl3
