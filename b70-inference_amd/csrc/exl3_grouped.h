// Rows grouped by expert: rows ends[e - 1] .. ends[e] - 1 of a matrix (from 0 for e = 0) belong to expert e, rows behind the last end
// to none. The ends lie on the GPU, so the grid holds as many blocks of BM rows as T rows over E experts can need, and a workgroup
// finds the expert of its block in a running sum of the experts' blocks, 64 experts at a time.
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

// Most blocks of BM rows that T rows over E experts have, with `rest` the rows of none among them.
inline int64_t group_slots(int64_t T, int64_t E, int64_t BM, bool rest) {
    const int64_t n = T / BM + E + (rest ? 1 : 0);
    return T < n ? T : n;
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ int wave_running_sum(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        v += lane >= o ? u : 0;
    }
    return v;
}

// The same value in every lane (wave-uniform). Blocks behind the last one have no rows.
template <int BM>
__device__ __forceinline__ GroupSlot group_slot(const int32_t* ends, int E, int T, unsigned slot) {
    const int lane = threadIdx.x & 63;
    GroupSlot s;
    unsigned first = 0;                // blocks of the experts before
    for (int i = 0; i <= E; i += 64) {
        const int e = i + lane;
        const int lo = e > 0 ? group_end(ends, e <= E ? e - 1 : E - 1, T) : 0, hi = e < E ? group_end(ends, e, T) : e == E ? T : lo;
        const int blocks = hi > lo ? (hi - lo + BM - 1) / BM : 0, sum = wave_running_sum(blocks);
        const uint64_t in = __ballot(first + (unsigned)sum > slot);
        if (in) {                      // uniform
            const int l = __builtin_ctzll(in);
            s.e = i + l;
            const int block = (int)(slot - first) - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(blocks, l));
            const int row = __builtin_amdgcn_readlane(lo, l) + block * BM, left = __builtin_amdgcn_readlane(hi, l) - row;
            s.row = row;
            s.rows = left < BM ? left : BM;
            return s;
        }
        first += (unsigned)__builtin_amdgcn_readlane(sum, 63);
    }
    s.e = E;
    s.row = 0;
    s.rows = 0;
    return s;
}

// The blocks there are, with `rest` those of the rows of none (wave-uniform).
template <int BM>
__device__ __forceinline__ unsigned group_blocks(const int32_t* ends, int E, int T, bool rest) {
    int n = 0;
    for (int i = 0; i < E + (rest ? 1 : 0); i += 64) {
        const int e = i + (threadIdx.x & 63);
        const int lo = e > 0 ? group_end(ends, e <= E ? e - 1 : E - 1, T) : 0, hi = e < E ? group_end(ends, e, T) : e == E && rest ? T : lo;
        n += __builtin_amdgcn_readlane(wave_running_sum(hi > lo ? (hi - lo + BM - 1) / BM : 0), 63);
    }
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
