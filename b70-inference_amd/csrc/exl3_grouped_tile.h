// Products of 16-bit matrices grouped by expert: tiles of BM x BN outputs on 16 x 16 x 32 MFMAs, contraction in steps of 64.
//   out[m, n] = sum_c A(m, c) B(n, c)
// Either operand lies in memory with the contraction along its rows ("along": x and dy rows, weights of the forward product) or
// across them ("across": row c holds all m or n; weights of the rows' gradient, both operands of the weights' gradient).
//
// Both go to LDS by direct loads of 16 bytes a lane, ST steps deep: a barrier per step, behind which the step read last is
// loaded anew. Along: 64 values (eight 16-byte units) of each of the tile's rows. Across: 64 rows of the tile's width, which the
// transposing LDS read turns: sixteen lanes read 4 rows of 16 columns and get a column's 4 values each.
// Units are permuted on their way in (by the address that a lane loads from) so that lanes that read together touch different banks.
//
// The MFMAs take n as their rows: a lane then holds four neighbouring n of one m. The products of two tiles of 16 n change hands at
// the end, so that a lane has eight neighbours and stores 16 bytes (or 32).
//
// Bound by the MFMAs for many rows (8192 x 8192 x 8192 bf16 1.36 to 1.40 PFLOP/s, as a large library product; 16384 rows over 16 experts of
// 7168 -> 4096 903 us, 1.07, with the experts' partial blocks and 4.5 rounds of tiles), by the weights' or outputs' bytes for few (2085
// rows over 512 experts of 2560 -> 1280 500 us). Tiles of 256 x 256 read each operand's LDS half as often as 128 x 128 and leave room
// for one workgroup to a CU, so that workgroup goes round the tiles and loads the next behind the stores (985 us with a workgroup for
// each tile); of the smaller tiles two fit a CU, one of which computes while the other begins or ends.
#pragma once

#include <type_traits>

#include "exl3_grouped.h"

namespace exl3 {

struct GroupedArgs {
    const uint16_t* a;                 // rows (x, dy)
    const uint16_t* b;                 // weights; of the weights' gradient x
    void* out;
    int64_t a_ld, b_ld, b_es, out_ld, out_es;   // elements from row to row, and from expert to expert
    const int32_t* ends;
    int E, T;
    int c;                             // contraction (the weights' gradient: the expert's rows)
    int m, n;                          // outputs: columns n; the weights' gradient has m rows
    int out_dtype, vec;                // vec: the kernel of few rows may store four neighbouring outputs at once
    int rest;                          // rows of no expert become 0
    int accumulate;                    // the weights' gradient is added to what out holds
    int splits;                        // the weights' gradient: parts of an expert's rows, whose sums lie E out_es behind one another
};

enum { kGroupRows = 0, kGroupWeights = 1 };

// Four values of a column each, from 4 rows of 16 columns: sixteen lanes give the addresses of four neighbours.
typedef short s4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 lds_read_tr(const char* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p));
}

// Bits 0, 1 and 3 of a row: what the rows that the transposing read takes together differ in.
__device__ __forceinline__ int swz_across(int r) { return (r & 3) | (r >> 1 & 4); }

// A tile of R rows (along: R x 64, across: 64 x R) in LDS.
template <int R, bool ACROSS, int THREADS, bool DIRECT>
struct GroupTile {
    static constexpr int kUnits = R * 8, kLoads = kUnits / THREADS;
    static_assert(kUnits % THREADS == 0, "whole loads per thread");
    const uint16_t* p;                 // first value of the tile's step
    int64_t step;                      // elements from step to step
    int64_t ld;
    int rows, cols;                    // along: rows there are (of R), contraction left; across: contraction left, columns there are
    uint32_t off[kLoads];              // bytes from p, or kMx4Out for what is not there at any step
    u32x4_t v[DIRECT ? 1 : kLoads];

    // unit u of a step: its row and the eight values (from 8 * second on) that lie there
    __device__ __forceinline__ static int2 place(int u) {
        if constexpr (!ACROSS) {
            const int r = u >> 3;
            return make_int2(r, (u & 7) ^ (r & 7));
        } else {
            constexpr int kRow = R / 8;
            const int r = u / kRow, q = u % kRow;
            return make_int2(r, (((q >> 1) ^ (swz_across(r) & (R / 16 - 1))) << 1) | (q & 1));   // 16 columns together
        }
    }
    // p_ at the tile's first row (along) or column (across); `have` rows or columns of the tile, `left` of the contraction
    __device__ __forceinline__ void set(const uint16_t* p_, int64_t ld_, int have, int left, int t) {
        p = p_;
        ld = ld_;
        step = ACROSS ? 64 * ld_ : 64;
        rows = ACROSS ? left : have;
        cols = ACROSS ? have : left;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int2 at = place(t + i * THREADS);
            const bool in = ACROSS ? 8 * at.y < have : at.x < have;
            off[i] = in ? (uint32_t)at.x * (uint32_t)(2 * ld_) + 16 * at.y : kMx4Out;
        }
    }
    // Eight values at p + e of which n are there: unaligned, the rest 0.
    __device__ __forceinline__ static u32x4_t load_any(const uint16_t* q, int n) {
        typedef u32x4_t any_t __attribute__((aligned(2)));
        if (n >= 8) return *(const __attribute__((address_space(1))) any_t*)q;
        u32x4_t r = {};
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < n) r[i >> 1] |= (uint32_t)ldg(q + i) << (16 * (i & 1));
        return r;
    }
    // load i of the next step: to LDS, or (not DIRECT) on its way to registers
    __device__ __forceinline__ void load_one(int i, u32x4_t* lds, int t) {
        const int2 at = place(t + i * THREADS);
        if constexpr (DIRECT) {
            const __amdgpu_buffer_rsrc_t r = mx4_rsrc(reinterpret_cast<const uint8_t*>(p), 0xE0000000LL);
            const bool in = ACROSS ? at.x < rows : 8 * at.y < cols;
            lds_load16(r, in ? off[i] : kMx4Out, lds + __builtin_amdgcn_readfirstlane(t >> 6) * 64 + i * THREADS);
        } else {
            const int n = at.x < rows ? cols - 8 * at.y : 0;
            v[i] = n > 0 ? load_any(p + at.x * ld + 8 * at.y, n) : u32x4_t{};
        }
    }
    // behind a step's loads
    __device__ __forceinline__ void next() {
        p += (ACROSS ? rows : cols) > 64 ? step : 0;           // (the last step's place stays inside the matrix)
        if constexpr (ACROSS) rows -= 64;
        else cols -= 64;
    }
    __device__ __forceinline__ void load(u32x4_t* lds, int t) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_one(i, lds, t);
        next();
    }
    __device__ __forceinline__ void store(u32x4_t* lds, int t) const {
        if constexpr (!DIRECT)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) lds[t + i * THREADS] = v[i];
    }
    // Fragment of the 16 rows (or columns) of tile i from w0 on, contraction 32 ks + 8 (lane >> 4) ..
    __device__ __forceinline__ static u32x4_t frag(const u32x4_t* lds, int w0, int i, int ks, int lane) {
        const int l = lane & 15, g = lane >> 4;
        if constexpr (!ACROSS) {
            const int r = w0 + 16 * i + l;
            return lds[r * 8 + ((4 * ks + g) ^ (r & 7))];
        } else {
            const int r = 32 * ks + 8 * g + (l >> 2);          // and r + 4: the permutation takes the same value
            const char* row = reinterpret_cast<const char*>(lds) + r * (2 * R);
            const int at = ((((w0 >> 4) + i) ^ (swz_across(r) & (R / 16 - 1))) << 5) + 8 * (l & 3);
            const uint2 lo = lds_read_tr(row + at), hi = lds_read_tr(row + 4 * (2 * R) + at);
            return u32x4_t{lo.x, lo.y, hi.x, hi.y};
        }
    }
};

template <int N>
__device__ __forceinline__ void wait_step() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ float load_as(const void* p, int64_t i, int dtype) {
    if (dtype == EXL3_F32) return ldg(reinterpret_cast<const float*>(p) + i);
    const uint16_t v = ldg(reinterpret_cast<const uint16_t*>(p) + i);
    return dtype == EXL3_F16 ? h2f(v) : bf2f(v);
}

typedef f4_t f4_any_t __attribute__((aligned(4)));
typedef u32x4_t u4_any_t __attribute__((aligned(2)));

// The outputs of two tiles of 16 n, four neighbours of each per lane, to eight neighbours: of lane groups 0 and 2 the first tile's n 0 .. 7
// and 8 .. 15, of 1 and 3 the second's.
__device__ __forceinline__ void grouped_pair(f4_t& v, f4_t& w) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const auto x = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, (float)v[q]), __builtin_bit_cast(uint32_t, (float)w[q]),
                                                        false, false);
        v[q] = __builtin_bit_cast(float, (uint32_t)x[0]);
        w[q] = __builtin_bit_cast(float, (uint32_t)x[1]);
    }
}

// Eight neighbouring outputs at element i, `left` of which are there. Whole pieces at any alignment, which global memory takes (200 rows
// over 64 experts, gradient of 2049 -> 2048 weights: 548 us by single values).
template <int OP>
__device__ __forceinline__ void grouped_store(const GroupedArgs& g, int64_t i, int left, f4_t v, f4_t w) {
    typedef __attribute__((address_space(1))) f4_any_t f4_g;
    typedef __attribute__((address_space(1))) u4_any_t u4_g;
    if (left < 8) {
#pragma unroll 1
        for (int q = 0; q < (left < 8 ? left : 8); ++q) {
            float f = q < 4 ? v[q & 3] : w[q & 3];
            if (OP == kGroupWeights && g.accumulate) f += load_as(g.out, i + q, g.out_dtype);
            store_as(g.out, i + q, f, g.out_dtype);
        }
        return;
    }
    if (g.out_dtype == EXL3_F32) {
        f4_g* o = (f4_g*)(reinterpret_cast<float*>(g.out) + i);
        if (OP == kGroupWeights && g.accumulate) {
            const f4_t p = o[0], r = o[1];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[q] += p[q];
                w[q] += r[q];
            }
        }
        o[0] = v;
        o[1] = w;
        return;
    }
    u4_g* o = (u4_g*)(reinterpret_cast<uint16_t*>(g.out) + i);
    if (OP == kGroupWeights && g.accumulate) {
        const u32x4_t p = *o;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const uint16_t h = (uint16_t)(p[q >> 1] >> (16 * (q & 1)));
            const float f = g.out_dtype == EXL3_F16 ? h2f(h) : bf2f(h);
            if (q < 4) v[q & 3] += f;
            else w[q & 3] += f;
        }
    }
    u32x4_t r;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        r[q] = g.out_dtype == EXL3_F16 ? __builtin_bit_cast(uint32_t, h2_t{(_Float16)v[2 * q], (_Float16)v[2 * q + 1]})
                                       : __builtin_bit_cast(uint32_t, b2_t{(__bf16)v[2 * q], (__bf16)v[2 * q + 1]});
        r[2 + q] = g.out_dtype == EXL3_F16 ? __builtin_bit_cast(uint32_t, h2_t{(_Float16)w[2 * q], (_Float16)w[2 * q + 1]})
                                           : __builtin_bit_cast(uint32_t, b2_t{(__bf16)w[2 * q], (__bf16)w[2 * q + 1]});
    }
    *o = r;
}

// ROUND: one workgroup to a CU, which goes round the tiles.
template <int XT, int OP, bool BACROSS, int BM, int BN, int WM, int WN, int ST, int OCC, bool DIRECT, bool ROUND>
__global__ __launch_bounds__(64 * WM * WN, OCC) void grouped_kernel(GroupedArgs g) {
    constexpr int kThreads = 64 * WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    static_assert(TM > 0 && TN > 1 && TN % 2 == 0, "pairs of tiles");
    typedef GroupTile<BM, OP == kGroupWeights, kThreads, DIRECT> A;
    typedef GroupTile<BN, BACROSS, kThreads, DIRECT> B;
    constexpr int kStep = A::kUnits + B::kUnits;
    __shared__ u32x4_t lds[ST * kStep];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const unsigned nnt = (unsigned)((g.n + BN - 1) / BN);
    // Blocks of rows there are; of the weights' gradient all tiles.
    unsigned nmt = (unsigned)((g.m + BM - 1) / BM);
    if constexpr (OP == kGroupRows) {
        const unsigned most = (unsigned)(g.T / BM + g.E + 1);  // (ends that do not ascend may count rows again)
        nmt = group_blocks<BM>(g.ends, g.E, g.T, g.rest);
        nmt = nmt < most ? nmt : most;
    }
    const unsigned tiles = nmt * nnt * (OP == kGroupRows ? 1 : g.E * g.splits);
    // Where the grid goes round, what is left for the last round is taken in halves of BM / 2 rows if that fills it no more than once.
    const unsigned left_over = tiles % gridDim.x, halves = ROUND && OP == kGroupRows && 2 * left_over <= gridDim.x ? left_over : 0,
                   whole = tiles - halves;
    struct Work {
        int e;                         // expert (the weights' gradient: and E for each split before)
        int64_t row, m0, n0;           // first row of the expert or block, first outputs
        int have, left, cols;          // rows and columns of outputs there are, contraction
    };
    // The tile of a place (uniform); false where there is none.
    const auto work = [&](unsigned id, Work& w) {
        if (id >= whole + 2 * halves) return false;
        const unsigned tile = id < whole ? id : whole + (id - whole) / 2;
        unsigned mt, nt;
        if constexpr (OP == kGroupRows) {
            grouped_tile(tile, nmt, nnt, mt, nt);
            GroupSlot s = group_slot<BM>(g.ends, g.E, g.T, mt);
            if (halves && id >= whole) {
                const int skip = (id - whole) & 1 ? BM / 2 : 0, rest = s.rows - skip;
                s.row += skip;
                s.rows = rest < 0 ? 0 : rest < BM / 2 ? rest : BM / 2;
            }
            w.e = s.e;
            w.row = s.row;
            w.m0 = 0;
            w.have = s.rows;
            w.left = s.e < g.E ? g.c : 0;
        } else {
            w.e = (int)(tile / (nmt * nnt));
            grouped_tile(tile - w.e * (nmt * nnt), nmt, nnt, mt, nt);
            const int sp = w.e / g.E, e = w.e - sp * g.E;
            const int lo = __builtin_amdgcn_readfirstlane(e > 0 ? group_end(g.ends, e - 1, g.T) : 0);
            const int hi = __builtin_amdgcn_readfirstlane(group_end(g.ends, e, g.T));
            const int rows = hi > lo ? hi - lo : 0, per = ((rows + 63) / 64 + g.splits - 1) / g.splits * 64, skip = sp * per;
            w.row = skip < rows ? lo + skip : 0;
            w.left = skip < rows ? rows - skip < per ? rows - skip : per : 0;
            w.m0 = (int64_t)mt * BM;
            w.have = g.accumulate && w.left == 0 ? 0 : (int)(g.m - w.m0 < BM ? g.m - w.m0 : BM);
        }
        w.n0 = (int64_t)nt * BN;
        w.cols = (int)(g.n - w.n0 < BN ? g.n - w.n0 : BN);
        return true;
    };
    A a;
    B b;
    const auto set = [&](const Work& w) {
        if constexpr (OP == kGroupRows) {
            a.set(g.a + w.row * g.a_ld, g.a_ld, w.have, w.left, t);
            const uint16_t* m = g.b + (w.e < g.E ? w.e : 0) * g.b_es;
            b.set(m + (BACROSS ? w.n0 : w.n0 * g.b_ld), g.b_ld, w.cols, w.left, t);
        } else {
            a.set(g.a + w.row * g.a_ld + w.m0, g.a_ld, w.have, w.left, t);
            b.set(g.b + w.row * g.b_ld + w.n0, g.b_ld, w.cols, w.left, t);
        }
    };
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    f4_t acc[TM][TN];
    constexpr int kLoads = A::kLoads + B::kLoads, kFrags = TM + TN, kMul = TM * TN;
    // Fragments of half a step (32) from `base`, with `loads` the loads of a step to `to`, and with `products` those of the half step
    // that ma and mb hold, in turn: reads or loads in a row wait for the LDS's and the caches' ports, and a wave issues in order, so
    // the MFMAs behind them would wait too. Reads and loads are through after three quarters.
    const auto half = [&](auto loads, auto products, const u32x4_t* base, int ks, u32x4_t (&fa)[TM], u32x4_t (&fb)[TN], u32x4_t* to,
                          const u32x4_t (&ma)[TM], const u32x4_t (&mb)[TN]) {
        constexpr int kLead = kMul * 3 / 4;
        const auto mul = [&](int m) { acc[m / TN][m % TN] = mfma16<XT>(mb[m % TN], ma[m / TN], acc[m / TN][m % TN]); };
#pragma unroll
        for (int f = 0; f < kFrags; ++f) {
            if constexpr (loads)
#pragma unroll
                for (int i = f * kLoads / kFrags; i < (f + 1) * kLoads / kFrags; ++i) {
                    if (i < A::kLoads) a.load_one(i, to, t);
                    else b.load_one(i - A::kLoads, to + A::kUnits, t);
                }
            if (f < TN) fb[f] = B::frag(base + A::kUnits, wn, f, ks, lane);
            else fa[f - TN] = A::frag(base, wm, f - TN, ks, lane);
            if constexpr (products) {
#pragma unroll
                for (int m = f * kLead / kFrags; m < (f + 1) * kLead / kFrags; ++m) mul(m);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (loads) {
            a.next();
            b.next();
        }
        if constexpr (products)
#pragma unroll
            for (int m = kLead; m < kMul; ++m) mul(m);
    };
    const std::true_type yes;
    const std::false_type no;
    const auto start = [&] {                                   // the first steps' loads
        if constexpr (DIRECT) {
#pragma unroll
            for (int c = 0; c < ST; ++c) {                     // (past the last: zeros)
                a.load(lds + c * kStep, t);
                b.load(lds + c * kStep + A::kUnits, t);
            }
        } else {
            a.load(nullptr, t);
            b.load(nullptr, t);
        }
    };
    const auto store = [&](const Work& w) {
        int64_t at = (OP == kGroupRows ? w.row * g.out_ld : w.e * g.out_es + w.m0 * g.out_ld) + w.n0;
        int m = wm + (lane & 15), n = wn + 16 * (lane >> 4 & 1) + 8 * (lane >> 5);
        asm volatile("" : "+v"(m), "+v"(n));                   // (addresses are worked out here, not kept)
        at += m * g.out_ld + n;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; j += 2) {
                grouped_pair(acc[i][j], acc[i][j + 1]);
                if (m + 16 * i < w.have && n + 16 * j < w.cols)
                    grouped_store<OP>(g, at + 16 * j, w.cols - n - 16 * j, acc[i][j], acc[i][j + 1]);
            }
            at += 16 * g.out_ld;
        }
    };
    unsigned block = blockIdx.x;
    Work w, next;
    if (!work(grouped_place(kChunk, block), w)) return;
    set(w);
    start();
    for (;;) {
        const int steps = (w.left + 63) / 64;
        const bool live = wm < w.have;                         // (uniform) this wave's rows are there
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{};
        u32x4_t fa[TM], fb[TN], ga[TM], gb[TN];
        if constexpr (DIRECT) {
            // Half a step's fragments are read while the half before is multiplied. The barrier is between the halves: behind it the
            // next step lies in LDS, and the one whose second half is on its way to the MFMAs is loaded anew.
            wait_step<kLoads * (ST - 1)>();
            __builtin_amdgcn_s_barrier();
            int at = 0;
            if (live) {
                half(no, no, lds, 0, fa, fb, nullptr, ga, gb);
                for (int c = 0; c < steps; ++c) {
                    const int then = at == ST - 1 ? 0 : at + 1;
                    __builtin_amdgcn_sched_barrier(0);
                    half(no, yes, lds + at * kStep, 1, ga, gb, nullptr, fa, fb);
                    __builtin_amdgcn_sched_barrier(0);
                    wait_step<kLoads * (ST - 2)>();
                    __builtin_amdgcn_s_barrier();
                    __builtin_amdgcn_sched_barrier(0);
                    half(yes, yes, lds + then * kStep, 0, fa, fb, lds + at * kStep, ga, gb);
                    at = then;
                }
            } else {                                           // loads alone
                for (int c = 0; c < steps; ++c) {
                    wait_step<kLoads * (ST - 2)>();
                    __builtin_amdgcn_s_barrier();
                    a.load(lds + at * kStep, t);
                    b.load(lds + at * kStep + A::kUnits, t);
                    at = at == ST - 1 ? 0 : at + 1;
                }
            }
            wait_step<0>();                                    // the LDS is the next tile's, or behind the end the next workgroup's
            if constexpr (ROUND) __builtin_amdgcn_s_barrier();
        } else {
            a.store(lds, t);
            b.store(lds + A::kUnits, t);
            __syncthreads();
            for (int c = 0; c < steps; ++c) {
                a.load(nullptr, t);
                b.load(nullptr, t);
                if (live) {
                    half(no, no, lds + (c & 1) * kStep, 0, fa, fb, nullptr, ga, gb);
                    half(no, yes, lds + (c & 1) * kStep, 1, ga, gb, nullptr, fa, fb);
#pragma unroll
                    for (int m = 0; m < kMul; ++m) acc[m / TN][m % TN] = mfma16<XT>(gb[m % TN], ga[m / TN], acc[m / TN][m % TN]);
                }
                u32x4_t* o = lds + (~c & 1) * kStep;
                a.store(o, t);
                b.store(o + A::kUnits, t);
                __syncthreads();
            }
        }
        block += gridDim.x;
        const bool more = ROUND && work(grouped_place(kChunk, block), next);
        if (more) {                                            // on their way while the outputs are stored
            set(next);
            start();
        }
        if (live) store(w);
        if (!more) return;
        w = next;
    }
}

// ------------------------------------------------------------------------------------------------ launches
// Tiles of a call: rows (and of the weights' gradient columns) of a workgroup; unaligned operands go through registers.
enum { kTile256 = 0, kTile128 = 1, kTile64 = 2, kTile32 = 3, kTileAny128 = 4, kTileAny32 = 5, kTileFew = 6 };

// The kernel timing may repeat a launch: one that adds to its output runs once, and untimed then.
#define GROUPED_LAUNCH(name, kernel, grid, block, accumulate, st, ...)                  \
    do {                                                                               \
        if ((accumulate) && prof_repeat() > 1) {                                       \
            EXL3_CHECK_ARG(grid_fits(grid, block), "%s: grid too large", name);        \
            hipLaunchKernelGGL(kernel, grid, block, 0, st, __VA_ARGS__);               \
            EXL3_CHECK_HIP(hipGetLastError());                                         \
        } else {                                                                       \
            EXL3_LAUNCH(name, kernel, grid, block, 0, st, __VA_ARGS__);                \
        }                                                                              \
    } while (0)

template <int XT, int OP, bool BACROSS, int BM, int BN, int WM, int WN, int ST, int OCC, bool DIRECT>
static int launch_grouped(const char* name, const GroupedArgs& g, hipStream_t st) {
    constexpr bool ROUND = BM == 256;
    const int64_t nmt = OP == kGroupRows ? group_slots(g.T, g.E, BM, g.rest) : (g.m + BM - 1) / BM * g.E * g.splits;
    const int64_t tiles = nmt * ((g.n + BN - 1) / BN);
    constexpr int64_t kRound = 8 * kChunk;
    EXL3_CHECK_ARG(tiles <= kMx4Grid * 256 / (64 * WM * WN) - kRound, "%s: grid too large", name);
    const int64_t grid = (tiles + kRound - 1) / kRound * kRound;
    const auto kernel = grouped_kernel<XT, OP, BACROSS, BM, BN, WM, WN, ST, OCC, DIRECT, ROUND>;
    GROUPED_LAUNCH(name, kernel, dim3((unsigned)(ROUND && grid > kRound ? kRound : grid)), dim3(64 * WM * WN), g.accumulate, st, g);
    return EXL3_OK;
}

template <int XT, bool BACROSS>
static int launch_grouped_rows(const GroupedArgs& g, int tile, hipStream_t st) {
    const char* name = "grouped_rows";
    switch (tile) {
        case kTile256: return launch_grouped<XT, kGroupRows, BACROSS, 256, 256, 2, 4, 2, 2, true>(name, g, st);
        case kTile128: return launch_grouped<XT, kGroupRows, BACROSS, 128, 128, 2, 2, 2, 2, true>(name, g, st);
        case kTile64: return launch_grouped<XT, kGroupRows, BACROSS, 64, 128, 1, 4, 3, 2, true>(name, g, st);
        case kTile32: return launch_grouped<XT, kGroupRows, BACROSS, 32, 128, 1, 4, 4, 2, true>(name, g, st);
        case kTileAny128: return launch_grouped<XT, kGroupRows, BACROSS, 128, 128, 2, 2, 2, 2, false>(name, g, st);
        default: return launch_grouped<XT, kGroupRows, BACROSS, 32, 128, 1, 4, 2, 2, false>(name, g, st);
    }
}

int grouped_rows_few(const GroupedArgs& g, int dtype, hipStream_t st);   // aligned, at most 8192 inputs
int grouped_rows_along(const GroupedArgs& g, int dtype, int tile, hipStream_t st);
int grouped_rows_across(const GroupedArgs& g, int dtype, int tile, hipStream_t st);
int grouped_weights(const GroupedArgs& g, int dtype, int tile, hipStream_t st);
// out = the sum of g.splits parts [E m][n4] that lie `stride` behind one another
int grouped_reduce(const GroupedArgs& g, const float* part, int64_t n4, int64_t stride, hipStream_t st);

}  // namespace exl3
