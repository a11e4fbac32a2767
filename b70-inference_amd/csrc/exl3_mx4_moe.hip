// Routed MoE layer over experts with MX4 weights. Per call, on the caller's stream:
//   align    pairs (token, slot) grouped by expert and cut into blocks of rows (exl3_moe.hip, shared with the EXL3 layer;
//            the tables' entries are (codes, scales, base) instead of (trellis, suh, svh))
//   gateup   workgroup per (block, 128 columns of I): both projections over H, act(gate, up) in fp32, rounded to x's type
//            (the down product's operand: one of more bits, in two parts, would double its MFMAs, its LDS and its reads of rows;
//            this rounding adds to the output's: 1.4 times the error of a 16-bit output, and an fp32 output has no more than
//            x's type's 8 or 11 bits of the middle). fp16 does not hold every magnitude that a product of two sums has, so fp16
//            middles carry a power of two per workgroup's columns (mid_exponent in exl3_mx4.h: 0.3 us of the one token's time
//            below, 3 of the 1024 tokens')
//   down     workgroup per (block, 256 columns of H) over I: y[pair] = routing weight * sum, fp32
//   combine  out[t] = sum of the token's y rows in slot order
// Few pairs take two launches instead: gateup per (pair, 16 columns of I), down per (token, 16 columns of H) over all of the
// token's slots.
// Bound by the weights' bytes: 1024 tokens, top-10 of 512 experts 2560 -> 640, 421 us for 1.35 GB (align 31, gateup 239, down 138,
// combine 18); 260 tokens, top-2 of 32 experts 7168 -> 2048 and a shared one, 256 us for 0.78 GB (14, 158, 89, 6); one token,
// top-10 of 512 experts 2048 -> 512, 12.3 us replayed for 17 MB, two chains of load, sum and store.
#include "exl3_moe.h"
#include "exl3_moe_dev.h"
#include "exl3_mx4.h"
#include "exl3_mx4_decode.h"
#include "exl3_mx4_wide.h"
#include "exl3_mx4_plan.h"
#include "exl3_plan.h"

namespace exl3 {

int launch_align(const RouteArgs& r, hipStream_t st);           // exl3_moe.hip

struct Mx4MoeArgs {
    const uint8_t* x;
    int64_t x_ld;                      // bytes
    int M, H, I, slots;
    const ItemDesc* blocks;
    int max_blocks;
    const int* pair_tok;
    const float* pair_w;
    const int* pair_of;
    uint16_t* mid;                     // [pairs][I] in x's type
    int8_t* mexp;                      // fp16: exponents of mid's groups of 128 columns, [pairs][ceil(I / 128)]
    float* y;                          // [pairs][H]
    int act;
    float limit;
    void* out;
    int64_t out_ld;
    int out_dtype;
};

// ------------------------------------------------------------------------------------------------ few pairs
// Without the align step: a workgroup takes a pair (token, slot) as it stands. An expert that several tokens picked is read
// once for each (from the L2).
struct Mx4PairArgs {
    const uint8_t* x;
    int64_t x_ld;                      // bytes
    int M, H, I, topk, slots, E, shared;
    const int32_t* ids;
    const float* tw;
    const int64_t* tables;             // [9][E]
    uint16_t* mid;                     // [M * slots][I]
    int8_t* mexp;                      // fp16: exponents of mid's groups of 16 columns, [M * slots][I / 16]
    int act;
    float limit;
    void* out;
    int64_t out_ld;
    int out_dtype, vec;
    // expert of slot j of token t, -1: none
    __device__ __forceinline__ int expert(int t, int j) const {
        const int e = j < topk ? ldg(ids + (int64_t)t * topk + j) : shared;
        return e >= 0 && e < E ? e : -1;
    }
    __device__ __forceinline__ int64_t entry(int row, int e) const { return ldg(tables + (int64_t)row * E + e); }
};

// Workgroup per (pair, 16 columns of I): the gate and the up tile.
template <int XT>
__global__ __launch_bounds__(512) void mx4_gateup_pair_kernel(Mx4PairArgs a, int xbytes) {
    extern __shared__ f4_t red[];
    char* lds = reinterpret_cast<char*>(red);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const unsigned nc = (unsigned)a.I / 16, pair = blockIdx.x / nc;
    const int t = pair / (unsigned)a.slots, e = __builtin_amdgcn_readfirstlane(a.expert(t, pair - t * a.slots)), i0 = (blockIdx.x % nc) * 16;
    if (e < 0) return;
    const int kb = a.H / 32, ng = (kb + 4 * kMx4Group - 1) / (4 * kMx4Group);
    Mx4Decode<XT> p[2];
    typename Mx4Decode<XT>::Group q[2], nx[2];
    int base[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        p[i].kb = kb;
        base[i] = XT == kRowF16 ? (int)a.entry(3 * i + 2, e) : 0;
        p[i].tile.set(reinterpret_cast<const uint8_t*>(a.entry(3 * i, e)), reinterpret_cast<const uint8_t*>(a.entry(3 * i + 1, e)), i0,
                      a.I, kb, lane);
        p[i].load(wave, lane, q[i]);
    }
    const Mx4X x = mx4_stage_x<XT>(lds, 1, kb, [&](int) { return a.x + (int64_t)t * a.x_ld; }, [](int) { return (const uint8_t*)nullptr; });
    __syncthreads();
    f4_t acc[2] = {f4_t{}, f4_t{}};
    for (int gi = wave; gi < ng; gi += waves) {
        const bool more = gi + waves < ng;                     // uniform
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (more) p[i].load(gi + waves, lane, nx[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            p[i].mul(gi, lane, x, 1, base[i], q[i], acc[i]);
            q[i] = nx[i];
        }
    }
    f4_t* out = reinterpret_cast<f4_t*>(lds + xbytes);
    out[wave * 64 + lane] = acc[0];
    out[(waves + wave) * 64 + lane] = acc[1];
    __syncthreads();
    if (wave != 0 || (lane & 15) != 0) return;                 // column 0 of the products is the row
    const f4_t g = mx4_decode_sum(out, waves, 0, lane), u = mx4_decode_sum(out, waves, 1, lane);
    f4_t v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        v[j] = act_mul_dev(__builtin_ldexpf(g[j], base[0]), __builtin_ldexpf(u[j], base[1]), a.act, a.limit);
    if constexpr (XT == kRowF16) {                             // (the four lanes here are all of them)
        uint32_t m = 0, top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, magnitude_bits(v[j]));
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, (uint32_t)__builtin_amdgcn_readlane((int)m, 16 * j));
        const int ex = mid_exponent(top);
        if (ex != 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __builtin_ldexpf(v[j], -ex);
        if (lane == 0) a.mexp[(int64_t)pair * nc + blockIdx.x % nc] = (int8_t)ex;
    }
    store4_as(a.mid, (int64_t)pair * a.I + i0 + 4 * (lane >> 4), v, XT == kRowF16 ? EXL3_F16 : EXL3_BF16);
}

// Workgroup per (token, 16 columns of H): the token's slots after one another, their groups of 512 rows of I over the waves; a
// wave adds a slot's sum, times its routing weight, when it goes on to another. fp16: the sum is held at the largest exponent of the
// middle's groups so far.
template <int XT>
__global__ __launch_bounds__(1024) void mx4_down_pair_kernel(Mx4PairArgs a, int xbytes) {
    extern __shared__ f4_t red[];
    char* lds = reinterpret_cast<char*>(red);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const unsigned nc = (unsigned)a.H / 16;
    const int t = blockIdx.x / nc, h0 = (blockIdx.x % nc) * 16;
    const int kb = a.I / 32, ng = (kb + 4 * kMx4Group - 1) / (4 * kMx4Group), all = a.slots * ng;
    Mx4Decode<XT> p;
    p.kb = kb;
    typename Mx4Decode<XT>::Group q, nx;
    constexpr int kNone = -1000;
    int base = 0, nbase = 0, e = -1, ne = -1;                  // of q's and nx's slots
    int held = XT == kRowF16 ? kNone : 0;                      // exponent of acc
    struct Exps {
        uint32_t b[kMx4Group];                                 // of this lane's block of each chunk, two bytes
    } qe, nqe;
    const auto fetch = [&](int gi, int& ex, int& bs, typename Mx4Decode<XT>::Group& o, Exps& oe) {
        const int j = gi / ng;
        ex = __builtin_amdgcn_readfirstlane(a.expert(t, j));
        if (ex < 0) return;                                    // uniform
        bs = XT == kRowF16 ? (int)a.entry(8, ex) : 0;
        p.tile.set(reinterpret_cast<const uint8_t*>(a.entry(6, ex)), reinterpret_cast<const uint8_t*>(a.entry(7, ex)), h0, a.H, kb, lane);
        p.load(gi - j * ng, lane, o);
        if constexpr (XT == kRowF16) {
            const uint16_t* ep = reinterpret_cast<const uint16_t*>(a.mexp + ((int64_t)t * a.slots + j) * (a.I / 16));
#pragma unroll
            for (int u = 0; u < kMx4Group; ++u) {
                const int b = 4 * (kMx4Group * (gi - j * ng) + u) + (lane >> 4);
                oe.b[u] = ldg(ep + (b < kb ? b : kb - 1));     // (past the row's end, beside x that is 0: the last block's)
            }
        }
    };
    fetch(wave, e, base, q, qe);
    // (slots without an expert have no middle row: their pair's, which nobody reads)
    const Mx4X x = mx4_stage_x<XT>(lds, a.slots, kb, [&](int j) {
        return reinterpret_cast<const uint8_t*>(a.mid + ((int64_t)t * a.slots + j) * a.I); }, [](int) { return (const uint8_t*)nullptr; });
    __syncthreads();
    f4_t tot = {}, acc = {};
    for (int gi = wave; gi < all; gi += waves) {
        const int j = gi / ng;
        const bool more = gi + waves < all;
        if (more) fetch(gi + waves, ne, nbase, nx, nqe);
        if (e >= 0) {
            const Mx4X xj = {x.p + j * x.stride, x.stride, x.sstride, x.scales};
            bool plain = true;
            if constexpr (XT == kRowF16) {
                int top = 0;
                plain = __ballot((qe.b[0] | qe.b[1] | qe.b[2] | qe.b[3]) != 0) == 0;
                if (!plain) {
                    top = -126;
#pragma unroll
                    for (int u = 0; u < kMx4Group; ++u) top = max(top, max((int)(int8_t)qe.b[u], (int)(int8_t)(qe.b[u] >> 8)));
                    top = max(top, __shfl_xor(top, 16));
                    top = __builtin_amdgcn_readfirstlane(max(top, __shfl_xor(top, 32)));
                }
                if (top > held) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i] = __builtin_ldexpf(acc[i], held - top);
                    held = top;
                }
                plain = plain && held == 0;
                if (!plain)
                    p.mul(gi - j * ng, lane, xj, 1, base, q, acc, [&](int u, int v, u32x4_t f) {
                        return half_shift(f, (int)(int8_t)(qe.b[u] >> (v < 2 ? 0 : 8)) - held);
                    });
            }
            if (plain) p.mul(gi - j * ng, lane, xj, 1, base, q, acc);
        }
        if (!more || (gi + waves) / ng != j) {
            if (e >= 0) {
                const float w = j < a.topk ? ldg(a.tw + (int64_t)t * a.topk + j) : 1.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) tot[i] += w * __builtin_ldexpf(acc[i], base + held);
            }
            acc = f4_t{};
            if (XT == kRowF16) held = kNone;
        }
        q = nx;
        qe = nqe;
        e = ne;
        base = nbase;
    }
    f4_t* out = reinterpret_cast<f4_t*>(lds + xbytes);
    out[wave * 64 + lane] = tot;
    __syncthreads();
    if (wave != 0 || (lane & 15) != 0) return;
    const f4_t v = mx4_decode_sum(out, waves, 0, lane);
    const int64_t o = (int64_t)t * a.out_ld + h0 + 4 * (lane >> 4);
    if (a.vec) {
        store4_as(a.out, o, v, a.out_dtype);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) store_as(a.out, o + i, v[i], a.out_dtype);
    }
}

// LDS of the two kernels; the pair path is taken where both are at most 64 KB.
struct Mx4PairShape {
    int wg, xg, wd, xd;
};
static bool pair_shape(int H, int I, int slots, Mx4PairShape& s) {
    const int kh = H / 32, ki = I / 32, gh = (kh + 4 * kMx4Group - 1) / (4 * kMx4Group), gi = (ki + 4 * kMx4Group - 1) / (4 * kMx4Group);
    s.wg = mx4_decode_waves(gh, 8);
    s.wd = mx4_decode_waves(gi * slots, 16);
    s.xg = mx4_x_bytes<kRowF16>(1, kh);
    s.xd = mx4_x_bytes<kRowF16>(slots, ki);
    return s.xg + s.wg * 2048 <= 65536 && s.xd + s.wd * 1024 <= 65536;
}

template <int XT>
static int launch_pairs(const Mx4PairArgs& a, const Mx4PairShape& s, hipStream_t st) {
    EXL3_LAUNCH("mx4_moe_gateup_pair", mx4_gateup_pair_kernel<XT>, dim3((unsigned)(a.M * a.slots * (a.I / 16))), dim3(64 * s.wg),
                (size_t)s.xg + s.wg * 2048, st, a, s.xg);
    EXL3_LAUNCH("mx4_moe_down_pair", mx4_down_pair_kernel<XT>, dim3((unsigned)(a.M * (a.H / 16))), dim3(64 * s.wd),
                (size_t)s.xd + s.wd * 1024, st, a, s.xd);
    return EXL3_OK;
}

// ------------------------------------------------------------------------------------------------ blocks of many rows
// Waves 0 and 1 take 64 gate columns each, waves 2 and 3 the up columns; they meet in LDS, 32 rows at a time.
constexpr int kMx4CS = 264;            // floats per row there: gate columns at 0, up columns at 132

template <int XT, int RG>
__global__ __launch_bounds__(256, mx4_wide_occ(RG)) void mx4_gateup_wide_kernel(Mx4MoeArgs a) {
    typedef Mx4Wide<XT, RG> L;
    constexpr int kC = 32 * kMx4CS * 4 / 16;
    __shared__ u32x4_t lds[L::kLds > kC ? L::kLds : kC];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const unsigned nc = ((unsigned)a.I + 127) / 128;
    const ItemDesc* d = a.blocks + blockIdx.x / nc;
    const int cnt = d->cnt, p0 = d->p0, i0 = (int)(blockIdx.x % nc) * 128, pj = wave >> 1;
    if (cnt == 0) return;
    L p;
    p.kb = a.H / 32;
    p.lds = lds;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
        const int m = (t >> 3) + 32 * i;
        p.xp[i] = a.x + (int64_t)ldg(a.pair_tok + p0 + (m < cnt ? m : cnt - 1)) * a.x_ld;
    }
    p.base = XT == kRowF16 ? (int)d->tab[3 * pj + 2] : 0;
    p.weights(reinterpret_cast<const uint8_t*>(d->tab[3 * pj]), reinterpret_cast<const uint8_t*>(d->tab[3 * pj + 1]),
              i0 + 64 * (wave & 1), a.I, lane);
    typename L::Acc acc;
    L::zero(acc);
    p.run(t, 0, 1 << 30, acc);
    const int bg = XT == kRowF16 ? (int)d->tab[2] : 0, bu = XT == kRowF16 ? (int)d->tab[5] : 0;
    float* C = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int j = 0; j < RG; ++j) {
        if (32 * j >= cnt) break;                              // uniform
        if (j > 0) __syncthreads();
        L::each(acc, j, lane, [&](int row, int n, f4_t v) {
            *reinterpret_cast<f4_t*>(C + row * kMx4CS + 132 * pj + 64 * (wave & 1) + n) = v;
        });
        __syncthreads();
        const int m = 32 * j + (t >> 3);
        f4_t v[4];
        uint32_t top = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = 32 * q + 4 * (t & 7);
            const f4_t gv = *reinterpret_cast<const f4_t*>(C + (t >> 3) * kMx4CS + col);
            const f4_t uv = *reinterpret_cast<const f4_t*>(C + (t >> 3) * kMx4CS + 132 + col);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[q][e] = act_mul_dev(__builtin_ldexpf(gv[e], bg), __builtin_ldexpf(uv[e], bu), a.act, a.limit);
                if (i0 + col < a.I) top = max(top, magnitude_bits(v[q][e]));
            }
        }
        if constexpr (XT == kRowF16) {                         // eight lanes hold a row's 128 columns
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
            const int ex = mid_exponent(top);
            if (__ballot(ex != 0))                             // uniform
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[q][e] = __builtin_ldexpf(v[q][e], -ex);
            if (m < cnt && (t & 7) == 0) a.mexp[(int64_t)(p0 + m) * nc + blockIdx.x % nc] = (int8_t)ex;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = 32 * q + 4 * (t & 7);
            if (m < cnt && i0 + col < a.I)
                store4_as(a.mid, (int64_t)(p0 + m) * a.I + i0 + col, v[q], XT == kRowF16 ? EXL3_F16 : EXL3_BF16);
        }
    }
}

template <int XT, int RG>
__global__ __launch_bounds__(256, mx4_wide_occ(RG)) void mx4_down_wide_kernel(Mx4MoeArgs a) {
    constexpr bool kMid = XT == kRowF16;
    typedef Mx4Wide<XT, RG, kMid> L;
    __shared__ u32x4_t lds[L::kLds];
    __shared__ int s_er[kMid ? 64 * RG : 1];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const unsigned nc = ((unsigned)a.H + 255) / 256;
    const ItemDesc* d = a.blocks + blockIdx.x / nc;
    const int cnt = d->cnt, p0 = d->p0, h0 = (int)(blockIdx.x % nc) * 256 + 64 * wave;
    if (cnt == 0) return;
    L p;
    p.kb = a.I / 32;
    p.lds = lds;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
        const int m = (t >> 3) + 32 * i;
        p.xp[i] = reinterpret_cast<const uint8_t*>(a.mid + (int64_t)(p0 + (m < cnt ? m : cnt - 1)) * a.I);
        if constexpr (kMid) s_er[32 * RG + m] = (m < cnt ? m : cnt - 1) * ((a.I + 127) / 128);   // (the wave's own rows: no barrier)
    }
    p.xe = kMid ? a.mexp + (int64_t)p0 * ((a.I + 127) / 128) : nullptr;
    p.er = s_er;
    p.base = XT == kRowF16 ? (int)d->tab[8] : 0;
    p.weights(reinterpret_cast<const uint8_t*>(d->tab[6]), reinterpret_cast<const uint8_t*>(d->tab[7]), h0, a.H, lane);
    typename L::Acc acc;
    L::zero(acc);
    p.run(t, 0, 1 << 30, acc);
#pragma unroll
    for (int j = 0; j < RG; ++j)
        L::each(acc, j, lane, [&](int row, int n, f4_t v) {
            const int m = 32 * j + row;
            if (m >= cnt || h0 + n >= a.H) return;
            const float w = ldg(a.pair_w + p0 + m);
            const int ex = p.base + (kMid ? s_er[m] : 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = w * __builtin_ldexpf(v[e], ex);
            *reinterpret_cast<f4_t*>(a.y + (int64_t)(p0 + m) * a.H + h0 + n) = v;
        });
}

// out[t] = sum of token t's y rows in slot order, four columns per thread; tokens from `first` on.
__global__ __launch_bounds__(256) void mx4_combine_kernel(Mx4MoeArgs a, int first, int ncb, int vec) {
    const int t = first + (int)(blockIdx.x / (unsigned)ncb), c = 4 * ((blockIdx.x % (unsigned)ncb) * 256 + threadIdx.x);
    if (c >= a.H) return;
    f4_t v = {};
    const int* po = a.pair_of + (int64_t)t * a.slots;
    for (int j0 = 0; j0 < a.slots; j0 += 8) {
        int pr[8];
        f4_t y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) pr[j] = j0 + j < a.slots ? po[j0 + j] : -1;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (pr[j] >= 0) y[j] = ldg(reinterpret_cast<const f4_t*>(a.y + (int64_t)pr[j] * a.H + c));   // uniform
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (pr[j] >= 0)
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] += y[j][q];
    }
    const int64_t o = (int64_t)t * a.out_ld + c;
    if (vec) {
        store4_as(a.out, o, v, a.out_dtype);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) store_as(a.out, o + q, v[q], a.out_dtype);
    }
}

template <int XT, int RG>
static int mx4_moe_wide(const Mx4MoeArgs& a, hipStream_t st) {
    EXL3_LAUNCH("mx4_moe_gateup_wide", (mx4_gateup_wide_kernel<XT, RG>), dim3((unsigned)(a.max_blocks * ((a.I + 127) / 128))),
                dim3(256), 0, st, a);
    EXL3_LAUNCH("mx4_moe_down_wide", (mx4_down_wide_kernel<XT, RG>), dim3((unsigned)(a.max_blocks * ((a.H + 255) / 256))),
                dim3(256), 0, st, a);
    return EXL3_OK;
}

template <int XT>
static int mx4_moe_launch(const Mx4MoeArgs& a, int rows, hipStream_t st) {
    if (rows == 32) return mx4_moe_wide<XT, 1>(a, st);
    if (rows == 64) return mx4_moe_wide<XT, 2>(a, st);
    return mx4_moe_wide<XT, 4>(a, st);
}

// Sizes that a call takes.
static bool moe_sizes(int64_t M, int64_t H, int64_t I, int64_t topk, int64_t E) {
    return M >= 0 && M <= (1 << 24) && topk >= 0 && topk <= 64 && E > 0 && E <= kMoeMaxExperts && H > 0 && I > 0 && H % 32 == 0 &&
           I % 32 == 0 && H <= (1 << 20) && I <= (1 << 20);
}

// The path of a call of npairs pairs and its scratch.
struct Mx4MoeShape {
    bool pairs;
    Mx4PairShape ps;
    int rows;                          // of a block
    int64_t max_blocks;
    size_t bytes;
};
// Pairs as they stand while they, and the weights they ask for, repeated experts and all, are few: pairs / blocks, us: 512 experts of
// 2048 -> 512 at 80 and 160 pairs 42 / 57, 71 / 90; of 2560 -> 640 at 80 and 160 69 / 74, 129 / 117; 64 of 4096 -> 1408 at 48
// 94.8 / 93.6; 32 of 7168 -> 2048 at 16 and 32 93 / 103, 173 / 150; 8 of 4096 -> 4096 at 8 and 12 54 / 73, 75 / 75.
static Mx4MoeShape moe_shape(int64_t npairs, int64_t H, int64_t I, int64_t slots, int64_t E) {
    Mx4MoeShape s{};
    const size_t np = (size_t)npairs;
    s.pairs = npairs > 0 && npairs <= 160 && npairs * H * I <= 210000000 && pair_shape((int)H, (int)I, (int)slots, s.ps);
    if (s.pairs) {
        s.bytes = carve_size(np * I, 2) + carve_size(np * I / 16, 1);
        return s;
    }
    s.rows = mx4_moe_rows(npairs, E);
    s.max_blocks = mx4_max_blocks(npairs, E, s.rows);
    s.bytes = carve_size((size_t)s.max_blocks, sizeof(ItemDesc)) + carve_size(2 * np, 4) + carve_size(np, 4) + carve_size(np * I, 2) +
              carve_size(np * ((I + 127) / 128), 1) + carve_size(np * H, 4);
    return s;
}

static int mx4_moe(const void* x, int64_t x_ld, int x_dtype, int64_t M, int64_t H, int64_t I, const int32_t* topk_ids,
                   const float* topk_w, int64_t topk, int64_t E, const int64_t* tables, int act, float act_limit, int64_t shared,
                   void* out, int64_t out_ld, int out_dtype, const CallScratch& s, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    EXL3_CHECK_ARG(x_dtype == EXL3_F16 || x_dtype == EXL3_BF16, "exl3_mx4_moe_forward: x must be fp16 or bf16");
    EXL3_CHECK_ARG(out_dtype == EXL3_F16 || out_dtype == EXL3_F32 || out_dtype == EXL3_BF16,
                   "exl3_mx4_moe_forward: out must be fp16, bf16 or fp32");
    EXL3_CHECK_ARG(act == EXL3_ACT_SILU || act == EXL3_ACT_GELU_TANH, "exl3_mx4_moe_forward: unknown activation %d", act);
    EXL3_CHECK_ARG(M >= 0 && topk >= 0 && topk <= 64 && E > 0 && E <= kMoeMaxExperts,
                   "exl3_mx4_moe_forward: M=%lld topk=%lld E=%lld out of range", (long long)M, (long long)topk, (long long)E);
    EXL3_CHECK_ARG(H > 0 && I > 0 && H % 32 == 0 && I % 32 == 0 && H <= (1 << 20) && I <= (1 << 20),
                   "exl3_mx4_moe_forward: H and I must be multiples of 32 (up to 2^20)");
    EXL3_CHECK_ARG(x_ld >= H && out_ld >= H, "exl3_mx4_moe_forward: row strides must cover H");
    EXL3_CHECK_ARG(shared < E, "exl3_mx4_moe_forward: shared expert index %lld >= E", (long long)shared);
    if (M == 0) return EXL3_OK;
    EXL3_CHECK_ARG(x && tables && out && (topk == 0 || (topk_ids && topk_w)), "exl3_mx4_moe_forward: null pointer");
    EXL3_CHECK_ARG(aligned(x, 16) && (M == 1 || x_ld % 8 == 0) && aligned(out, out_dtype == EXL3_F32 ? 4 : 2),
                   "exl3_mx4_moe_forward: x rows must be 16-byte aligned");
    const int64_t slots = topk + (shared >= 0 ? 1 : 0), npairs = M * slots;
    // pairs index 32-bit tables; the grids hold a workgroup per block and 16 columns
    EXL3_CHECK_ARG(M <= (1 << 24) && npairs <= (1 << 24) && M <= ((int64_t)1 << 45) / x_ld && M <= ((int64_t)1 << 45) / out_ld,
                   "exl3_mx4_moe_forward: too many tokens");

    const int vec = out_ld % 4 == 0 && aligned(out, out_dtype == EXL3_F32 ? 16 : 8);
    const Mx4MoeShape sh = moe_shape(npairs, H, I, slots, E);
    if (sh.pairs) {
        const size_t np = (size_t)npairs;
        Carve c{};
        const int rc = call_scratch("exl3_mx4_moe_forward", sh.bytes, s, st, &c);
        if (rc) return rc;
        uint16_t* mid = c.take<uint16_t>(np * I);
        int8_t* mexp = c.take<int8_t>(np * I / 16);
        if (!mexp) return fail(EXL3_ERR_INVALID, "exl3_mx4_moe_forward: workspace carve failed");
        const Mx4PairArgs p{reinterpret_cast<const uint8_t*>(x), 2 * x_ld, (int)M, (int)H, (int)I, (int)topk, (int)slots, (int)E,
                            (int)shared, topk_ids, topk_w, tables, mid, mexp, act, act_limit, out,
                            out_ld, out_dtype, vec};
        return x_dtype == EXL3_F16 ? launch_pairs<kRowF16>(p, sh.ps, st) : launch_pairs<kRowBF16>(p, sh.ps, st);
    }

    Mx4MoeArgs a{};
    a.x = reinterpret_cast<const uint8_t*>(x);
    a.x_ld = 2 * x_ld;
    a.M = (int)M;
    a.H = (int)H;
    a.I = (int)I;
    a.slots = (int)slots;
    a.act = act;
    a.limit = act_limit;
    a.out = out;
    a.out_ld = out_ld;
    a.out_dtype = out_dtype;
    const int rows = sh.rows;
    a.max_blocks = (int)sh.max_blocks;
    const int64_t nci = (I + 127) / 128, nch = (H + 255) / 256;
    EXL3_CHECK_ARG(a.max_blocks * (nci > nch ? nci : nch) <= kMx4Grid, "exl3_mx4_moe_forward: grid too large");
    ItemDesc* blocks = nullptr;
    int* pairs = nullptr;
    if (npairs > 0) {
        const size_t np = (size_t)npairs;
        Carve c{};
        const int rc = call_scratch("exl3_mx4_moe_forward", sh.bytes, s, st, &c);
        if (rc) return rc;
        blocks = c.take<ItemDesc>(a.max_blocks);
        pairs = c.take<int>(2 * np);
        float* pw = c.take<float>(np);
        a.blocks = blocks;
        a.pair_tok = pairs;
        a.pair_of = pairs + np;
        a.pair_w = pw;
        a.mid = c.take<uint16_t>(np * I);
        a.mexp = c.take<int8_t>(np * ((I + 127) / 128));
        a.y = c.take<float>(np * H);
        if (!a.y) return fail(EXL3_ERR_INVALID, "exl3_mx4_moe_forward: workspace carve failed");

        RouteArgs r{};
        r.ids = topk_ids;
        r.tw = topk_w;
        r.M = a.M;
        r.topk = (int)topk;
        r.slots = a.slots;
        r.E = (int)E;
        r.shared = (int)shared;
        r.MR = 0;                      // every expert's rows go into blocks
        r.items = blocks;              // (none: max_items is 0)
        r.tables = tables;
        r.use_mfma = 1;
        r.cut = mx4_cut(rows);
        r.blocks = blocks;
        r.max_blocks = a.max_blocks;
        r.pair_tok = pairs;
        r.pair_w = pw;
        r.pair_of = pairs + np;
        int rc2 = launch_align(r, st);
        if (rc2) return rc2;
        rc2 = x_dtype == EXL3_F16 ? mx4_moe_launch<kRowF16>(a, rows, st) : mx4_moe_launch<kRowBF16>(a, rows, st);
        if (rc2) return rc2;
    }
    const int64_t ncb = (H + 1023) / 1024;
    for (int64_t t = 0; t < M; t += kMx4Grid / ncb) {
        const int64_t n = M - t < kMx4Grid / ncb ? M - t : kMx4Grid / ncb;
        EXL3_LAUNCH("mx4_moe_combine", mx4_combine_kernel, dim3((unsigned)(n * ncb)), dim3(256), 0, st, a, (int)t, (int)ncb, vec);
    }
    return EXL3_OK;
}

}  // namespace exl3

extern "C" {

using namespace exl3;

int64_t exl3_mx4_moe_scratch(int64_t M, int64_t H, int64_t I, int64_t topk, int64_t E, int64_t shared) {
    if (!moe_sizes(M, H, I, topk, E) || M == 0) return 0;
    const int64_t slots = topk + (shared >= 0 ? 1 : 0);
    if (slots == 0 || M * slots > (1 << 24)) return 0;
    return (int64_t)moe_shape(M * slots, H, I, slots, E).bytes;
}

int exl3_mx4_moe_forward(const void* x, int64_t x_ld, int x_dtype, int64_t M, int64_t H, int64_t I, const int32_t* topk_ids,
                         const float* topk_w, int64_t topk, int64_t E, const int64_t* tables, int act, float act_limit,
                         int64_t shared, void* out, int64_t out_ld, int out_dtype, void* stream) {
    return mx4_moe(x, x_ld, x_dtype, M, H, I, topk_ids, topk_w, topk, E, tables, act, act_limit, shared, out, out_ld, out_dtype,
                   kLibScratch, stream);
}

int exl3_mx4_moe_forward_in(const void* x, int64_t x_ld, int x_dtype, int64_t M, int64_t H, int64_t I, const int32_t* topk_ids,
                            const float* topk_w, int64_t topk, int64_t E, const int64_t* tables, int act, float act_limit,
                            int64_t shared, void* out, int64_t out_ld, int out_dtype, void* scratch, int64_t scratch_bytes,
                            void* stream) {
    return mx4_moe(x, x_ld, x_dtype, M, H, I, topk_ids, topk_w, topk, E, tables, act, act_limit, shared, out, out_ld, out_dtype,
                   CallScratch{scratch, scratch_bytes, false}, stream);
}

}  // extern "C"
