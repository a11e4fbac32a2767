// Routed MoE layer over experts with MX4 weights. Per call, on the caller's stream:
//   align    pairs (token, slot) grouped by expert and cut into blocks of rows (exl3_moe.hip, shared with the EXL3 layer;
//            the tables' entries are (codes, scales, base) instead of (trellis, suh, svh))
//   gateup   workgroup per (block, 16 columns of I): both projections over H, act(gate, up) in fp32, rounded to x's type
//            (the down product's operand: fp32 rows would double its MFMAs; its rounding is that of the 16-bit output)
//   down     workgroup per (block, columns of H) over I: y[pair] = routing weight * sum, fp32
//   combine  out[t] = sum of the token's y rows in slot order
#include "exl3_moe.h"
#include "exl3_moe_dev.h"
#include "exl3_mx4.h"
#include "exl3_mx4_rows.h"
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
    float* y;                          // [pairs][H]
    int act;
    float limit;
    void* out;
    int64_t out_ld;
    int out_dtype;
};

// The weight row `row` (of `rows`, `k` wide) of projection p of block d: its codes, scales and base (fp16 rows only).
template <int XT>
__device__ __forceinline__ void mx4_expert_row(const ItemDesc* d, int p, int row, int rows, int k, const uint8_t*& wq,
                                               const uint8_t*& wsc, int& base) {
    const int64_t r = row < rows ? row : rows - 1;
    wq = reinterpret_cast<const uint8_t*>(d->tab[3 * p]) + r * (k / 2);
    wsc = reinterpret_cast<const uint8_t*>(d->tab[3 * p + 1]) + r * (k / 32);
    base = XT == kRowF16 ? (int)d->tab[3 * p + 2] : 0;
}

// Gate and up tiles of CT x 16 columns, blocks of up to 16 MT rows. I and H are multiples of 32, so 16 CT columns (CT 1, 2) are whole.
template <int XT, int CT, int MT, int U>
__global__ __launch_bounds__(512) void mx4_gateup_rows_kernel(Mx4MoeArgs a) {
    extern __shared__ f4_t red[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const unsigned nc = (unsigned)a.I / (16 * CT);
    const ItemDesc* d = a.blocks + blockIdx.x / nc;
    const int cnt = d->cnt, p0 = d->p0, i0 = (int)(blockIdx.x % nc) * (16 * CT), r = lane & 15;
    if (cnt == 0) return;                                      // past the call's blocks
    const uint8_t *wq[2 * CT], *wsc[2 * CT], *xq[MT], *xsc[MT];
    int base[2 * CT];
    f4_t acc[2 * CT][MT];
#pragma unroll
    for (int i = 0; i < 2 * CT; ++i) {
        mx4_expert_row<XT>(d, i & 1, i0 + 16 * (i >> 1) + r, a.I, a.H, wq[i], wsc[i], base[i]);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f4_t{};
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = 16 * j + r;
        xq[j] = a.x + (int64_t)ldg(a.pair_tok + p0 + (m < cnt ? m : cnt - 1)) * a.x_ld;
        xsc[j] = nullptr;
    }
    const int kb = a.H / 32;
    mx4_rows_loop<XT, 2 * CT, MT, U>(wq, wsc, base, xq, xsc, kb, wave, waves, (kb + 3) / 4, lane >> 4, acc);
    mx4_rows_put(red, wave, lane, acc);
    for (int t = threadIdx.x; t < CT * MT * 64; t += blockDim.x) {
        const int l = t & 63, j = (t >> 6) % MT, i = (t >> 6) / MT, m = 16 * j + (l & 15);
        if (m >= cnt) continue;
        const f4_t g = mx4_rows_sum<2 * CT, MT>(red, waves, 2 * i, j, l), u = mx4_rows_sum<2 * CT, MT>(red, waves, 2 * i + 1, j, l);
        f4_t v;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = act_mul_dev(__builtin_ldexpf(g[q], base[0]), __builtin_ldexpf(u[q], base[1]), a.act, a.limit);
        store4_as(a.mid, (int64_t)(p0 + m) * a.I + i0 + 16 * i + 4 * (l >> 4), v, XT == kRowF16 ? EXL3_F16 : EXL3_BF16);
    }
}

template <int XT, int NT, int MT, int U>
__global__ __launch_bounds__(512) void mx4_down_rows_kernel(Mx4MoeArgs a) {
    extern __shared__ f4_t red[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const unsigned nc = (unsigned)a.H / (16 * NT);
    const ItemDesc* d = a.blocks + blockIdx.x / nc;
    const int cnt = d->cnt, p0 = d->p0, h0 = (int)(blockIdx.x % nc) * (16 * NT), r = lane & 15;
    if (cnt == 0) return;
    const uint8_t *wq[NT], *wsc[NT], *xq[MT], *xsc[MT];
    int base[NT];
    f4_t acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        mx4_expert_row<XT>(d, 2, h0 + 16 * i + r, a.H, a.I, wq[i], wsc[i], base[i]);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f4_t{};
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = 16 * j + r;
        xq[j] = reinterpret_cast<const uint8_t*>(a.mid + (int64_t)(p0 + (m < cnt ? m : cnt - 1)) * a.I);
        xsc[j] = nullptr;
    }
    const int kb = a.I / 32;
    mx4_rows_loop<XT, NT, MT, U>(wq, wsc, base, xq, xsc, kb, wave, waves, (kb + 3) / 4, lane >> 4, acc);
    mx4_rows_put(red, wave, lane, acc);
    for (int t = threadIdx.x; t < NT * MT * 64; t += blockDim.x) {
        const int l = t & 63, j = (t >> 6) % MT, i = (t >> 6) / MT, m = 16 * j + (l & 15);
        if (m >= cnt) continue;
        const float w = a.pair_w[p0 + m];
        f4_t v = mx4_rows_sum<NT, MT>(red, waves, i, j, l);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = w * __builtin_ldexpf(v[q], base[0]);
        *reinterpret_cast<f4_t*>(a.y + (int64_t)(p0 + m) * a.H + h0 + 16 * i + 4 * (l >> 4)) = v;
    }
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
    p.run(t, acc);
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
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = 32 * q + 4 * (t & 7);
            const f4_t gv = *reinterpret_cast<const f4_t*>(C + (t >> 3) * kMx4CS + col);
            const f4_t uv = *reinterpret_cast<const f4_t*>(C + (t >> 3) * kMx4CS + 132 + col);
            f4_t v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = act_mul_dev(__builtin_ldexpf(gv[e], bg), __builtin_ldexpf(uv[e], bu), a.act, a.limit);
            if (m < cnt && i0 + col < a.I)
                store4_as(a.mid, (int64_t)(p0 + m) * a.I + i0 + col, v, XT == kRowF16 ? EXL3_F16 : EXL3_BF16);
        }
    }
}

template <int XT, int RG>
__global__ __launch_bounds__(256, mx4_wide_occ(RG)) void mx4_down_wide_kernel(Mx4MoeArgs a) {
    typedef Mx4Wide<XT, RG> L;
    __shared__ u32x4_t lds[L::kLds];
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
    }
    p.base = XT == kRowF16 ? (int)d->tab[8] : 0;
    p.weights(reinterpret_cast<const uint8_t*>(d->tab[6]), reinterpret_cast<const uint8_t*>(d->tab[7]), h0, a.H, lane);
    typename L::Acc acc;
    L::zero(acc);
    p.run(t, acc);
#pragma unroll
    for (int j = 0; j < RG; ++j)
        L::each(acc, j, lane, [&](int row, int n, f4_t v) {
            const int m = 32 * j + row;
            if (m >= cnt || h0 + n >= a.H) return;
            const float w = ldg(a.pair_w + p0 + m);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = w * __builtin_ldexpf(v[e], p.base);
            *reinterpret_cast<f4_t*>(a.y + (int64_t)(p0 + m) * a.H + h0 + n) = v;
        });
}

// out[t] = sum of token t's y rows in slot order, four columns per thread.
__global__ __launch_bounds__(256) void mx4_combine_kernel(Mx4MoeArgs a, int ncb, int vec) {
    const int t = blockIdx.x / (unsigned)ncb, c = 4 * ((blockIdx.x % (unsigned)ncb) * 256 + threadIdx.x);
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

typedef void (*mx4_moe_fn)(Mx4MoeArgs);

static int mx4_moe_rows(int64_t npairs, int64_t E) {
    const int e = env_int("MX4_MOE_ROWS", 0);
    if (e) return e;
    return npairs <= 16 * E ? 16 : npairs <= 48 * E ? 32 : npairs <= 96 * E ? 64 : 128;
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
    if (rows == 128) return mx4_moe_wide<XT, 4>(a, st);
    const int wg = mx4_rows_waves((a.H / 32 + 3) / 4), wd = mx4_rows_waves((a.I / 32 + 3) / 4);
    const mx4_moe_fn gu = mx4_gateup_rows_kernel<XT, 1, 1, 4>, dn = mx4_down_rows_kernel<XT, 2, 1, 4>;
    EXL3_LAUNCH("mx4_moe_gateup", gu, dim3((unsigned)(a.max_blocks * (a.I / 16))), dim3(64 * wg), (size_t)wg * 2048, st, a);
    EXL3_LAUNCH("mx4_moe_down", dn, dim3((unsigned)(a.max_blocks * (a.H / 32))), dim3(64 * wd), (size_t)wd * 2048, st, a);
    return EXL3_OK;
}

}  // namespace exl3

extern "C" {

using namespace exl3;

int exl3_mx4_moe_forward(const void* x, int64_t x_ld, int x_dtype, int64_t M, int64_t H, int64_t I, const int32_t* topk_ids,
                         const float* topk_w, int64_t topk, int64_t E, const int64_t* tables, int act, float act_limit,
                         int64_t shared, void* out, int64_t out_ld, int out_dtype, void* stream) {
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
    const int rows = mx4_moe_rows(npairs, E);
    a.max_blocks = (int)mx4_max_blocks(npairs, E, rows);
    EXL3_CHECK_ARG((int64_t)a.max_blocks * ((H > I ? H : I) / 16) <= 0x7FFFFFFF, "exl3_mx4_moe_forward: grid too large");
    ItemDesc* blocks = nullptr;
    int* pairs = nullptr;
    if (npairs > 0) {
        Workspace ws;
        const size_t np = (size_t)npairs;
        const int rc = workspace(carve_size(a.max_blocks, sizeof(ItemDesc)) + carve_size(2 * np, 4) + carve_size(np, 4) +
                                     carve_size(np * I, 2) + carve_size(np * H, 4), 0, st, &ws);
        if (rc) return rc;
        Carve c{ws.scratch, ws.scratch_bytes};
        blocks = c.take<ItemDesc>(a.max_blocks);
        pairs = c.take<int>(2 * np);
        float* pw = c.take<float>(np);
        a.blocks = blocks;
        a.pair_tok = pairs;
        a.pair_of = pairs + np;
        a.pair_w = pw;
        a.mid = c.take<uint16_t>(np * I);
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
    EXL3_CHECK_ARG(M * ncb <= 0x7FFFFFFF, "exl3_mx4_moe_forward: grid too large");
    const int vec = out_ld % 4 == 0 && aligned(out, out_dtype == EXL3_F32 ? 16 : 8);
    EXL3_LAUNCH("mx4_moe_combine", mx4_combine_kernel, dim3((unsigned)(M * ncb)), dim3(256), 0, st, a, (int)ncb, vec);
    return EXL3_OK;
}

}  // extern "C"
