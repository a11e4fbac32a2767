// Products with 4-bit weights and group scales: entry points, the choice of kernel, and matrices of fewer than four scales.
#include "exl3_g4.h"

namespace exl3 {

// One output per thread: tensors of fewer than four scales, which the other kernels' loads of scales do not fit.
template <int XT>
__global__ __launch_bounds__(256) void g4_tiny_kernel(G4Args g, int group) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / g.n, n = i - m * g.n;
    if (m >= g.T) return;
    int e = 0;
    if (g.ends)
        while (e < g.E && group_end(g.ends, e, g.T) <= m) ++e;
    if (e == g.E) {
        if (g.rest) store_as(g.out, m * g.out_ld + n, 0.f, g.out_dtype);
        return;
    }
    const int64_t row = (int64_t)e * g.n + n;
    float sum = 0.f;
    for (int G = 0; G < g.groups; ++G) {
        const int z = g.zeros ? ldg(g.zeros + row * g.groups + G) & 15 : 8;
        float part = 0.f;
        for (int k = G * group; k < (G + 1) * group; ++k) {
            const uint16_t v = ldg(g.x + m * g.x_ld + k);
            part += (XT == kRowF16 ? h2f(v) : bf2f(v)) * (float)((ldg(g.codes + row * (g.k / 2) + k / 2) >> (4 * (k & 1)) & 15) - z);
        }
        sum += g4_scale(ldg(g.scales + row * g.groups + G), g.scale_bf16) * part;
    }
    store_as(g.out, m * g.out_ld + n, sum + (g.bias ? ldg(g.bias + n) : 0.f), g.out_dtype);
}

// The splits' sums in order, the bias, one rounding: four neighbours per thread, four rows of a tile per workgroup.
__global__ __launch_bounds__(256) void g4_reduce_kernel(G4Args g, int bm) {
    const unsigned nnt = (unsigned)((g.n + 255) / 256), all = g.slots * nnt, tail = all - g.whole, groups = (g.part_rows + 3) / 4,
                   at = blockIdx.x / groups, r = (blockIdx.x - at * groups) * 4 + threadIdx.x / 64;
    unsigned mt, nt;
    grouped_tile(g.whole + at, (unsigned)g.slots, nnt, mt, nt);
    const int64_t m = (int64_t)mt * bm + r, n = (int64_t)nt * 256 + 4 * (threadIdx.x & 63);
    if ((int)r >= g.part_rows || m >= g.T || n >= g.n) return;
    const int64_t stride = (int64_t)tail * g.part_rows * 256;
    const float* p = g.part + ((int64_t)at * g.part_rows + r) * 256 + 4 * (threadIdx.x & 63);
    f4_t v = {};
    for (int s0 = 0; s0 < g.splits; s0 += 4) {
        f4_t t[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) t[s] = ldg(reinterpret_cast<const f4_t*>(p + (s0 + s < g.splits ? s0 + s : s0) * stride));
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s0 + s < g.splits)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += t[s][e];
    }
    g4_store4(g, m, n, v);
}

// Kernel and splits of a call: the least time by an estimate from measurements (1 to 512 rows of nine shapes from 640 -> 2560 to
// 8192 -> 8192 and 5376 -> 21504), in microseconds for 256 CUs. Six rows of 8192 -> 8192, fp16: 16 with the kernel of few rows, 18
// with the other; of 5376 -> 21504 21 and 22, in groups of 32 21 and 27; 24 rows of it 36 and 25; of 4096 -> 4096 13 and 17. Splits are the linear's alone: experts have workgroups enough, or few
// rows, and rows of no expert have no sums.
struct G4Plan {
    int tile;
    int64_t whole, splits, spc;
};
static int64_t g4_rows(int tile) { return 16 << tile; }
static int64_t g4_tiles(int tile, int64_t m, int64_t n) { return (m + g4_rows(tile) - 1) / g4_rows(tile) * ((n + 255) / 256); }
static G4Plan g4_plan(int64_t m, int64_t n, int64_t k, int64_t group, int64_t E, bool split) {
    const int64_t steps = (k + 127) / 128;
    G4Plan best = {0, 0, 1, steps};
    double least = 1e30;
    // blocks of 16 rows: the groups of 512 inputs of all tiles, spread over the CUs
    const int64_t live = E == 1 ? (m + 15) / 16 : m / 16 + (m < E ? m : E);
    if (k <= 8192 && (E == 1 || m <= 16 * E))
        least = 6.5 + (double)(live * ((n + 15) / 16) * ((k + 511) / 512)) / 256.0 * (0.245 + 0.003 * (double)(m < 16 ? m : 16));
    if (least <= 8.0 + 1.35 * (double)((steps + 15) / 16) && least <= 5.0 + 1.35 * (double)steps) return best;   // none below is less
    // blocks of 32, 64, 128 rows: time of a step with one, two, three workgroups to a CU; all tiles in splits, or full rounds of whole
    // tiles and the rest in splits (1021 rows of 5376 -> 21504, 672 tiles for 512 places: 250 us whole, 223 with the last 160 in three)
    static const double kStep[3][4] = {{1.45, 2.05, 2.85, 3.7}, {1.65, 2.6, 4.2}, {2.6, 3.9}};
    const bool more = !split && group >= 128;                  // experts: a workgroup more to a CU
    const int kOcc[3] = {more ? 4 : 3, more ? 3 : 2, 2};
    const double scales = group >= 128 ? 0.95 : group == 64 ? 1.05 : 1.25;
    for (int t = 0; t < 3; ++t) {
        const int64_t bm = 32 << t, room = 256 * kOcc[t], blocks = E == 1 ? (m + bm - 1) / bm : m / bm + (m < E ? m : E),
                      tiles = blocks * ((n + 255) / 256), rounds = tiles / room;
        const auto time = [&](int64_t wgs, int64_t spc) {
            const int64_t full = wgs / room, left = wgs - full * room;
            return (double)full * (3.0 + scales * (double)spc * kStep[t][kOcc[t] - 1]) +
                   (left ? 3.0 + scales * (double)spc * kStep[t][(left + 255) / 256 - 1] : 0.0);
        };
        for (int tail = 0; tail < (split && rounds ? 2 : 1); ++tail) {
            const int64_t whole = tail ? rounds * room : 0, rest = tiles - whole;
            if (rest == 0) break;
            for (int64_t p = tail ? 2 : 1; p <= (!split ? 1 : steps < 16 ? steps : 16); ++p) {
                const int64_t spc = (steps + p - 1) / p;
                if ((steps + spc - 1) / spc != p) continue;
                double us = 2.0 + time(whole, steps) + time(rest * p, spc);
                if (p > 1) us += 3.0 + (tail ? (double)(p * rest * bm * 256) : (double)(p * m * n)) * 1.2e-6;
                if (us < least) {
                    least = us;
                    best = {t + 1, whole, p, spc};
                }
            }
        }
    }
    return best;
}
static int64_t g4_part_rows(const G4Plan& p, int64_t m) { return m < g4_rows(p.tile) ? m : g4_rows(p.tile); }
static int64_t g4_part_bytes(const G4Plan& p, int64_t m, int64_t n) {
    return p.splits == 1 ? 0 : p.splits * (g4_tiles(p.tile, m, n) - p.whole) * g4_part_rows(p, m) * 1024;
}

static int out_size(int t) { return t == EXL3_F32 ? 4 : 2; }

static int g4_product(const char* what, const void* x, int64_t x_ld, int dtype, int64_t m, int64_t k, const uint8_t* codes,
                      const void* scales, int scale_dtype, const uint8_t* zeros, int64_t group, int64_t n, const int32_t* ends,
                      int64_t E, const float* bias, void* out, int64_t out_ld, int out_dtype, int rest, const CallScratch& s,
                      void* stream) {
    EXL3_CHECK_ARG(m >= 0 && m <= 0x3FFFFFFF && n > 0 && n <= 0x3FFFFFFF && E > 0 && E <= 65536 && k > 0 && k <= (1 << 22) &&
                       k % 32 == 0 && n * E <= ((int64_t)1 << 42) / k,
                   "%s: bad sizes (%lld rows, %lld outputs, %lld inputs, %lld matrices; inputs a multiple of 32)", what,
                   (long long)m, (long long)n, (long long)k, (long long)E);
    EXL3_CHECK_ARG(dtype == EXL3_F16 || dtype == EXL3_BF16, "%s: rows must be fp16 or bf16", what);
    EXL3_CHECK_ARG(scale_dtype == EXL3_F16 || scale_dtype == EXL3_BF16, "%s: scales must be fp16 or bf16", what);
    EXL3_CHECK_ARG(out_dtype == EXL3_F16 || out_dtype == EXL3_F32 || out_dtype == EXL3_BF16, "%s: the output must be fp16, bf16 or "
                   "fp32", what);
    if (group != 32 && group != 64 && (group <= 0 || group % 128))
        return fail(EXL3_ERR_UNSUPPORTED, "%s: groups of %lld (32, 64 and multiples of 128)", what, (long long)group);
    EXL3_CHECK_ARG(k % group == 0, "%s: %lld inputs are not whole groups of %lld", what, (long long)k, (long long)group);
    EXL3_CHECK_ARG(m <= 1 || (x_ld >= k && x_ld <= (1 << 22) && out_ld >= n && out_ld <= ((int64_t)1 << 40)),
                   "%s: bad strides (rows %lld, output %lld)", what, (long long)x_ld, (long long)out_ld);
    if (m == 0) return EXL3_OK;
    EXL3_CHECK_ARG(x && codes && scales && out, "%s: null pointer", what);
    EXL3_CHECK_ARG(aligned(x, 16) && (m == 1 || x_ld % 8 == 0) && aligned(codes, 16), "%s: rows and codes must be 16-byte aligned", what);
    EXL3_CHECK_ARG(aligned(scales, 2) && aligned(out, out_size(out_dtype)) && (!bias || aligned(bias, 4)) && (!ends || aligned(ends, 4)),
                   "%s: misaligned pointer", what);
    G4Args g{};
    g.x = reinterpret_cast<const uint16_t*>(x);
    g.x_ld = m == 1 ? k : x_ld;
    g.codes = codes;
    g.scales = reinterpret_cast<const uint16_t*>(scales);
    g.zeros = zeros;
    g.bias = bias;
    g.out = out;
    g.out_ld = m == 1 ? n : out_ld;
    g.ends = ends;
    g.E = (int)E;
    g.T = (int)m;
    g.k = (int)k;
    g.n = (int)n;
    g.groups = (int)(k / group);
    g.per = group > 128 ? (int)(group / 128) : 1;
    g.scale_bf16 = scale_dtype == EXL3_BF16;
    g.out_dtype = out_dtype;
    g.vec = n % 4 == 0 && g.out_ld % 4 == 0 && aligned(out, 4 * out_size(out_dtype));
    g.rest = rest;
    hipStream_t st = (hipStream_t)stream;
    if (E * n * g.groups < 4) {
        EXL3_CHECK_ARG(m <= kMx4Grid * 256 / n, "%s: grid too large", what);
        const dim3 grid((unsigned)((m * n + 255) / 256));
        if (dtype == EXL3_F16) EXL3_LAUNCH("g4_tiny", g4_tiny_kernel<kRowF16>, grid, dim3(256), 0, st, g, (int)group);
        else EXL3_LAUNCH("g4_tiny", g4_tiny_kernel<kRowBF16>, grid, dim3(256), 0, st, g, (int)group);
        return EXL3_OK;
    }
    G4Plan plan = g4_plan(m, n, k, group, E, !ends);
    const int want = env_int("EXL3MI_G4_TILE", 0);
    if (want > (k <= 8192 ? 0 : 1) && want <= 4) plan = {want - 1, 0, 1, (k + 127) / 128};
    g.whole = (int)plan.whole;
    g.splits = (int)plan.splits;
    g.spc = (int)plan.spc;
    g.part_rows = (int)g4_part_rows(plan, m);
    if (plan.splits > 1) {
        Carve c{};
        const int rc = call_scratch(what, (size_t)g4_part_bytes(plan, m, n), s, st, &c);
        if (rc) return rc;
        g.part = reinterpret_cast<float*>(c.p);
    }
    const int rc = dtype == EXL3_F16 ? g4_run_f16(g, (int)group, plan.tile, st) : g4_run_bf16(g, (int)group, plan.tile, st);
    if (rc || plan.splits == 1) return rc;
    g.slots = (int)((m + g4_rows(plan.tile) - 1) / g4_rows(plan.tile));
    const int64_t wgs = (g4_tiles(plan.tile, m, n) - plan.whole) * ((g.part_rows + 3) / 4);
    EXL3_CHECK_ARG(wgs <= kMx4Grid, "%s: grid too large", what);
    EXL3_LAUNCH("g4_reduce", g4_reduce_kernel, dim3((unsigned)wgs), dim3(256), 0, st, g, (int)g4_rows(plan.tile));
    return EXL3_OK;
}

}  // namespace exl3

extern "C" {

using namespace exl3;

int64_t exl3_g4_linear_scratch(int64_t m, int64_t k, int64_t n, int64_t group) {
    if (m <= 0 || m > 0x3FFFFFFF || n <= 0 || n > 0x3FFFFFFF || k <= 0 || k > (1 << 22) || group <= 0 || n * (k / group) < 4) return 0;
    return g4_part_bytes(g4_plan(m, n, k, group, 1, true), m, n);
}

int exl3_g4_linear(const void* x, int64_t x_ld, int x_dtype, int64_t m, int64_t k, const uint8_t* codes, const void* scales,
                   int scale_dtype, const uint8_t* zeros, int64_t group, int64_t n, const float* bias, void* C, int64_t c_ld,
                   int c_dtype, void* stream) {
    return g4_product("exl3_g4_linear", x, x_ld, x_dtype, m, k, codes, scales, scale_dtype, zeros, group, n, nullptr, 1, bias, C, c_ld,
                      c_dtype, 0, kLibScratch, stream);
}

int exl3_g4_linear_in(const void* x, int64_t x_ld, int x_dtype, int64_t m, int64_t k, const uint8_t* codes, const void* scales,
                      int scale_dtype, const uint8_t* zeros, int64_t group, int64_t n, const float* bias, void* C, int64_t c_ld,
                      int c_dtype, void* scratch, int64_t scratch_bytes, void* stream) {
    return g4_product("exl3_g4_linear", x, x_ld, x_dtype, m, k, codes, scales, scale_dtype, zeros, group, n, nullptr, 1, bias, C, c_ld,
                      c_dtype, 0, CallScratch{scratch, scratch_bytes, false}, stream);
}

int exl3_grouped_g4(const void* x, int64_t x_ld, int x_dtype, int64_t T, int64_t k, const uint8_t* codes, const void* scales,
                    int scale_dtype, const uint8_t* zeros, int64_t group, int64_t n, const int32_t* ends, int64_t E, void* out,
                    int64_t out_ld, int out_dtype, int rest, void* stream) {
    EXL3_CHECK_ARG(ends, "exl3_grouped_g4: null pointer");
    EXL3_CHECK_ARG(rest == 0 || rest == 1, "exl3_grouped_g4: rest %d", rest);
    return g4_product("exl3_grouped_g4", x, x_ld, x_dtype, T, k, codes, scales, scale_dtype, zeros, group, n, ends, E, nullptr, out,
                      out_ld, out_dtype, rest, kLibScratch, stream);
}

}  // extern "C"
