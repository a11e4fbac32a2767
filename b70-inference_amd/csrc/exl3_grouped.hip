// Products grouped by expert with 16-bit weights and their gradients: entry points, and the products whose weights lie along the
// contraction.
#include "exl3_grouped_tile.h"

namespace exl3 {

int grouped_rows_along(const GroupedArgs& g, int dtype, int tile, hipStream_t st) {
    return dtype == EXL3_F16 ? launch_grouped_rows<kRowF16, false>(g, tile, st) : launch_grouped_rows<kRowBF16, false>(g, tile, st);
}

static int out_size(int t) { return t == EXL3_F32 ? 4 : 2; }
static bool out_type(int t) { return t == EXL3_F16 || t == EXL3_F32 || t == EXL3_BF16; }

constexpr int64_t kMostRows = 0x3FFFFFFF, kMostWidth = 1 << 22;

// What the products and the weights' gradient check alike.
static int grouped_setup(const char* what, int dtype, int64_t T, int64_t n, int64_t k, const int32_t* ends, int64_t E, int out_dtype) {
    EXL3_CHECK_ARG(T >= 0 && T <= kMostRows && n > 0 && n <= kMostWidth && k > 0 && k <= kMostWidth && E > 0 && E <= 65536,
                   "%s: bad sizes (%lld rows, %lld and %lld columns, %lld experts)", what, (long long)T, (long long)n, (long long)k,
                   (long long)E);
    EXL3_CHECK_ARG(dtype == EXL3_F16 || dtype == EXL3_BF16, "%s: rows and weights must be fp16 or bf16", what);
    EXL3_CHECK_ARG(out_type(out_dtype), "%s: the output must be fp16, bf16 or fp32", what);
    EXL3_CHECK_ARG(ends && aligned(ends, 4), "%s: ends must be a 4-byte aligned pointer", what);
    return EXL3_OK;
}

// Matrices of n x k behind one another, or whose rows lie between one another's.
static bool apart(int64_t E, int64_t n, int64_t k, int64_t ld, int64_t es) {
    return E == 1 || es >= (n - 1) * ld + k || (es >= k && ld >= (E - 1) * es + k);
}

static bool units16(const void* p, int64_t ld, int64_t cols) { return aligned(p, 16) && ld % 8 == 0 && cols % 8 == 0; }

// Microseconds that `tiles` tiles of `steps` steps take by an estimate from measurements: a step and the rest of a tile, with `occ`
// workgroups to a CU and with one, full rounds and what is left.
// (Of twenty products and gradients of 300 to 16384 rows over 1 to 512 experts of 512 to 7168 columns eighteen take at most a tenth more
// than with the best of the four.)
struct TileCost {
    int bm, bn, occ;
    double step, step1, rest;
};
static const TileCost kTileCost[4] = {{256, 256, 1, 1.65, 1.65, 8.0}, {128, 128, 2, 1.1, 0.65, 5.0}, {64, 128, 2, 0.65, 0.42, 4.0}, {32, 128, 2, 0.5, 0.36, 4.0}};
static double tile_time(const TileCost& t, double tiles, double steps) {
    const int64_t n = (int64_t)(tiles + 0.999), full = n / (256 * t.occ), left = n - full * 256 * t.occ;
    return (double)full * (steps * t.step + t.rest) + (left == 0 ? 0.0 : steps * (left > 256 ? t.step : t.step1) + t.rest);
}

// Tile of the products of T rows over E experts (few: the kernel of few rows is there for them).
static int rows_tile(int64_t T, int64_t E, int64_t n, int64_t k, bool few) {
    const double live = (double)(T < E ? T : E);
    int best = 0;
    double least = 1e30;
    for (int i = 0; i < 4; ++i) {
        const TileCost& t = kTileCost[i];
        double blocks = (double)T / t.bm + 0.5 * live;
        if (blocks < live) blocks = live;
        if (E == 1) blocks = (double)((T + t.bm - 1) / t.bm);
        const double us = tile_time(t, blocks * (double)((n + t.bn - 1) / t.bn), (double)((k + 63) / 64));
        if (us < least) {
            least = us;
            best = i;
        }
    }
    // Blocks of 16 rows by 16 outputs: the weights at the rate that a CU with most of them reaches, against the tiles' time or the bytes'
    // (us, few rows' kernel and the best tile: one row of 4096 -> 4096 11 and 30, 40 over 512 experts of 2048 -> 1024 28 and 35, 24
    // over 64 of 4096 -> 4096 114 and 130, 300 over 64 of 512 -> 512 10 and 7). Above 4096 inputs one workgroup fills a CU, and its
    // waves wait for each other: 8 rows over 16 experts of 7168 -> 4096 88 and 70.
    if (few && T <= 16 * E && (k <= 4096 || live * (double)(n * k) <= (double)(1 << 27))) {
        const double used = group_live(T, E), load = std::ceil((used + (double)(T / 16)) * (double)((n + 15) / 16) / 256.0),
                     bytes = 2.0 + used * (double)(n * k) * 2.0 / 5.5e6;
        if (4.0 + 0.72 * load * (double)k * 32.0 / 19.5e3 <= (least > bytes ? least : bytes)) return kTileFew;
    }
    return best;
}
// Tile of the weights' gradient, and the parts of an expert's rows: few small matrices of many rows leave CUs idle (16384 rows over 8
// experts of 512 x 512, replayed from a graph: 41 us whole and 32 in parts where a router leans towards some experts, 28 and 25 where not).
struct WeightsPlan {
    int tile, splits;
};
static int64_t n8(int64_t n) { return (n + 7) & ~(int64_t)7; }
static WeightsPlan weights_plan(int64_t T, int64_t E, int64_t n, int64_t k, bool direct) {
    WeightsPlan best = {0, 1};
    double least = 1e30;
    for (int i = direct ? 0 : 1; i < 2; ++i) {
        const TileCost& t = kTileCost[i];
        const double tiles = (double)(E * ((n + t.bm - 1) / t.bm)) * (double)((k + t.bn - 1) / t.bn);
        for (int p = 1; p <= 16; p *= 2) {
            if (p > 1 && (tiles * p > 512.0 || (double)T / (double)E < 256.0 * p)) break;
            double us = tile_time(t, tiles * p, (double)T / (double)(E * p) / 64.0 + 0.5);
            if (p > 1) us += 3.0 + (double)p * (double)(E * n) * (double)n8(k) * 1.6e-6;
            if (us < least) {
                least = us;
                best = {direct ? i == 0 ? kTile256 : kTile128 : kTileAny128, p};
            }
        }
    }
    return best;
}
static int64_t weights_part_bytes(const WeightsPlan& p, int64_t E, int64_t n, int64_t k) {
    return p.splits == 1 ? 0 : (int64_t)p.splits * E * n * n8(k) * 4;
}

static int weights_gradient(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype, int64_t T, int64_t n, int64_t k,
                            const int32_t* ends, int64_t E, void* dw, int64_t dw_ld, int64_t dw_es, int dw_dtype, int accumulate,
                            const CallScratch& s, void* stream) {
    const char* what = "exl3_grouped_mm_dw";
    const int rc = grouped_setup(what, dtype, T, n, k, ends, E, dw_dtype);
    if (rc) return rc;
    EXL3_CHECK_ARG(accumulate == 0 || accumulate == 1, "%s: accumulate %d", what, accumulate);
    EXL3_CHECK_ARG((T <= 1 || (dy_ld >= n && x_ld >= k)) && dy_ld <= kMostWidth && x_ld <= kMostWidth && (n == 1 || dw_ld >= k) &&
                       dw_ld <= ((int64_t)1 << 40) && dw_es >= 0 && dw_es <= ((int64_t)1 << 45) && apart(E, n, k, dw_ld, dw_es),
                   "%s: bad strides (gradients %lld, rows %lld, output %lld and %lld)", what, (long long)dy_ld, (long long)x_ld,
                   (long long)dw_ld, (long long)dw_es);
    EXL3_CHECK_ARG((T == 0 || (dy && x && aligned(dy, 2) && aligned(x, 2))) && dw && aligned(dw, out_size(dw_dtype)),
                   "%s: null or misaligned pointer", what);
    GroupedArgs g{};
    g.a = reinterpret_cast<const uint16_t*>(dy);
    g.b = reinterpret_cast<const uint16_t*>(x);
    g.out = dw;
    g.a_ld = T <= 1 ? n : dy_ld;
    g.b_ld = T <= 1 ? k : x_ld;
    g.out_ld = n == 1 ? k : dw_ld;
    g.out_es = dw_es;
    g.ends = ends;
    g.E = (int)E;
    g.T = (int)T;
    g.m = (int)n;
    g.n = (int)k;
    g.out_dtype = dw_dtype;
    g.accumulate = accumulate;
    const bool direct = units16(dy, g.a_ld, n) && units16(x, g.b_ld, k);
    hipStream_t st = (hipStream_t)stream;
    WeightsPlan plan = weights_plan(T, E, n, k, direct);
    const int want = env_int("EXL3MI_GROUPED_TILE", 0);
    if (direct && want > 0 && want <= 2) plan = {want - 1, 1};
    g.splits = plan.splits;
    if (plan.splits == 1) return grouped_weights(g, dtype, plan.tile, st);
    Carve c{};
    const int rs = call_scratch(what, (size_t)weights_part_bytes(plan, E, n, k), s, st, &c);
    if (rs) return rs;
    GroupedArgs h = g;                                         // the parts: fp32, padded rows
    h.out = c.p;
    h.out_ld = n8(k);
    h.out_es = n * h.out_ld;
    h.out_dtype = EXL3_F32;
    h.accumulate = 0;
    const int rc2 = grouped_weights(h, dtype, plan.tile, st);
    return rc2 ? rc2 : grouped_reduce(g, reinterpret_cast<const float*>(c.p), h.out_ld, E * h.out_es, st);
}

}  // namespace exl3

extern "C" {

using namespace exl3;

int exl3_grouped_mm(const void* x, int64_t x_ld, int dtype, int64_t T, int64_t k, const void* w, int64_t w_ld, int64_t w_es,
                    int w_layout, int64_t n, const int32_t* ends, int64_t E, void* out, int64_t out_ld, int out_dtype, int rest,
                    void* stream) {
    const char* what = "exl3_grouped_mm";
    const int rc = grouped_setup(what, dtype, T, n, k, ends, E, out_dtype);
    if (rc) return rc;
    EXL3_CHECK_ARG(w_layout == EXL3_GROUPED_W_NK || w_layout == EXL3_GROUPED_W_KN, "%s: weight layout %d", what, w_layout);
    EXL3_CHECK_ARG(rest == 0 || rest == 1, "%s: rest %d", what, rest);
    const bool across = w_layout == EXL3_GROUPED_W_KN;
    EXL3_CHECK_ARG(w_ld >= (across ? n : k) && w_ld <= kMostWidth && w_es >= 0 && (T <= 1 || (x_ld >= k && out_ld >= n)) &&
                       x_ld <= kMostWidth && out_ld <= ((int64_t)1 << 40),
                   "%s: bad strides (rows %lld, weights %lld and %lld, output %lld)", what, (long long)x_ld, (long long)w_ld,
                   (long long)w_es, (long long)out_ld);
    if (T == 0) return EXL3_OK;
    EXL3_CHECK_ARG(x && w && out && aligned(x, 2) && aligned(w, 2) && aligned(out, out_size(out_dtype)),
                   "%s: null or misaligned pointer", what);
    GroupedArgs g{};
    g.a = reinterpret_cast<const uint16_t*>(x);
    g.b = reinterpret_cast<const uint16_t*>(w);
    g.out = out;
    g.a_ld = T == 1 ? k : x_ld;
    g.b_ld = w_ld;
    g.b_es = w_es;
    g.out_ld = T == 1 ? n : out_ld;
    g.ends = ends;
    g.E = (int)E;
    g.T = (int)T;
    g.c = (int)k;
    g.n = (int)n;
    g.out_dtype = out_dtype;
    g.vec = n % 4 == 0 && g.out_ld % 4 == 0 && aligned(out, 4 * out_size(out_dtype));
    g.rest = rest;
    const bool direct = units16(x, g.a_ld, k) && units16(w, w_ld, across ? n : k) && (E == 1 || w_es % 8 == 0);
    // Tiles of operands that go through registers: 32 rows, or 128 where an expert has more than 48 on average (us, 32 and 128 rows: 40
    // rows for each of 64 experts of 2049 -> 2048 176 and 186, 64 rows 215 and 194; of 4097 -> 4096 639 and 571, 804 and 616; for
    // each of 16 experts 184 and 207, 240 and 223, of 1025 -> 513 20 and 28, 20 and 29). By rows alone, so not the faster one everywhere:
    // 256 rows of one matrix of 4097 -> 4096 60 and 85.
    const int64_t mean = T / E;
    int tile = !direct ? (mean <= 48 ? kTileAny32 : kTileAny128) : rows_tile(T, E, n, k, !across && k <= 8192);
    const int want = env_int("EXL3MI_GROUPED_TILE", 0);
    if (direct && want > 0 && want <= 4) tile = want - 1;
    if (direct && want == 5 && !across && k <= 8192) tile = kTileFew;
    if (tile == kTileFew) return grouped_rows_few(g, dtype, (hipStream_t)stream);
    return (across ? grouped_rows_across : grouped_rows_along)(g, dtype, tile, (hipStream_t)stream);
}

// The plan does not know how the operands lie: the larger of both plans' scratch.
int64_t exl3_grouped_mm_dw_scratch(int64_t T, int64_t n, int64_t k, int64_t E) {
    if (T < 0 || T > kMostRows || n <= 0 || n > kMostWidth || k <= 0 || k > kMostWidth || E <= 0 || E > 65536) return 0;
    const int64_t a = weights_part_bytes(weights_plan(T, E, n, k, true), E, n, k), b = weights_part_bytes(weights_plan(T, E, n, k, false), E, n, k);
    return a > b ? a : b;
}

int exl3_grouped_mm_dw(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype, int64_t T, int64_t n, int64_t k,
                       const int32_t* ends, int64_t E, void* dw, int64_t dw_ld, int64_t dw_es, int dw_dtype, int accumulate,
                       void* stream) {
    return weights_gradient(dy, dy_ld, x, x_ld, dtype, T, n, k, ends, E, dw, dw_ld, dw_es, dw_dtype, accumulate, kLibScratch, stream);
}

int exl3_grouped_mm_dw_in(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype, int64_t T, int64_t n, int64_t k,
                          const int32_t* ends, int64_t E, void* dw, int64_t dw_ld, int64_t dw_es, int dw_dtype, int accumulate,
                          void* scratch, int64_t scratch_bytes, void* stream) {
    return weights_gradient(dy, dy_ld, x, x_ld, dtype, T, n, k, ends, E, dw, dw_ld, dw_es, dw_dtype, accumulate,
                            CallScratch{scratch, scratch_bytes, false}, stream);
}

}  // extern "C"
