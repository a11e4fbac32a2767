// MX4 (microscaled 4-bit) quantisation, its inverse, and the dense products with MX4 weights: 16-bit rows (exl3_mx4_linear)
// and MX4 rows (exl3_mx4_gemm).
#include "exl3_mx4.h"
#include "exl3_mx4_decode.h"
#include "exl3_mx4_plan.h"
#include "exl3_mx4_wide.h"

namespace exl3 {

// ================================================================================================ quantise
// A block's scale is 2^(floor(log2 a) - 2), a its largest magnitude, so that a / scale lies in [4, 8) and the largest
// code, 6, is within a factor 4/3 of it: the byte is a's float exponent less 2, at least 0 (subnormal a, and 0). A block
// with an infinity or a NaN (exponent 255) has byte 255 and codes 0. Four lanes share a block, eight values each; integer maxima
// of the magnitude bits order floats, infinities and NaNs alike. Bound by the bytes: 2039 rows of 5376 fp16 values 6.3 us, back
// 5.7 us (27.7 MB: 4.4 and 4.9 TB/s, a large copy 5.1).
template <int DT>
struct QuantIn;
template <>
struct QuantIn<EXL3_F16> {
    u32x4_t v;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        v = ldg(reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(p) + i));
    }
    __device__ __forceinline__ uint32_t top() const {          // float bits of the largest magnitude
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, max(v[j] & 0x7FFFu, v[j] >> 16 & 0x7FFFu));
        return __builtin_bit_cast(uint32_t, h2f((uint16_t)m));
    }
    __device__ __forceinline__ uint32_t codes(float s) const {
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, (uint32_t)v[0]), s, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, (uint32_t)v[1]), s, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, (uint32_t)v[2]), s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, (uint32_t)v[3]), s, 3);
    }
};
template <>
struct QuantIn<EXL3_BF16> {
    u32x4_t v;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        v = ldg(reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(p) + i));
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, max(v[j] & 0x7FFFu, v[j] >> 16 & 0x7FFFu));
        return m << 16;
    }
    __device__ __forceinline__ uint32_t codes(float s) const {
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, (uint32_t)v[0]), s, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, (uint32_t)v[1]), s, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, (uint32_t)v[2]), s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, (uint32_t)v[3]), s, 3);
    }
};
template <>
struct QuantIn<EXL3_F32> {
    f4_t a, b;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        const f4_t* q = reinterpret_cast<const f4_t*>(reinterpret_cast<const float*>(p) + i);
        a = ldg(q);
        b = ldg(q + 1);
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            m = max(m, max(__builtin_bit_cast(uint32_t, (float)a[j]) & 0x7FFFFFFFu,
                           __builtin_bit_cast(uint32_t, (float)b[j]) & 0x7FFFFFFFu));
        return m;
    }
    __device__ __forceinline__ uint32_t codes(float s) const {
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, a[0], a[1], s, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, a[2], a[3], s, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, b[0], b[1], s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, b[2], b[3], s, 3);
    }
};

// Units of eight values per thread: enough loads in flight to cover the memory's latency.
constexpr int kQuantUnits = 2;

// `upr`: units of eight values per row (a multiple of 4: a block never straddles waves), `cpr` workgroups per row.
template <int DT>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const void* __restrict__ x, int64_t x_ld, int64_t upr, int cpr,
                                                           uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int64_t row = blockIdx.x / (unsigned)cpr, u0 = (int64_t)(blockIdx.x % (unsigned)cpr) * (256 * kQuantUnits);
    QuantIn<DT> in[kQuantUnits];
#pragma unroll
    for (int i = 0; i < kQuantUnits; ++i) {
        const int64_t u = u0 + 256 * i + threadIdx.x;
        in[i].load(x, row * x_ld + 8 * (u < upr ? u : upr - 1));
    }
#pragma unroll
    for (int i = 0; i < kQuantUnits; ++i) {
        const int64_t u = u0 + 256 * i + threadIdx.x;
        uint32_t top = in[i].top();
        top = max(top, (uint32_t)__shfl_xor((int)top, 1));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2));
        const int ex = (int)(top >> 23), e = ex == 255 ? 255 : ex > 2 ? ex - 2 : 0;
        const uint32_t q = in[i].codes(__builtin_bit_cast(float, (e == 255 ? 127 : e) << 23));
        if (u < upr) {
            codes[row * upr + u] = e == 255 ? 0u : q;
            if ((u & 3) == 0) scales[(row * upr + u) >> 2] = (uint8_t)e;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, int64_t upr, int cpr,
                                                             void* __restrict__ out, int64_t out_ld) {
    const int64_t row = blockIdx.x / (unsigned)cpr, u0 = (int64_t)(blockIdx.x % (unsigned)cpr) * (256 * kQuantUnits);
    uint32_t q[kQuantUnits];
    int s[kQuantUnits];
#pragma unroll
    for (int i = 0; i < kQuantUnits; ++i) {
        const int64_t u = u0 + 256 * i + threadIdx.x, at = row * upr + (u < upr ? u : upr - 1);
        q[i] = ldg(codes + at);
        s[i] = ldg(scales + (at >> 2));
    }
#pragma unroll
    for (int i = 0; i < kQuantUnits; ++i) {
        const int64_t u = u0 + 256 * i + threadIdx.x;
        if (u >= upr) break;
        const float sc = mx4_scale(s[i], 0);
        if constexpr (DT == EXL3_F32) {
            float* o = reinterpret_cast<float*>(out) + row * out_ld + 8 * u;
            const auto v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], sc, 0),
                       v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], sc, 1),
                       v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], sc, 2),
                       v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], sc, 3);
            reinterpret_cast<f4_t*>(o)[0] = f4_t{v0[0], v0[1], v1[0], v1[1]};
            reinterpret_cast<f4_t*>(o)[1] = f4_t{v2[0], v2[1], v3[0], v3[1]};
        } else {
            *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(out) + row * out_ld + 8 * u) =
                mx4_frag<DT == EXL3_F16 ? kRowF16 : kRowBF16>(q[i], sc);
        }
    }
}

// Units and workgroups of a row, and the rows of a launch. Rows without gaps are one, as long as a launch can hold it.
struct QuantGrid {
    int64_t rows, upr, cpr, most;
};
static bool quant_grid(int64_t rows, int64_t k, int64_t ld, QuantGrid& g) {
    constexpr int64_t kWg = 256 * kQuantUnits;
    if (ld == k && (rows * (k / 8) + kWg - 1) / kWg <= kMx4Grid) {
        k *= rows;
        rows = 1;
    }
    g.rows = rows;
    g.upr = k / 8;
    g.cpr = (g.upr + kWg - 1) / kWg;
    if (g.cpr > kMx4Grid) return false;
    g.most = kMx4Grid / g.cpr;
    return true;
}

// ================================================================================================ dense products
struct Mx4Args {
    const uint8_t* x;                  // rows: 16-bit values, or MX4 codes
    const uint8_t* xs;                 // MX4 rows: scales
    int64_t x_ld;                      // bytes from row to row
    const uint8_t* w;
    const uint8_t* ws;
    const float* bias;                 // [n] or null
    void* out;
    int64_t out_ld;
    int64_t m, n;
    int k, base, out_dtype, vec;       // vec: four neighbouring outputs may be stored together; 2: eight 16-bit ones
    // k split over workgroups: `splits` of `bps` steps of 128 k each, their sums in part [splits][m][n4]
    float* part;
    int splits, bps;
    int64_t n4;                        // n rounded up to 4
};

// A dense output's four neighbours n, n + 1, ... of row m: 2^base of the sum, the bias, one rounding.
__device__ __forceinline__ void mx4_store(const Mx4Args& a, int64_t m, int64_t n, f4_t v) {
    if (m >= a.m) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (a.base) v[q] = __builtin_ldexpf(v[q], a.base);
        if (a.bias && n + q < a.n) v[q] += ldg(a.bias + n + q);
    }
    if (a.vec) {
        if (n < a.n) store4_as(a.out, m * a.out_ld + n, v, a.out_dtype);
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (n + q < a.n) store_as(a.out, m * a.out_ld + n + q, v[q], a.out_dtype);
}

// Four neighbouring sums of row m of split `sp`.
__device__ __forceinline__ void mx4_put(const Mx4Args& a, int sp, int64_t m, int64_t n, f4_t v) {
    if (!a.part) {
        mx4_store(a, m, n, v);
    } else if (m < a.m && n < a.n4) {
        *reinterpret_cast<f4_t*>(a.part + ((int64_t)sp * a.m + m) * a.n4 + n) = v;
    }
}

// Outputs of a 32 x 32 product: of row m, sixteen from n on; lane group g (lane >> 5) holds those at 4 g in v and at 8 + 4 g in w.
// 16-bit outputs change hands between the groups, so that a lane stores eight neighbours (16 bytes) instead of twice four: the
// stores of 16-byte pieces of 32 rows bound the epilogue.
__device__ __forceinline__ void mx4_put16(const Mx4Args& a, int sp, int64_t m, int64_t n, int g, f4_t v, f4_t w) {
    if (a.part || a.vec != 2) {                                // uniform
        mx4_put(a, sp, m, n + 4 * g, v);
        mx4_put(a, sp, m, n + 8 + 4 * g, w);
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (a.base) {
            v[q] = __builtin_ldexpf(v[q], a.base);
            w[q] = __builtin_ldexpf(w[q], a.base);
        }
        if (a.bias) {
            v[q] += ldg(a.bias + (n + 4 * g + q < a.n ? n + 4 * g + q : 0));
            w[q] += ldg(a.bias + (n + 8 + 4 * g + q < a.n ? n + 8 + 4 * g + q : 0));
        }
    }
    uint32_t p[2], r[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        if (a.out_dtype == EXL3_F16) {                         // uniform
            p[q] = __builtin_bit_cast(uint32_t, h2_t{(_Float16)v[2 * q], (_Float16)v[2 * q + 1]});
            r[q] = __builtin_bit_cast(uint32_t, h2_t{(_Float16)w[2 * q], (_Float16)w[2 * q + 1]});
        } else {
            p[q] = __builtin_bit_cast(uint32_t, b2_t{(__bf16)v[2 * q], (__bf16)v[2 * q + 1]});
            r[q] = __builtin_bit_cast(uint32_t, b2_t{(__bf16)w[2 * q], (__bf16)w[2 * q + 1]});
        }
        const auto x = __builtin_amdgcn_permlane32_swap(p[q], r[q], false, false);
        p[q] = x[0];
        r[q] = x[1];
    }
    if (m < a.m && n + 8 * g < a.n)
        *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(a.out) + m * a.out_ld + n + 8 * g) = u32x4_t{p[0], p[1], r[0], r[1]};
}

// The splits' sums in order, 2^base, the bias, one rounding.
__global__ __launch_bounds__(256) void mx4_reduce_kernel(Mx4Args a) {
    const int64_t q4 = a.n4 / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / q4, n = 4 * (i - m * q4);
    if (m >= a.m) return;
    const float* p = a.part + m * a.n4 + n;
    f4_t v = {};
    for (int s0 = 0; s0 < a.splits; s0 += 4) {
        f4_t t[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
            t[s] = ldg(reinterpret_cast<const f4_t*>(p + (int64_t)(s0 + s < a.splits ? s0 + s : s0) * a.m * a.n4));
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s0 + s < a.splits)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += t[s][e];
    }
    mx4_store(a, m, n, v);
}

static int64_t mx4_n4(int64_t n) { return (n + 3) & ~(int64_t)3; }

// Bytes of a plan's partials.
static int64_t mx4_part_bytes(const Mx4Plan& plan, int64_t m, int64_t n) {
    return plan.P == 1 ? 0 : (int64_t)plan.P * m * mx4_n4(n) * 4;
}

// The plan's splits, with the partials in the call's scratch. One split: the kernel writes the output itself.
static int mx4_split(const char* what, Mx4Args& a, const Mx4Plan& plan, const CallScratch& s, hipStream_t st) {
    a.splits = plan.P;
    a.bps = plan.bps;
    a.n4 = mx4_n4(a.n);
    a.part = nullptr;
    if (a.splits == 1) return EXL3_OK;
    Carve c{};
    const int rc = call_scratch(what, (size_t)mx4_part_bytes(plan, a.m, a.n), s, st, &c);
    a.part = reinterpret_cast<float*>(c.p);
    return rc;
}

static int launch_reduce(const Mx4Args& a, hipStream_t st) {
    if (a.splits == 1) return EXL3_OK;
    const int64_t wgs = (a.m * (a.n4 / 4) + 255) / 256;
    EXL3_CHECK_ARG(wgs <= kMx4Grid, "mx4: grid too large");
    EXL3_LAUNCH("mx4_reduce", mx4_reduce_kernel, dim3((unsigned)wgs), dim3(256), 0, st, a);
    return EXL3_OK;
}

// One output per thread: matrices of fewer than 16 scale bytes, which the other kernels' 16-byte loads of scales do not fit. A block's
// sum is of plain codes, times both scales at once: one of them alone may leave fp32 where the product does not.
template <int XT>
__global__ __launch_bounds__(256) void mx4_tiny_kernel(Mx4Args a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / a.n, n = i - m * a.n;
    if (m >= a.m) return;
    const int kb = a.k / 32;
    float sum = 0.f;
    for (int b = 0; b < kb; ++b) {
        const int ws = a.ws[n * kb + b], xs = XT == kRowMX4 ? a.xs[m * kb + b] : 127;
        float part = 0.f;
        for (int e = 0; e < 16; ++e) {
            const auto w = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a.w[n * (a.k / 2) + 16 * b + e], 1.f, 0);
            float x0, x1;
            if constexpr (XT == kRowMX4) {
                const auto x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a.x[m * a.x_ld + 16 * b + e], 1.f, 0);
                x0 = x[0];
                x1 = x[1];
            } else {
                const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x + m * a.x_ld) + 32 * b + 2 * e;
                x0 = XT == kRowF16 ? h2f(x[0]) : bf2f(x[0]);
                x1 = XT == kRowF16 ? h2f(x[1]) : bf2f(x[1]);
            }
            part += x0 * w[0] + x1 * w[1];
        }
        sum += ws == 255 || xs == 255 ? __builtin_nanf("") : __builtin_ldexpf(part, ws + xs - 254 - a.base);
    }
    if (a.base) sum = __builtin_ldexpf(sum, a.base);
    if (a.bias) sum += ldg(a.bias + n);
    store_as(a.out, m * a.out_ld + n, sum, a.out_dtype);
}

template <int XT>
static int launch_tiny(const char* name, const Mx4Args& a, hipStream_t st) {
    EXL3_CHECK_ARG(a.m <= kMx4Grid * 256 / a.n, "%s: grid too large", name);
    EXL3_LAUNCH(name, mx4_tiny_kernel<XT>, dim3((unsigned)((a.m * a.n + 255) / 256)), dim3(256), 0, st, a);
    return EXL3_OK;
}

// Up to 16 rows, x in LDS. A workgroup takes every gridDim-th tile of 16 outputs, so x is staged once per resident workgroup.
// Six rows of 5376 -> 21504 17.5 us among eager calls, 18.4 as a graph's node (62 MB: 3.5 and 3.4 TB/s; the same with 6, 8 or 10
// waves), one of 4096 -> 4096 4.8 as a graph's node (a chain of the first load, the sum and the store).
template <int XT>
__global__ __launch_bounds__(1024) void mx4_decode_kernel(Mx4Args a, int xbytes) {
    extern __shared__ f4_t red[];
    char* lds = reinterpret_cast<char*>(red);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int rows = (int)a.m, kb = a.k / 32, ng = (kb + 4 * kMx4Group - 1) / (4 * kMx4Group);
    const unsigned tiles = (unsigned)((a.n + 15) / 16);
    Mx4Decode<XT> p;
    p.kb = kb;
    p.tile.set(a.w, a.ws, (int64_t)blockIdx.x * 16, a.n, kb, lane);
    typename Mx4Decode<XT>::Group q, nx;
    p.load(wave, lane, q);
    const Mx4X x = mx4_stage_x<XT>(lds, rows, kb, [&](int i) { return a.x + i * a.x_ld; }, [&](int i) { return a.xs + (int64_t)i * kb; });
    __syncthreads();
    f4_t* const out = reinterpret_cast<f4_t*>(lds + xbytes);
    unsigned tile = blockIdx.x;
    for (int buf = 0;; buf ^= 1) {                             // (waves <= ng: every wave has a group of every tile)
        f4_t acc = {};
        const unsigned next = tile + gridDim.x;
        for (int gi = wave; gi < ng; gi += waves) {
            const bool last = gi + waves >= ng;                // (uniform) then on to the next tile
            if (!last) {
                p.load(gi + waves, lane, nx);
            } else if (next < tiles) {
                p.tile.set(a.w, a.ws, (int64_t)next * 16, a.n, kb, lane);
                p.load(wave, lane, nx);
            }
            p.mul(gi, lane, x, rows, a.base, q, acc);
            q = nx;
        }
        f4_t* o = out + buf * waves * 64;                      // two, so that one barrier a tile is enough
        o[wave * 64 + lane] = acc;
        __syncthreads();
        if (wave == 0) mx4_store(a, lane & 15, (int64_t)tile * 16 + 4 * (lane >> 4), mx4_decode_sum(o, waves, 0, lane));
        if (next >= tiles) break;
        tile = next;
    }
}

// LDS of a CU, all of which one workgroup may take.
constexpr int kMx4Lds = 163840;

// Rows that the decode kernel takes: up to 16 with 16-bit rows, with MX4 rows up to eight (16 rows, decode / tiles: 4096 x 4096 10.2 /
// 9.9 us, 5376 -> 21504 23.0 / 19.8; 4 rows: 6.0 / 9.0, 16.5 / 19.0). Waves and LDS bytes of a call: eight waves, sixteen where x leaves room for one workgroup per CU only (eight rows of
// 5376 -> 21504: 25.1 us with eight, 21.4 with sixteen). False if x does not fit.
template <int XT>
static bool decode_shape(int64_t m, int64_t k, int& waves, int& xb, int& lds) {
    if (m > (XT == kRowMX4 ? 8 : 16) || k > 1 << 20) return false;
    const int kb = (int)k / 32, ng = (kb + 4 * kMx4Group - 1) / (4 * kMx4Group);
    xb = mx4_x_bytes<XT>((int)m, kb);
    waves = mx4_decode_waves(ng, 8);
    if (2 * (xb + 2 * waves * 1024) > kMx4Lds && xb + 2 * 16 * 1024 <= kMx4Lds) waves = mx4_decode_waves(ng, 16);
    lds = xb + 2 * waves * 1024;
    return lds <= kMx4Lds;
}

template <int XT>
static int launch_decode(const char* name, const Mx4Args& a, int waves, int xb, int lds, hipStream_t st) {
    // resident workgroups: LDS, and registers for 16 waves per CU
    const int occ = kMx4Lds / lds < 16 / waves ? kMx4Lds / lds : 16 / waves;
    // the fewest that need no more rounds (six rows of 5376 -> 21504: 448 of 512 workgroups, 18.7 -> 18.4 us)
    const int64_t tiles = (a.n + 15) / 16, rounds = (tiles + 256 * occ - 1) / (256 * occ), grid = (tiles + rounds - 1) / rounds;
    EXL3_CHECK_ARG(tiles <= 0x3FFFFFFF, "%s: grid too large", name);
    EXL3_LAUNCH(name, mx4_decode_kernel<XT>, dim3((unsigned)grid), dim3(64 * waves), (size_t)lds, st, a, xb);
    return EXL3_OK;
}

// ------------------------------------------------------------------------------------------------ many 16-bit rows
template <int XT, int RG>
__global__ __launch_bounds__(256, mx4_wide_occ(RG)) void mx4_wide_kernel(Mx4Args a) {
    typedef Mx4Wide<XT, RG> L;
    __shared__ u32x4_t lds[L::kLds];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    unsigned mt, nt, sp;
    if (!mx4_tile_of((unsigned)((a.m + 32 * RG - 1) / (32 * RG)), (unsigned)((a.n + 255) / 256), a.splits, mt, nt, sp)) return;
    const int64_t m0 = (int64_t)mt * (32 * RG), n0 = (int64_t)nt * 256 + 64 * wave;
    L p;
    p.kb = a.k / 32;
    p.lds = lds;
    p.base = XT == kRowF16 ? a.base : 0;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
        const int64_t m = m0 + (t >> 3) + 32 * i;
        p.xp[i] = a.x + (m < a.m ? m : a.m - 1) * a.x_ld;
    }
    p.weights(a.w, a.ws, n0, a.n, lane);
    typename L::Acc acc;
    L::zero(acc);
    p.run(t, sp * a.bps, a.bps, acc);
#pragma unroll
    for (int j = 0; j < RG; ++j) {
        if constexpr (RG == 4)
            L::each16(acc, j, lane, [&](int row, int n, f4_t v, f4_t w) { mx4_put16(a, sp, m0 + 32 * j + row, n0 + n, lane >> 5, v, w); });
        else
            L::each(acc, j, lane, [&](int row, int n, f4_t v) { mx4_put(a, sp, m0 + 32 * j + row, n0 + n, v); });
    }
}

template <int XT, int RG>
static int launch_wide(Mx4Args a, const Mx4Plan& plan, const CallScratch& s, hipStream_t st) {
    const int64_t tiles = (a.m + 32 * RG - 1) / (32 * RG) * ((a.n + 255) / 256);
    EXL3_CHECK_ARG(tiles * plan.P <= kMx4Grid - 7, "exl3_mx4_linear: grid too large");
    const int rc = mx4_split("exl3_mx4_linear", a, plan, s, st);
    if (rc) return rc;
    EXL3_LAUNCH("mx4_linear_wide", (mx4_wide_kernel<XT, RG>), dim3((unsigned)((tiles * a.splits + 7) & ~7)), dim3(256), 0, st, a);
    return launch_reduce(a, st);
}

template <int XT>
static int linear_run(const Mx4Args& a, const CallScratch& s, hipStream_t st) {
    if (a.n * (a.k / 32) < 16) return launch_tiny<XT>("mx4_linear_tiny", a, st);
    int waves, xb, lds;
    if (decode_shape<XT>(a.m, a.k, waves, xb, lds)) return launch_decode<XT>("mx4_linear", a, waves, xb, lds, st);
    const Mx4Plan p = mx4_linear_plan(a.m, a.n, a.k, 256);
    return p.tile == 0 ? launch_wide<XT, 1>(a, p, s, st) : p.tile == 1 ? launch_wide<XT, 2>(a, p, s, st)
                                                                       : launch_wide<XT, 4>(a, p, s, st);
}

// ------------------------------------------------------------------------------------------------ many MX4 rows
// Tile of a product of two MX4 matrices on 32 x 32 x 64 scaled MFMAs, for many rows: WM x WN waves of TM x TN products each.
// Steps of 128 k: 64 bytes of codes per row of either operand, staged through registers into one of two LDS buffers while
// the other is multiplied, two steps' loads under way (one: 205 us instead of 183); the scales of four steps (16 bytes per row)
// likewise. Lane l of a fragment takes blocks
// 2 (l >> 5) and 2 (l >> 5) + 1 of its row's four, one per MFMA, so that both scales are neighbouring bytes of one word.
// In LDS a row's four 16-byte units are permuted by its row number, so that eight neighbouring lanes reading eight rows, or writing
// two, touch every bank once (the counters show conflicts for a third of the LDS cycles nevertheless).
// 2048 rows of 5376 -> 21504 (256 x 256) 165 us, 2.9 PFLOP/s: a step takes 2500 cycles for 1024 of MFMAs and 1050 to 1400 of LDS (42 %,
// 56 % with the conflicts); the barrier keeps the waves in step, so that little of either hides behind the other; and 672 tiles
// take three rounds of the CUs for 2.6 rounds' work.
template <int TM, int TN, int WM, int WN>
struct Mx4Tile {
    static constexpr int kThreads = 64 * WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, R = BM + BN;
    static constexpr int kUnits = R * 4 / kThreads, kScaleRows = (R + kThreads - 1) / kThreads;
    static constexpr int kLds = 2 * R * 64 + 2 * R * 16;
    static_assert(R * 4 % kThreads == 0 && BM % (kThreads / 4) == 0, "staging");
};

__device__ __forceinline__ int mx4_unit(int row, int unit) { return row * 4 + (unit ^ (row >> 1 & 3)); }

template <int TM, int TN, int WM, int WN, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void mx4_tile_kernel(Mx4Args a) {
    typedef Mx4Tile<TM, TN, WM, WN> T;
    __shared__ u32x4_t codes[2][T::R * 4];
    __shared__ uint32_t scales[2][4][T::R];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const unsigned nmt = (unsigned)((a.m + T::BM - 1) / T::BM), nnt = (unsigned)((a.n + T::BN - 1) / T::BN);
    unsigned mt, nt, sp;
    if (!mx4_tile_of(nmt, nnt, a.splits, mt, nt, sp)) return;
    const int64_t m0 = (int64_t)mt * T::BM, n0 = (int64_t)nt * T::BN;
    const int kb = a.k / 32, c0 = sp * a.bps, nch = (kb + 3) / 4 - c0 < a.bps ? (kb + 3) / 4 - c0 : a.bps;

    // staging: this thread's unit t & 3 of rows (t >> 2) + i kThreads / 4, the x rows first, at 32-bit offsets from the
    // tile's first rows; buffer loads return 0 past the matrix, and x units past their row's end are moved there
    const __amdgpu_buffer_rsrc_t xr = mx4_rsrc(a.x + m0 * a.x_ld, (a.m - m0) * a.x_ld),
                                 wr = mx4_rsrc(a.w + n0 * (a.k / 2), (a.n - n0) * (a.k / 2));
    constexpr int kStep = T::kThreads / 4;
    uint32_t src[T::kUnits];
#pragma unroll
    for (int i = 0; i < T::kUnits; ++i) {
        const int r = (t >> 2) + i * kStep;
        src[i] = (uint32_t)(r < T::BM ? r : r - T::BM) * (uint32_t)(a.k / 2) + 16 * (t & 3);
    }
    u32x4_t st[2][T::kUnits], ss[T::kScaleRows];             // codes of steps c + 1 and c + 2 under way
    const auto load_codes = [&](int c, u32x4_t (&d)[T::kUnits]) {
        const bool in = 4 * (c0 + c) + (t & 3) < kb;
#pragma unroll
        for (int i = 0; i < T::kUnits; ++i)
            d[i] = i * kStep < T::BM ? mx4_buffer16(xr, in ? src[i] + 64 * (c0 + c) : kMx4Out) : mx4_buffer16(wr, src[i] + 64 * (c0 + c));
    };
    const auto load_scales = [&](int s) {
#pragma unroll
        for (int i = 0; i < T::kScaleRows; ++i) {
            const int r = t + i * T::kThreads;
            if (T::R % T::kThreads != 0 && r >= T::R) break;
            const int64_t m = m0 + r, n = n0 + r - T::BM;
            const bool ix = r < T::BM;
            const int64_t row = ix ? (m < a.m ? m : a.m - 1) : (n < a.n ? n : a.n - 1);
            ss[i] = mx4_scales16((ix ? a.xs : a.ws) + row * kb, 4 * c0 + 16 * s, ((ix ? a.m : a.n) - row) * kb);
        }
    };
    const auto store_codes = [&](int buf, const u32x4_t (&d)[T::kUnits]) {
#pragma unroll
        for (int i = 0; i < T::kUnits; ++i) codes[buf][mx4_unit((t >> 2) + i * kStep, t & 3)] = d[i];
    };
    const auto store_scales = [&](int s) {                     // bytes past a row's end are the next row's: 0 (255 times 0 is NaN)
#pragma unroll
        for (int i = 0; i < T::kScaleRows; ++i) {
            const int r = t + i * T::kThreads;
            if (T::R % T::kThreads != 0 && r >= T::R) break;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int left = kb - 4 * c0 - 16 * s - 4 * q;
                scales[s & 1][q][r] = ss[i][q] & (left >= 4 ? ~0u : left > 0 ? (1u << (8 * left)) - 1 : 0u);
            }
        }
    };

    const int r = lane & 31, g = lane >> 5, rm = (wave / WN) * 32 * TM + r, rn = T::BM + (wave % WN) * 32 * TN + r;
    f16_t acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f16_t{};

    load_codes(0, st[0]);
    load_scales(0);
    load_codes(1, st[1]);
    store_codes(0, st[0]);
    store_scales(0);
    __syncthreads();
    const int nsup = (nch + 3) / 4;
    for (int sp = 0; sp < nsup; ++sp) {
        load_scales(sp + 1 < nsup ? sp + 1 : sp);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
            const int c = 4 * sp + cc;
            if (c >= nch) break;                               // uniform
            load_codes(c + 2, st[cc & 1]);                     // (past the last: not used)
            __builtin_amdgcn_sched_barrier(0);                 // on their way before the products
            const u32x4_t* cb = codes[cc & 1];
            const uint32_t* sb = scales[sp & 1][cc];
            int sx[TM], sw[TN];
#pragma unroll
            for (int j = 0; j < TM; ++j) sx[j] = (int)(sb[rm + 32 * j] >> (16 * g));
#pragma unroll
            for (int i = 0; i < TN; ++i) sw[i] = (int)(sb[rn + 32 * i] >> (16 * g));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4_t x[TM], w[TN];
#pragma unroll
                for (int j = 0; j < TM; ++j) x[j] = cb[mx4_unit(rm + 32 * j, 2 * g + s)];
#pragma unroll
                for (int i = 0; i < TN; ++i) w[i] = cb[mx4_unit(rn + 32 * i, 2 * g + s)];
#pragma unroll
                for (int i = 0; i < TN; ++i)
#pragma unroll
                    for (int j = 0; j < TM; ++j)
                        acc[i][j] = s == 0 ? mfma32_mx4<0>(w[i], sw[i], x[j], sx[j], acc[i][j])
                                           : mfma32_mx4<1>(w[i], sw[i], x[j], sx[j], acc[i][j]);
            }
            __builtin_amdgcn_sched_barrier(0);                 // the loads are waited for here, behind the products
            store_codes(~cc & 1, st[~cc & 1]);
            if (cc == 3) store_scales(sp + 1);
            __syncthreads();
        }
    }
    // lane l holds column l & 31 (a row of x), rows 8 q + 4 (l >> 5) + 0 .. 3 (neighbouring outputs)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; q += 2)
                mx4_put16(a, sp, m0 + rm + 32 * j, n0 + rn - T::BM + 32 * i - r + 8 * q, g,
                          f4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]},
                          f4_t{acc[i][j][4 * q + 4], acc[i][j][4 * q + 5], acc[i][j][4 * q + 6], acc[i][j][4 * q + 7]});
}

template <int TM, int TN, int WM, int WN, int OCC>
static int launch_tile(Mx4Args a, const Mx4Plan& plan, const CallScratch& s, hipStream_t st) {
    typedef Mx4Tile<TM, TN, WM, WN> T;
    const int64_t tiles = (a.m + T::BM - 1) / T::BM * ((a.n + T::BN - 1) / T::BN);
    EXL3_CHECK_ARG(tiles * plan.P <= kMx4Grid * 256 / T::kThreads - 7, "exl3_mx4_gemm: grid too large");
    const int rc = mx4_split("exl3_mx4_gemm", a, plan, s, st);
    if (rc) return rc;
    EXL3_LAUNCH("mx4_gemm_tile", (mx4_tile_kernel<TM, TN, WM, WN, OCC>), dim3((unsigned)((tiles * a.splits + 7) & ~7)),
                dim3(T::kThreads), 0, st, a);
    return launch_reduce(a, st);
}

static bool mx4_dtype(int t) { return t == EXL3_F16 || t == EXL3_F32 || t == EXL3_BF16; }
static int elem_size(int t) { return t == EXL3_F32 ? 4 : 2; }

// Sizes that both products take.
static bool mx4_sizes(int64_t m, int64_t n, int64_t k) {
    return m >= 0 && n > 0 && k > 0 && k % 32 == 0 && k <= (1 << 24) && m <= ((int64_t)1 << 40) / k && n <= ((int64_t)1 << 40) / k;
}

// What both products check of their weights and output; sets those of the kernel's arguments.
static int mx4_setup(const char* what, int64_t m, int64_t n, int64_t k, const uint8_t* w, const uint8_t* ws,
                     const float* bias, void* C, int64_t c_ld, int c_dtype, Mx4Args& a) {
    EXL3_CHECK_ARG(m >= 0 && n > 0 && k > 0 && k % 32 == 0 && k <= (1 << 24), "%s: bad sizes (m %lld, n %lld, k %lld; k a "
                   "multiple of 32, at most 2^24)", what, (long long)m, (long long)n, (long long)k);
    EXL3_CHECK_ARG(mx4_dtype(c_dtype), "%s: the output must be fp16, bf16 or fp32", what);
    EXL3_CHECK_ARG(c_ld >= n, "%s: output row stride %lld < n", what, (long long)c_ld);
    EXL3_CHECK_ARG(m <= ((int64_t)1 << 40) / k && n <= ((int64_t)1 << 40) / k, "%s: operand too large", what);
    if (m == 0) return EXL3_OK;
    a.splits = 1;
    EXL3_CHECK_ARG(w && ws && C, "%s: null pointer", what);
    EXL3_CHECK_ARG(aligned(w, 16), "%s: weight codes must be 16-byte aligned", what);
    EXL3_CHECK_ARG(aligned(C, elem_size(c_dtype)) && (!bias || aligned(bias, 4)), "%s: misaligned output or bias", what);
    a.w = w;
    a.ws = ws;
    a.bias = bias;
    a.out = C;
    a.out_ld = c_ld;
    a.m = m;
    a.n = n;
    a.k = (int)k;
    a.out_dtype = c_dtype;
    a.vec = n % 4 == 0 && c_ld % 4 == 0 && aligned(C, 4 * elem_size(c_dtype));
    if (c_dtype != EXL3_F32 && n % 8 == 0 && c_ld % 8 == 0 && aligned(C, 16)) a.vec = 2;
    return EXL3_OK;
}

static int mx4_linear(const void* x, int64_t x_ld, int x_dtype, int64_t m, int64_t k, const uint8_t* codes, const uint8_t* scales,
                      int64_t n, int scale_base, const float* bias, void* C, int64_t c_ld, int c_dtype, const CallScratch& s,
                      void* stream) {
    EXL3_CHECK_ARG(x_dtype == EXL3_F16 || x_dtype == EXL3_BF16, "exl3_mx4_linear: x must be fp16 or bf16");
    EXL3_CHECK_ARG(x_ld >= k, "exl3_mx4_linear: x row stride %lld < k", (long long)x_ld);
    EXL3_CHECK_ARG(scale_base >= -140 && scale_base <= 140, "exl3_mx4_linear: scale_base %d out of range", scale_base);
    Mx4Args a{};
    const int rc = mx4_setup("exl3_mx4_linear", m, n, k, codes, scales, bias, C, c_ld, c_dtype, a);
    if (rc || m == 0) return rc;
    EXL3_CHECK_ARG(x && aligned(x, 16) && (m == 1 || x_ld % 8 == 0), "exl3_mx4_linear: x rows must be 16-byte aligned");
    EXL3_CHECK_ARG(m <= ((int64_t)1 << 45) / x_ld, "exl3_mx4_linear: operand too large");
    a.x = reinterpret_cast<const uint8_t*>(x);
    a.x_ld = 2 * x_ld;
    a.base = x_dtype == EXL3_F16 ? scale_base : 0;
    return x_dtype == EXL3_F16 ? linear_run<kRowF16>(a, s, (hipStream_t)stream) : linear_run<kRowBF16>(a, s, (hipStream_t)stream);
}

static int mx4_gemm(const uint8_t* a_codes, const uint8_t* a_scales, int64_t m, int64_t k, const uint8_t* b_codes,
                    const uint8_t* b_scales, int64_t n, const float* bias, void* C, int64_t c_ld, int c_dtype, const CallScratch& s,
                    void* stream) {
    Mx4Args a{};
    const int rc = mx4_setup("exl3_mx4_gemm", m, n, k, b_codes, b_scales, bias, C, c_ld, c_dtype, a);
    if (rc || m == 0) return rc;
    EXL3_CHECK_ARG(a_codes && a_scales && aligned(a_codes, 16), "exl3_mx4_gemm: row codes must be 16-byte aligned");
    a.x = a_codes;
    a.xs = a_scales;
    a.x_ld = k / 2;
    hipStream_t st = (hipStream_t)stream;
    if (m * (k / 32) < 16 || n * (k / 32) < 16) return launch_tiny<kRowMX4>("mx4_gemm_tiny", a, st);
    int waves, xb, lds;
    if (decode_shape<kRowMX4>(m, k, waves, xb, lds)) return launch_decode<kRowMX4>("mx4_gemm", a, waves, xb, lds, st);
    const Mx4Plan p = mx4_gemm_plan(m, n, k, 256);
    return p.tile == 0 ? launch_tile<2, 1, 1, 4, 4>(a, p, s, st) : p.tile == 1 ? launch_tile<2, 2, 2, 2, 3>(a, p, s, st)
                                                              : launch_tile<4, 2, 2, 4, 2>(a, p, s, st);
}

}  // namespace exl3

extern "C" {

using namespace exl3;

int exl3_mx4_quantize(const void* x, int64_t x_ld, int64_t rows, int64_t k, int x_dtype, uint8_t* codes, uint8_t* scales,
                      void* stream) {
    EXL3_CHECK_ARG(rows >= 0 && k > 0 && k % 32 == 0 && x_ld >= k, "exl3_mx4_quantize: bad sizes (rows %lld, k %lld, row "
                   "stride %lld; k a multiple of 32)", (long long)rows, (long long)k, (long long)x_ld);
    EXL3_CHECK_ARG(mx4_dtype(x_dtype), "exl3_mx4_quantize: x must be fp16, bf16 or fp32");
    if (rows == 0) return EXL3_OK;
    EXL3_CHECK_ARG(x && codes && scales, "exl3_mx4_quantize: null pointer");
    EXL3_CHECK_ARG(aligned(x, 16) && (rows == 1 || x_ld * elem_size(x_dtype) % 16 == 0) && aligned(codes, 4),
                   "exl3_mx4_quantize: rows must be 16-byte aligned and codes 4-byte");
    EXL3_CHECK_ARG(rows <= ((int64_t)1 << 45) / x_ld, "exl3_mx4_quantize: too large");
    const int elem = elem_size(x_dtype);
    const auto fn = x_dtype == EXL3_F16 ? mx4_quantize_kernel<EXL3_F16>
                  : x_dtype == EXL3_BF16 ? mx4_quantize_kernel<EXL3_BF16> : mx4_quantize_kernel<EXL3_F32>;
    QuantGrid g;
    if (!quant_grid(rows, k, x_ld, g)) return fail(EXL3_ERR_INVALID, "exl3_mx4_quantize: too large");
    for (int64_t r = 0; r < g.rows; r += g.most) {
        const int64_t n = g.rows - r < g.most ? g.rows - r : g.most;
        EXL3_LAUNCH("mx4_quantize", fn, dim3((unsigned)(n * g.cpr)), dim3(256), 0, (hipStream_t)stream,
                    reinterpret_cast<const char*>(x) + r * x_ld * elem, x_ld, g.upr, (int)g.cpr,
                    reinterpret_cast<uint32_t*>(codes) + r * g.upr, scales + r * (g.upr / 4));
    }
    return EXL3_OK;
}

int exl3_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, void* out, int64_t out_ld,
                        int out_dtype, void* stream) {
    EXL3_CHECK_ARG(rows >= 0 && k > 0 && k % 32 == 0 && out_ld >= k, "exl3_mx4_dequantize: bad sizes (rows %lld, k %lld, "
                   "row stride %lld; k a multiple of 32)", (long long)rows, (long long)k, (long long)out_ld);
    EXL3_CHECK_ARG(mx4_dtype(out_dtype), "exl3_mx4_dequantize: the output must be fp16, bf16 or fp32");
    if (rows == 0) return EXL3_OK;
    EXL3_CHECK_ARG(out && codes && scales, "exl3_mx4_dequantize: null pointer");
    EXL3_CHECK_ARG(aligned(out, 16) && (rows == 1 || out_ld * elem_size(out_dtype) % 16 == 0) && aligned(codes, 4),
                   "exl3_mx4_dequantize: rows must be 16-byte aligned and codes 4-byte");
    EXL3_CHECK_ARG(rows <= ((int64_t)1 << 45) / out_ld, "exl3_mx4_dequantize: too large");
    const int elem = elem_size(out_dtype);
    const auto fn = out_dtype == EXL3_F16 ? mx4_dequantize_kernel<EXL3_F16>
                  : out_dtype == EXL3_BF16 ? mx4_dequantize_kernel<EXL3_BF16> : mx4_dequantize_kernel<EXL3_F32>;
    QuantGrid g;
    if (!quant_grid(rows, k, out_ld, g)) return fail(EXL3_ERR_INVALID, "exl3_mx4_dequantize: too large");
    for (int64_t r = 0; r < g.rows; r += g.most) {
        const int64_t n = g.rows - r < g.most ? g.rows - r : g.most;
        EXL3_LAUNCH("mx4_dequantize", fn, dim3((unsigned)(n * g.cpr)), dim3(256), 0, (hipStream_t)stream,
                    reinterpret_cast<const uint32_t*>(codes) + r * g.upr, scales + r * (g.upr / 4), g.upr, (int)g.cpr,
                    reinterpret_cast<char*>(out) + r * out_ld * elem, out_ld);
    }
    return EXL3_OK;
}

int64_t exl3_mx4_linear_scratch(int64_t m, int64_t k, int64_t n) {
    int waves, xb, lds;
    if (!mx4_sizes(m, n, k) || m == 0 || n * (k / 32) < 16 || decode_shape<kRowF16>(m, k, waves, xb, lds)) return 0;
    return mx4_part_bytes(mx4_linear_plan(m, n, k, 256), m, n);
}

int64_t exl3_mx4_gemm_scratch(int64_t m, int64_t k, int64_t n) {
    int waves, xb, lds;
    if (!mx4_sizes(m, n, k) || m == 0 || m * (k / 32) < 16 || n * (k / 32) < 16 || decode_shape<kRowMX4>(m, k, waves, xb, lds)) return 0;
    return mx4_part_bytes(mx4_gemm_plan(m, n, k, 256), m, n);
}

int exl3_mx4_linear(const void* x, int64_t x_ld, int x_dtype, int64_t m, int64_t k, const uint8_t* codes,
                    const uint8_t* scales, int64_t n, int scale_base, const float* bias, void* C, int64_t c_ld,
                    int c_dtype, void* stream) {
    return mx4_linear(x, x_ld, x_dtype, m, k, codes, scales, n, scale_base, bias, C, c_ld, c_dtype, kLibScratch, stream);
}

int exl3_mx4_linear_in(const void* x, int64_t x_ld, int x_dtype, int64_t m, int64_t k, const uint8_t* codes,
                       const uint8_t* scales, int64_t n, int scale_base, const float* bias, void* C, int64_t c_ld,
                       int c_dtype, void* scratch, int64_t scratch_bytes, void* stream) {
    return mx4_linear(x, x_ld, x_dtype, m, k, codes, scales, n, scale_base, bias, C, c_ld, c_dtype,
                      CallScratch{scratch, scratch_bytes, false}, stream);
}

int exl3_mx4_gemm(const uint8_t* a_codes, const uint8_t* a_scales, int64_t m, int64_t k, const uint8_t* b_codes,
                  const uint8_t* b_scales, int64_t n, const float* bias, void* C, int64_t c_ld, int c_dtype, void* stream) {
    return mx4_gemm(a_codes, a_scales, m, k, b_codes, b_scales, n, bias, C, c_ld, c_dtype, kLibScratch, stream);
}

int exl3_mx4_gemm_in(const uint8_t* a_codes, const uint8_t* a_scales, int64_t m, int64_t k, const uint8_t* b_codes,
                     const uint8_t* b_scales, int64_t n, const float* bias, void* C, int64_t c_ld, int c_dtype, void* scratch,
                     int64_t scratch_bytes, void* stream) {
    return mx4_gemm(a_codes, a_scales, m, k, b_codes, b_scales, n, bias, C, c_ld, c_dtype, CallScratch{scratch, scratch_bytes, false},
                    stream);
}

}  // extern "C"
