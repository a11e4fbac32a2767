// Router balance: per-expert counts, mean shares and the balance loss, and its gradient.
//   s = score(logit), S = sum s over the row, p = s / S; loss = coef sum_e f_e P_e with f_e = E c_e / (k N) (constant in the
//   gradient) and P_e = sum over live rows of p / N. With a_e = grad coef f_e / N and abar = sum_e p_e a_e:
//     softmax        d/dl_j = p_j (a_j - abar)
//     sigmoid        d/dl_j = p_j (1 - s_j) (a_j - abar)                   (ds/dl = s (1 - s))
//     sqrt-softplus  d/dl_j = p_j sigma(l_j) / (2 softplus(l_j)) (a_j - abar)   (ds/dl = sigma / (2 s))
// A wave takes a row (E <= 2048; above, the four waves of a workgroup share one) and holds it in registers, so each pass
// reads the logits once. 32768 padded rows of 512, half of them live: gradient 21.0 us, near its bytes (101 MB); forward 17.3 for 34
// MB, a wait for memory per live row, since its picks arrive behind the next row's logits, and 6.9 for the partials. A decode
// step's few rows are bound by launch latency.
#include "exl3_device.h"
#include "exl3_runtime.h"

namespace exl3 {

struct BalanceArgs {
    const float* z;
    int64_t ld;
    int M, E, topk;
    const int32_t* ids;
    const uint8_t* mask;               // or null
    float coef;
    float* loss;
    int32_t* counts;
    float* prob;
    int32_t* rows;
    // several workgroups: partials [G][E] (sums of shares, counts) and [G] (live rows), loss terms of the column blocks
    float* part_p;
    int32_t* part_c;
    int32_t* part_n;
    float* part_l;
    int* arrived;
    int G;
    // gradient
    const float* grad;
    float* dz;
    int64_t d_ld;
};

// Sum or maximum over the lanes that share a row: a wave, or W waves of the workgroup through LDS.
template <int W>
__device__ __forceinline__ float row_sum(float v, float* tmp) {
    v = wave_sum_f32(v);
    if constexpr (W > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
        __syncthreads();
        v = tmp[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v += tmp[w];
    }
    return v;
}
template <int W>
__device__ __forceinline__ float row_max(float v, float* tmp) {
    uint32_t k = wave_max_u32(float_key(v));
    if constexpr (W > 1) {
        uint32_t* t = reinterpret_cast<uint32_t*>(tmp);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) t[threadIdx.x >> 6] = k;
        __syncthreads();
        k = t[0];
#pragma unroll
        for (int w = 1; w < W; ++w) k = max(k, t[w]);
    }
    return key_float(k);
}

// Rows first, first + step, .. of a workgroup's or wave's share: fn(row, the next live one or -1, whether it is the first) for
// the live ones of 64 rows at a time, whose mask bytes are one load; dead(row) for the others.
template <typename F, typename G>
__device__ __forceinline__ void each_row(const uint8_t* mask, int M, int first, int step, F fn, G dead) {
    const int lane = threadIdx.x & 63;
    for (int64_t r0 = first; r0 < M; r0 += 64 * (int64_t)step) {
        const int64_t r = r0 + lane * (int64_t)step;
        const uint64_t in = __ballot(r < M), live = mask ? __ballot(r < M && ldg(mask + (r < M ? r : 0)) != 0) : in;
        for (uint64_t b = live; b; b &= b - 1) {
            const uint64_t rest = b & (b - 1);
            fn((int)(r0 + __builtin_ctzll(b) * (int64_t)step), rest ? (int)(r0 + __builtin_ctzll(rest) * (int64_t)step) : -1, b == live);
        }
        for (uint64_t b = in & ~live; b; b &= b - 1) dead((int)(r0 + __builtin_ctzll(b) * (int64_t)step));
    }
}

template <int V, int W>
__device__ __forceinline__ void load_row(const float* z, int E, float (&f)[V]) {
    const int l = W > 1 ? threadIdx.x : threadIdx.x & 63;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = l + 64 * W * v;
        f[v] = ldg(z + (e < E ? e : E - 1));
    }
}

// Shares p of a row's logits f (0 past E), which lie at z; in the gradient also each score's derivative over the score, ds / (s dl).
// Far below 0 sigmoid(l) is e^l and sqrt(softplus(l)) is e^(l / 2), the forms taken where the others' parts leave fp32 (l < -80). A row
// whose scores add up to so little that all its logits are below -16 takes them relative to its largest logit, as softmax
// does: its shares stay what they are however low it lies.
template <int V, int W, int SC, bool GRAD>
__device__ __forceinline__ void row_shares(float (&f)[V], float (&d)[V], const float* zrow, int E, float* tmp) {
    const int l = W > 1 ? threadIdx.x : threadIdx.x & 63;
    float mx = 0.f;
    if constexpr (SC == EXL3_SCORE_SOFTMAX) {
        mx = -__builtin_inff();
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (l + 64 * W * v < E) mx = fmaxf(mx, f[v]);
        mx = row_max<W>(mx, tmp);
        if (mx == -__builtin_inff()) mx = 0.f;                 // every logit -inf: scores 0
    }
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float z = f[v];
        float s;
        if constexpr (SC == EXL3_SCORE_SOFTMAX) {
            s = expf(z - mx);
        } else if constexpr (SC == EXL3_SCORE_SIGMOID) {
            const float e = expf(z < -80.f ? z : -z);
            s = z < -80.f ? e : 1.f / (1.f + e);
            if constexpr (GRAD) d[v] = 1.f / (1.f + expf(z));
        } else {
            const float e = expf(z < -80.f ? 0.5f * z : z), sp = z > 20.f ? z : log1pf(e);
            s = z < -80.f ? e : sqrtf(sp);
            // sigma / softplus tends to 1 below; past e^-17 it is 1 to fp32 (and softplus may be 0)
            if constexpr (GRAD) d[v] = z < -17.f ? 0.5f : 0.5f / ((1.f + expf(-z)) * sp);
        }
        f[v] = l + 64 * W * v < E ? s : 0.f;
        sum += f[v];
    }
    sum = row_sum<W>(sum, tmp);
    if constexpr (SC != EXL3_SCORE_SOFTMAX) {
        // e^l < 2^-24 for every l (a wave's, or with W > 1 the workgroup's, common value)
        if (__builtin_amdgcn_readfirstlane(sum < (SC == EXL3_SCORE_SIGMOID ? 0x1p-24f : 0x1p-12f))) {
            load_row<V, W>(zrow, E, f);
            mx = -__builtin_inff();
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (l + 64 * W * v < E) mx = fmaxf(mx, f[v]);
            mx = row_max<W>(mx, tmp);
            if (mx == -__builtin_inff()) mx = 0.f;             // every logit -inf: scores 0
            sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f[v] = l + 64 * W * v < E ? expf((SC == EXL3_SCORE_SIGMOID ? 1.f : 0.5f) * (f[v] - mx)) : 0.f;
                sum += f[v];
            }
            sum = row_sum<W>(sum, tmp);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] *= inv;
}

__device__ __forceinline__ float balance_fraction(int c, int E, int topk, int n) {
    return n > 0 ? (float)c * ((float)E / ((float)topk * (float)n)) : 0.f;
}

// Shares, counts and live rows of this workgroup's rows. One workgroup: the results; else partials. LDS: E counts, and with a
// row per wave E floats, to which the waves' sums are added in wave order (a row per workgroup: each thread has its columns'
// sums).
template <int V, int W, int SC>
__global__ __launch_bounds__(512) void balance_kernel(BalanceArgs a) {
    extern __shared__ float sm[];
    int* sc = reinterpret_cast<int*>(sm);
    float* sp = sm + a.E;
    __shared__ float tmp[8];
    __shared__ int s_live;
    const int t = threadIdx.x, T = blockDim.x, waves = T >> 6, wave = t >> 6, l = W > 1 ? t : t & 63;
    for (int e = t; e < a.E; e += T) {
        sc[e] = 0;
        if constexpr (W == 1) sp[e] = 0.f;
    }
    if (t == 0) s_live = 0;
    __syncthreads();
    const int nrow = W > 1 ? 1 : waves;                        // rows at a time
    const int first = W > 1 ? blockIdx.x : blockIdx.x * nrow + wave, step = gridDim.x * nrow;
    float acc[V], d[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
    int live = 0;
    float f[V], nx[V];
    each_row(a.mask, a.M, first, step, [&](int r, int next, bool start) {
        ++live;
        if (start) load_row<V, W>(a.z + (int64_t)r * a.ld, a.E, nx);
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = nx[v];
        if (next >= 0) load_row<V, W>(a.z + (int64_t)next * a.ld, a.E, nx);
        for (int j = l; j < a.topk; j += 64 * W) {
            const int e = ldg(a.ids + (int64_t)r * a.topk + j);
            if (e >= 0 && e < a.E) atomicAdd(&sc[e], 1);
        }
        row_shares<V, W, SC, false>(f, d, a.z + (int64_t)r * a.ld, a.E, tmp);
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += f[v];
    }, [](int) {});
    if (l == 0) atomicAdd(&s_live, live);
    if constexpr (W == 1) {
        for (int w = 0; w < waves; ++w) {
            if (w == wave)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (l + 64 * v < a.E) sp[l + 64 * v] += acc[v];
            __syncthreads();
        }
    } else {
        __syncthreads();
    }
    // column e of this thread with its sum
    const auto columns = [&](auto fn) {
        if constexpr (W == 1) {
            for (int e = t; e < a.E; e += T) fn(e, sp[e]);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (t + 64 * W * v < a.E) fn(t + 64 * W * v, acc[v]);
        }
    };
    if (gridDim.x > 1) {
        columns([&](int e, float p) {
            a.part_p[(int64_t)blockIdx.x * a.E + e] = p;
            a.part_c[(int64_t)blockIdx.x * a.E + e] = sc[e];
        });
        if (t == 0) a.part_n[blockIdx.x] = s_live;
        if (t == 0 && blockIdx.x == 0) *a.arrived = 0;         // (counted by the reduction, a launch later)
        return;
    }
    const int n = s_live;
    float term = 0.f;
    columns([&](int e, float p) {
        p = n > 0 ? p / (float)n : 0.f;
        a.prob[e] = p;
        a.counts[e] = sc[e];
        term += balance_fraction(sc[e], a.E, a.topk, n) * p;
    });
    term = wave_sum_f32(term);
    __syncthreads();
    if ((t & 63) == 0) tmp[wave] = term;
    __syncthreads();
    if (t == 0) {
        float s = 0.f;
        for (int w = 0; w < waves; ++w) s += tmp[w];
        a.loss[0] = a.coef * s;
        a.rows[0] = n;
    }
}

// Sums of the partials in workgroup order for 16 columns: 16 threads' groups take every 16th partial each, then one adds
// them. The workgroup that arrives last adds the column blocks' loss terms in order.
__global__ __launch_bounds__(256) void balance_reduce_kernel(BalanceArgs a) {
    __shared__ float s_p[16][17];
    __shared__ int s_c[16][17], s_n[4], s_last;
    const int t = threadIdx.x, q = t & 15, g = t >> 4, e = blockIdx.x * 16 + q, ec = e < a.E ? e : a.E - 1;
    int n = 0;
    for (int i = t; i < a.G; i += 256) n += ldg(a.part_n + i);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    if ((t & 63) == 0) s_n[t >> 6] = n;
    float p = 0.f;
    int c = 0;
    for (int i0 = g; i0 < a.G; i0 += 128) {                    // eight loads of each kind under way
        float pv[8];
        int cv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = i0 + 16 * i < a.G ? i0 + 16 * i : i0;
            pv[i] = ldg(a.part_p + (int64_t)at * a.E + ec);
            cv[i] = ldg(a.part_c + (int64_t)at * a.E + ec);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p += i0 + 16 * i < a.G ? pv[i] : 0.f;
            c += i0 + 16 * i < a.G ? cv[i] : 0;
        }
    }
    s_p[g][q] = p;
    s_c[g][q] = c;
    __syncthreads();
    n = s_n[0] + s_n[1] + s_n[2] + s_n[3];
    float term = 0.f;
    if (t < 16) {
        p = s_p[0][q];
        c = s_c[0][q];
        for (int i = 1; i < 16; ++i) {
            p += s_p[i][q];
            c += s_c[i][q];
        }
        p = n > 0 ? p / (float)n : 0.f;
        if (e < a.E) {
            a.prob[e] = p;
            a.counts[e] = c;
            term = balance_fraction(c, a.E, a.topk, n) * p;
        }
    }
    if (t < 64) {
        term = wave_sum_f32(term);
        if (t == 0) {
            __hip_atomic_store(a.part_l + blockIdx.x, term, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = __hip_atomic_fetch_add(a.arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!s_last || t >= 64) return;
    float s = 0.f;
    for (int i = t; i < (int)gridDim.x; i += 64)
        s += __hip_atomic_load(a.part_l + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = wave_sum_f32(s);
    if (t == 0) {
        a.loss[0] = a.coef * s;
        a.rows[0] = n;
        __hip_atomic_store(a.arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

template <int V, int W, int SC>
__global__ __launch_bounds__(256) void balance_grad_kernel(BalanceArgs a) {
    __shared__ float tmp[8];
    const int t = threadIdx.x, wave = t >> 6, l = W > 1 ? t : t & 63;
    const int n = ldg(a.rows);
    const float g = (a.grad ? ldg(a.grad) : 1.f) * a.coef;
    float w[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = l + 64 * W * v;
        w[v] = n > 0 && e < a.E ? g * balance_fraction(ldg(a.counts + e), a.E, a.topk, n) / (float)n : 0.f;
    }
    const int nrow = W > 1 ? 1 : 4;
    float f[V], nx[V], d[V];
    each_row(a.mask, a.M, W > 1 ? blockIdx.x : blockIdx.x * nrow + wave, gridDim.x * nrow, [&](int r, int next, bool start) {
        if (start) load_row<V, W>(a.z + (int64_t)r * a.ld, a.E, nx);
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = nx[v];
        if (next >= 0) load_row<V, W>(a.z + (int64_t)next * a.ld, a.E, nx);
        row_shares<V, W, SC, true>(f, d, a.z + (int64_t)r * a.ld, a.E, tmp);
        float m = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) m += f[v] * w[v];
        m = row_sum<W>(m, tmp);
        float* o = a.dz + (int64_t)r * a.d_ld;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float s = SC == EXL3_SCORE_SOFTMAX ? f[v] : f[v] * d[v];
            if (l + 64 * W * v < a.E) o[l + 64 * W * v] = s * (w[v] - m);
        }
    }, [&](int r) {
        float* o = a.dz + (int64_t)r * a.d_ld;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (l + 64 * W * v < a.E) o[l + 64 * W * v] = 0.f;
    });
}

typedef void (*balance_fn)(BalanceArgs);

template <int SC>
static balance_fn balance_pick(int E, bool grad) {
#define EXL3_BALANCE(V, W) (grad ? balance_grad_kernel<V, W, SC> : balance_kernel<V, W, SC>)
    return E <= 64 ? EXL3_BALANCE(1, 1) : E <= 128 ? EXL3_BALANCE(2, 1) : E <= 256 ? EXL3_BALANCE(4, 1)
         : E <= 512 ? EXL3_BALANCE(8, 1) : E <= 1024 ? EXL3_BALANCE(16, 1) : E <= 2048 ? EXL3_BALANCE(32, 1)
         : EXL3_BALANCE(32, 4);
#undef EXL3_BALANCE
}
static balance_fn balance_pick(int score, int E, bool grad) {
    return score == EXL3_SCORE_SOFTMAX ? balance_pick<EXL3_SCORE_SOFTMAX>(E, grad)
         : score == EXL3_SCORE_SIGMOID ? balance_pick<EXL3_SCORE_SIGMOID>(E, grad)
         : balance_pick<EXL3_SCORE_SQRT_SOFTPLUS>(E, grad);
}

static int balance_setup(const char* what, const float* logits, int64_t ld, int64_t M, int64_t E, int64_t topk, int score,
                         const uint8_t* mask, float coef, BalanceArgs& a) {
    EXL3_CHECK_ARG(M >= 0 && M <= 0x3FFFFFFF && E > 0 && E <= 8192 && topk > 0 && topk <= E && ld >= E &&
                       M <= 0x7FFFFFFF / topk,
                   "%s: bad sizes (M %lld, E %lld, topk %lld, row stride %lld)", what, (long long)M, (long long)E,
                   (long long)topk, (long long)ld);
    if (score != EXL3_SCORE_SOFTMAX && score != EXL3_SCORE_SIGMOID && score != EXL3_SCORE_SQRT_SOFTPLUS)
        return fail(EXL3_ERR_UNSUPPORTED, "%s: scoring %d not supported", what, score);
    EXL3_CHECK_ARG(M == 0 || logits, "%s: null pointer", what);
    a.z = logits;
    a.ld = ld;
    a.M = (int)M;
    a.E = (int)E;
    a.topk = (int)topk;
    a.mask = mask;
    a.coef = coef;
    return EXL3_OK;
}

// Workgroups of a forward pass, eight rows at a time in each (one of more than 2048 experts): one up to seven rounds of rows, then one
// for every four rounds, up to 480. Not a power of two: a wave's rows would all lie at one place of padded sequences, all
// live or all dead.
static int balance_groups(int64_t M, int64_t E) {
    const int per = E > 2048 ? 1 : 8;
    const int64_t rounds = (M + per - 1) / per;
    return (int)(rounds < 8 ? 1 : rounds / 4 < 480 ? rounds / 4 : 480);
}
static size_t balance_bytes(int G, int64_t E) {
    return carve_size((size_t)G * E, 4) * 2 + carve_size(G, 4) + carve_size((size_t)(E + 15) / 16, 4) + carve_size(1, 4);
}

static int balance(const float* logits, int64_t ld, int64_t M, int64_t E, const int32_t* ids, int64_t topk, const uint8_t* mask,
                   int score, float coef, float* loss, int32_t* counts, float* prob, int32_t* rows, const CallScratch& s,
                   void* stream) {
    hipStream_t st = (hipStream_t)stream;
    BalanceArgs a{};
    int rc = balance_setup("exl3_route_balance", logits, ld, M, E, topk, score, mask, coef, a);
    if (rc) return rc;
    EXL3_CHECK_ARG((M == 0 || ids) && loss && counts && prob && rows, "exl3_route_balance: null pointer");
    a.ids = ids;
    a.loss = loss;
    a.counts = counts;
    a.prob = prob;
    a.rows = rows;
    a.G = balance_groups(M, E);
    if (a.G > 1) {
        const size_t ge = (size_t)a.G * E;
        const int ncb = (int)((E + 15) / 16);
        Carve c{};
        rc = call_scratch("exl3_route_balance", balance_bytes(a.G, E), s, st, &c);
        if (rc) return rc;
        a.part_p = c.take<float>(ge);
        a.part_c = c.take<int32_t>(ge);
        a.part_n = c.take<int32_t>(a.G);
        a.part_l = c.take<float>(ncb);
        a.arrived = c.take<int>(1);
        if (!a.arrived) return fail(EXL3_ERR_INVALID, "exl3_route_balance: workspace carve failed");
    }
    EXL3_LAUNCH("route_balance", balance_pick(score, a.E, false), dim3((unsigned)a.G), dim3(E > 2048 ? 256 : 512),
                (size_t)E * (E > 2048 ? 4 : 8), st, a);
    if (a.G > 1)
        EXL3_LAUNCH("route_balance_reduce", balance_reduce_kernel, dim3((unsigned)((E + 15) / 16)), dim3(256), 0, st, a);
    return EXL3_OK;
}

}  // namespace exl3

extern "C" {

using namespace exl3;

int64_t exl3_route_balance_scratch(int64_t M, int64_t E) {
    if (M < 0 || M > 0x3FFFFFFF || E < 1 || E > 8192) return 0;
    const int G = balance_groups(M, E);
    return G > 1 ? (int64_t)balance_bytes(G, E) : 0;
}

int exl3_route_balance(const float* logits, int64_t ld, int64_t M, int64_t E, const int32_t* ids, int64_t topk,
                       const uint8_t* mask, int score, float coef, float* loss, int32_t* counts, float* prob, int32_t* rows,
                       void* stream) {
    return balance(logits, ld, M, E, ids, topk, mask, score, coef, loss, counts, prob, rows, kLibScratch, stream);
}

int exl3_route_balance_in(const float* logits, int64_t ld, int64_t M, int64_t E, const int32_t* ids, int64_t topk,
                          const uint8_t* mask, int score, float coef, float* loss, int32_t* counts, float* prob, int32_t* rows,
                          void* scratch, int64_t scratch_bytes, void* stream) {
    return balance(logits, ld, M, E, ids, topk, mask, score, coef, loss, counts, prob, rows, CallScratch{scratch, scratch_bytes, false},
                   stream);
}

int exl3_route_balance_grad(const float* logits, int64_t ld, int64_t M, int64_t E, int64_t topk, const uint8_t* mask,
                            int score, float coef, const int32_t* counts, const int32_t* rows, const float* grad,
                            float* dlogits, int64_t d_ld, void* stream) {
    BalanceArgs a{};
    const int rc = balance_setup("exl3_route_balance_grad", logits, ld, M, E, topk, score, mask, coef, a);
    if (rc || M == 0) return rc;
    EXL3_CHECK_ARG(counts && rows && dlogits && d_ld >= E, "exl3_route_balance_grad: null pointer or row stride < E");
    a.counts = const_cast<int32_t*>(counts);
    a.rows = const_cast<int32_t*>(rows);
    a.grad = grad;
    a.dz = dlogits;
    a.d_ld = d_ld;
    const int64_t wgs = E > 2048 ? M : (M + 3) / 4;
    EXL3_LAUNCH("route_balance_grad", balance_pick(score, a.E, true), dim3((unsigned)(wgs < 1920 ? wgs : 1920)), dim3(256), 0,
                (hipStream_t)stream, a);
    return EXL3_OK;
}

}  // extern "C"
