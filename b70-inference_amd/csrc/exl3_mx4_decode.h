// Products of up to 16 rows with MX4 weights for decode: tiles of 16 weight rows (outputs), k split over the waves of a
// workgroup, x in LDS. Bound by the weights' bytes and, for small matrices, by the latency of one load after another:
// a wave asks for 512 k of its tiles (4 KB of codes and 16 scale bytes per row) at once, the first of them before x is staged,
// the next before the last are multiplied.
//
// Lane l of a 16 x 16 x 32 MFMA (x 16-bit) or 16 x 16 x 128 one (x MX4) holds weight row l & 15 and block l >> 4 of a chunk of
// four blocks: a load takes 64 neighbouring bytes of 16 rows. One MFMA takes a wave as long as the four v_dot2 that it
// replaces at one row, and serves up to 16 rows for it. Reading x from memory instead costs four loads per chunk beside the
// one of the weights, for 16 times the bytes that one row has.
#pragma once

#include "exl3_mx4.h"

namespace exl3 {

constexpr int kMx4Group = 4;           // chunks of 128 k that a wave loads at once

// x in LDS: rows of `stride` bytes, values first (MX4: codes, scales behind all rows' codes)
struct Mx4X {
    char* p;
    int stride, sstride, scales;
};

template <int XT>
__host__ __device__ __forceinline__ int mx4_x_stride(int kb) {
    // whole chunks, and 16 bytes to spread the rows over the banks
    return (kb + 3) / 4 * (XT == kRowMX4 ? 64 : 256) + 16;
}
template <int XT>
__host__ __device__ __forceinline__ int mx4_x_bytes(int rows, int kb) {
    return rows * mx4_x_stride<XT>(kb) + (XT == kRowMX4 ? (rows * ((kb + 3) / 4 * 4 + 4) + 15) / 16 * 16 : 0);
}

// Row i and place u of this thread's elements in one run over rows of `per` elements, a workgroup's threads T apart.
struct Mx4Walk {
    unsigned i, u, per, di, du;
    __device__ __forceinline__ Mx4Walk(unsigned per_, unsigned T) : per(per_) {
        i = threadIdx.x / per;
        u = threadIdx.x - i * per;
        di = T / per;
        du = T - di * per;
    }
    __device__ __forceinline__ void next() {
        i += di;
        u += du;
        if (u >= per) {
            u -= per;
            ++i;
        }
    }
};

// The workgroup copies rows row(0) .. row(rows - 1) (16-byte aligned; MX4: srow their scales) to LDS, zeros past k. All rows'
// units in one run over the threads, eight loads under way: row after row is a round trip to the L2 for each (the routed
// layer's ten rows of 512: 14.1 -> 12.0 us for both launches).
template <int XT, typename Row, typename SRow>
__device__ __forceinline__ Mx4X mx4_stage_x(char* lds, int rows, int kb, Row row, SRow srow) {
    constexpr int kLoads = 8;
    Mx4X x;
    x.p = lds;
    x.stride = mx4_x_stride<XT>(kb);
    x.scales = rows * x.stride;
    x.sstride = (kb + 3) / 4 * 4 + 4;
    const unsigned units = (kb + 3) / 4 * (XT == kRowMX4 ? 4 : 16), have = kb * (XT == kRowMX4 ? 1 : 4), T = blockDim.x;   // of 16 bytes
    if (rows == 1 && XT != kRowMX4) {                          // uniform: no places to work out
        const uint8_t* r = row(0);
        for (unsigned u = threadIdx.x; u < units; u += T)
            *reinterpret_cast<u32x4_t*>(lds + 16 * u) = u < have ? ldg(reinterpret_cast<const u32x4_t*>(r) + u) : u32x4_t{};
        return x;
    }
    Mx4Walk ld(units, T), st = ld;
    for (unsigned u0 = 0; u0 < rows * units; u0 += kLoads * T) {
        u32x4_t v[kLoads];
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
            if (u0 + l * T < rows * units)                     // uniform
                v[l] = ldg(reinterpret_cast<const u32x4_t*>(row(ld.i < (unsigned)rows ? ld.i : rows - 1)) + (ld.u < have ? ld.u : have - 1));
            ld.next();
        }
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
            if (st.i < (unsigned)rows)
                *reinterpret_cast<u32x4_t*>(lds + st.i * x.stride + 16 * st.u) = st.u < have ? v[l] : u32x4_t{};
            st.next();
        }
    }
    if constexpr (XT == kRowMX4) {
        Mx4Walk lb(x.sstride, T), sb = lb;
        for (unsigned b0 = 0; b0 < (unsigned)(rows * x.sstride); b0 += kLoads * T) {
            uint8_t v[kLoads];
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
                if (b0 + l * T < (unsigned)(rows * x.sstride))
                    v[l] = ldg(srow(lb.i < (unsigned)rows ? lb.i : rows - 1) + (lb.u < (unsigned)kb ? lb.u : kb - 1));
                lb.next();
            }
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
                if (sb.i < (unsigned)rows)
                    lds[x.scales + sb.i * x.sstride + sb.u] = sb.u < (unsigned)kb ? (char)v[l] : 0;
                sb.next();
            }
        }
    }
    return x;
}

// A tile: 16 weight rows from n0 of a matrix's `rows`.
struct Mx4Tile16 {
    __amdgpu_buffer_rsrc_t w;          // codes, 0 past the matrix
    const uint8_t* sc;                 // this lane's row's scales
    int64_t sleft;
    __device__ __forceinline__ void set(const uint8_t* codes, const uint8_t* scales, int64_t n0, int64_t rows, int kb, int lane) {
        const int64_t left = rows - n0 < 16 ? rows - n0 : 16, n = n0 + (lane & 15) < rows ? n0 + (lane & 15) : rows - 1;
        w = mx4_rsrc(codes + n0 * kb * 16, left * kb * 16);
        sc = scales + n * kb;
        sleft = (rows - n) * kb;
    }
};

template <int XT>
struct Mx4Decode {
    Mx4Tile16 tile;
    int kb;
    struct Group {
        u32x4_t w[kMx4Group], s;
    };
    __device__ __forceinline__ void load(int gi, int lane, Group& q) const {
        const uint32_t off = (uint32_t)(lane & 15) * (uint32_t)(kb * 16) + 16 * (lane >> 4);
#pragma unroll
        for (int u = 0; u < kMx4Group; ++u) q.w[u] = mx4_buffer16(tile.w, off + 64 * (kMx4Group * gi + u));
        q.s = mx4_scales16(tile.sc, 4 * kMx4Group * gi, tile.sleft);
    }
    // acc += the group's products, the weights times 2^-base; rows: of x (columns past them repeat the last); fx(u, v, word): the
    // eight values of x beside word v of chunk u, as they are multiplied
    __device__ __forceinline__ void mul(int gi, int lane, const Mx4X& x, int rows, int base, Group& q, f4_t& acc) const {
        mul(gi, lane, x, rows, base, q, acc, [](int, int, u32x4_t v) { return v; });
    }
    template <typename F>
    __device__ __forceinline__ void mul(int gi, int lane, const Mx4X& x, int rows, int base, Group& q, f4_t& acc, F fx) const {
        const int g = lane >> 4, r = (lane & 15) < rows ? lane & 15 : rows - 1, left = kb - 4 * kMx4Group * gi;
        if (left < 4 * kMx4Group) {                            // uniform: scale bytes past the row's end are the next row's
#pragma unroll
            for (int u = 0; u < kMx4Group; ++u) {
                const int b = left - 4 * u;
                q.s[u] &= b >= 4 ? ~0u : b > 0 ? (1u << (8 * b)) - 1 : 0u;
            }
        }
#pragma unroll
        for (int u = 0; u < kMx4Group; ++u) {
            if (4 * u >= left) break;                          // uniform
            const int c = kMx4Group * gi + u, sb = (int)(q.s[u] >> (8 * g) & 255);
            if constexpr (XT == kRowMX4) {
                const u32x4_t xv = *reinterpret_cast<const u32x4_t*>(x.p + r * x.stride + 64 * c + 16 * g);
                acc = mfma16_mx4(q.w[u], sb, xv, (uint8_t)x.p[x.scales + r * x.sstride + 4 * c + g], acc);
            } else {
                const u32x4_t* xp = reinterpret_cast<const u32x4_t*>(x.p + r * x.stride + 256 * c + 64 * g);
                const float s = mx4_scale(sb, base);
#pragma unroll
                for (int v = 0; v < 4; ++v) acc = mfma16<XT>(mx4_frag<XT>(q.w[u][v], s), fx(u, v, xp[v]), acc);
            }
        }
    }
};

// Sum over the waves, in order, of tile i's values of lane l (`red`: tiles x waves x 64).
__device__ __forceinline__ f4_t mx4_decode_sum(const f4_t* red, int waves, int i, int l) {
    f4_t s = red[i * waves * 64 + l];
    for (int w = 1; w < waves; ++w) {
        const f4_t t = red[(i * waves + w) * 64 + l];
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += t[q];
    }
    return s;
}

// Waves for `groups` groups of work: as few rounds as `most` waves take, with as few waves as do them.
inline int mx4_decode_waves(int groups, int most) {
    const int rounds = (groups + most - 1) / most;
    return rounds > 0 ? (groups + rounds - 1) / rounds : 1;
}

}  // namespace exl3
