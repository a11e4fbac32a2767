// Microscaled 4-bit values (MX4): 32 consecutive values of a row share a scale 2^(s - 127) held in a byte (255: not a
// number); a value is sign, two exponent bits and one mantissa bit (0, .5, 1, 1.5, 2, 3, 4, 6), two to a byte, the even
// one in the low half. A matrix is codes uint8 [rows][k / 2] and scales uint8 [rows][k / 32], both row-major. Every value
// times its scale is exact in bf16 and fp32 for scales to 2^125 (above, 4 2^126 and 2 2^127 are 2^128), and in fp16 for 2^-23 .. 2^13.
//
// The gfx950 conversions take the scale's exponent bits as that byte (the mantissa is not read, exponent 0 is 2^-127),
// round to nearest even and saturate; the scaled MFMAs take the codes as they lie in memory: lane l of a 16 x 16 x 128
// product holds the 32 values (16 bytes, one scale) of row l & 15 that begin at 32 (l >> 4), of a 32 x 32 x 64 one those
// of row l & 31 at 32 (l >> 5). The kernels here use that lane layout for the 16-bit MFMAs too: a lane's block of 32 is
// four (16 x 16 x 32) or four (32 x 32 x 16) fragments of eight, both operands permuted alike along k, so a lane reads
// whole blocks and needs one scale for each.
#pragma once

#include "exl3_device.h"
#include "exl3_runtime.h"

namespace exl3 {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef int i8_t __attribute__((ext_vector_type(8)));

// Workgroups of 256 threads that one launch can have: a dimension of the grid has fewer than 2^32 threads.
constexpr int64_t kMx4Grid = (1 << 24) - 1;

// Type of the rows that a product takes: 16-bit values, or MX4 codes and scales.
enum { kRowF16 = 0, kRowBF16 = 1, kRowMX4 = 2 };

// Scale byte s less the power of two taken out of the matrix (fp16 rows), as the float whose exponent the conversions
// read. A block whose scale leaves 2^-127 .. 2^127 so holds zeros only (the host checks the range); 255 stays 255.
__device__ __forceinline__ float mx4_scale(int s, int base) {
    const int e = s - base;
    return __builtin_bit_cast(float, (s == 255 ? 255 : e < 0 ? 0 : e > 254 ? 254 : e) << 23);
}

// Eight codes (one word) times the scale, as fp16 or bf16.
template <int XT>
__device__ __forceinline__ u32x4_t mx4_frag(uint32_t q, float s) {
    u32x4_t r;
    if constexpr (XT == kRowF16) {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 0));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 1));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 2));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 3));
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3));
    }
    return r;
}

template <int XT>
__device__ __forceinline__ f4_t mfma16(u32x4_t a, u32x4_t b, f4_t c) {
    if constexpr (XT == kRowF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

// 16 x 16 x 128 product of MX4 codes (sa, sb: the lane's scale bytes).
__device__ __forceinline__ f4_t mfma16_mx4(u32x4_t a, int sa, u32x4_t b, int sb, f4_t c) {
    const i8_t av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i8_t bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, sa, 0, sb);
}

// 32 x 32 x 64 product of MX4 codes; byte OP of each lane's scale words.
template <int OP>
__device__ __forceinline__ f16_t mfma32_mx4(u32x4_t a, int sa, u32x4_t b, int sb, f16_t c) {
    const i8_t av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i8_t bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, OP, sa, OP, sb);
}

// Scale bytes [at, at + 16) from p, `left` bytes before the end of the matrix's scales (which are 16 or more, from any row on or
// before p); those past the end are 0. Rows of scales have any alignment.
__device__ __forceinline__ u32x4_t mx4_scales16(const uint8_t* p, int at, int64_t left) {
    typedef u32x4_t any_t __attribute__((aligned(1)));
    const int64_t over = at + 16 - left;
    if (over >= 16) return u32x4_t{};
    const int d = over > 0 ? (int)over : 0;                    // read d bytes earlier, shift them out
    u32x4_t v = *(const __attribute__((address_space(1))) any_t*)(p + at - d);
    if (d) {
        uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
        if (d >= 8) {
            lo = hi >> (8 * (d - 8));
            hi = 0;
        } else {
            lo = lo >> (8 * d) | hi << (64 - 8 * d);
            hi >>= 8 * d;
        }
        v = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
    return v;
}

// Buffer loads of 16 bytes: 0 past the `bytes` from p (which one of fewer than 2^32 - 2^29 may not reach). The whole offset is
// in the vector register: the hardware does not check a scalar one.
constexpr uint32_t kMx4Out = 0xF0000000u;  // an offset past every buffer

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx4_rsrc(const uint8_t* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, (int)(bytes < 0xE0000000LL ? bytes : 0xE0000000LL), 0x00020000);
}
__device__ __forceinline__ u32x4_t mx4_buffer16(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0));
}

// This workgroup's tile of nmt x nnt (rows x columns) and its split of k. Ids go round robin over the 8 XCDs; an XCD takes a
// contiguous run of tiles, a tile's splits and then eight rows of tiles after one another for each column, so that the
// workgroups that run together on it share their columns' and rows' operands in its L2. The grid is the tiles times the
// splits, rounded up to 8; false past them.
__device__ __forceinline__ bool mx4_tile_of(unsigned nmt, unsigned nnt, int splits, unsigned& mt, unsigned& nt, unsigned& sp) {
    const unsigned all = nmt * nnt * splits, per = gridDim.x >> 3, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= all) return false;
    const unsigned t = id / (unsigned)splits;
    sp = id - t * splits;
    const unsigned band = t / (8 * nnt), in = t - band * 8 * nnt, h = nmt - 8 * band < 8 ? nmt - 8 * band : 8;
    nt = in / h;
    mt = 8 * band + in - nt * h;
    return true;
}

__device__ __forceinline__ uint16_t f2bf(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
__device__ __forceinline__ float bf2f(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }

// A value of an output or intermediate of type `dtype` (EXL3_F16, EXL3_F32, EXL3_BF16), one rounding.
__device__ __forceinline__ void store_as(void* p, int64_t i, float v, int dtype) {
    if (dtype == EXL3_F32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = dtype == EXL3_F16 ? f2h(v) : f2bf(v);
}

// Four neighbouring values at an offset that is a multiple of four from a pointer aligned to four values.
__device__ __forceinline__ void store4_as(void* p, int64_t i, f4_t v, int dtype) {
    if (dtype == EXL3_F32) {
        *reinterpret_cast<f4_t*>(reinterpret_cast<float*>(p) + i) = v;
        return;
    }
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = dtype == EXL3_F16 ? f2h(v[j]) : f2bf(v[j]);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// fp16 intermediates with a power of two per group of a row's columns, which is held as v 2^-e. A group whose largest magnitude
// (`top`, float bits) lies in [2^-8, 2^15) stands as it is, e = 0: what falls below fp16's normal range is then off by 2^-17 of the
// largest at most. Any other has its largest value in [2^14, 2^15), zeros the least e. A group with an infinity or a NaN keeps
// them.
__device__ __forceinline__ int mid_exponent(uint32_t top) {
    const int f = (int)(top >> 23) - 127;
    return f >= -8 && f < 15 ? 0 : f - 14 < -126 ? -126 : f - 14;
}
// v 2^d (d <= 0), eight fp16 values: what brings a group to its row's largest exponent (d: its own less that one). fp16 has no
// factor below 2^-24, but the group's largest values stay above its least step down to d = -39.
__device__ __forceinline__ u32x4_t half_times(u32x4_t v, int d) {
    const uint32_t h = d >= -14 ? (uint32_t)(15 + d) << 10 : d >= -24 ? 1u << (24 + d) : 0u, p = h | h << 16;
    u32x4_t r;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        r[q] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, (uint32_t)v[q]) * __builtin_bit_cast(h2_t, p));
    return r;
}
__device__ __forceinline__ u32x4_t half_shift(u32x4_t v, int d) {
    if (d < -24) {
        v = half_times(v, -24);
        d += 24;
    }
    return half_times(v, d);
}
__device__ __forceinline__ uint32_t magnitude_bits(float f) { return __builtin_bit_cast(uint32_t, f) & 0x7FFFFFFFu; }

}  // namespace exl3
