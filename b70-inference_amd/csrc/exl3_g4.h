// 4-bit weights with group scales (G4): w = (q - z) s, whole numbers q and z from 0 to 15 (z = 8 where none are given) and one
// 16-bit scale s, one z for each `group` neighbouring inputs (32, 64 or a multiple of 128). A matrix is codes uint8 [n][k / 2] (two
// q to a byte, the even one in the low half), scales fp16 or bf16 [n][k / group], zeros uint8 [n][k / group].
//
//   y[m, n] = sum over groups G of s[n, G] (sum over k in G of (q - z) x[m, k])
// q - z is exact in 16 bits, so the inner sums are MFMAs over exact operands and the scales multiply fp32 sums: no weight is
// rounded. That is four multiply-adds per 16 x 16 outputs and group, beside the conversion of the weights.
//
// Lane l of a 16 x 16 x 32 product loads 16 bytes, block l >> 4 (32 inputs) of a chunk of 128 inputs of weight row l & 15: 64
// neighbouring bytes of 16 rows. Four swaps then turn the 4 x 4 words of blocks and lane groups, so that product v takes block
// v alone (a group of 32 is one product), the lane its inputs 8 (l >> 4) .. + 7, in the order in which x has them.
//
// The weights are the second operand: a lane's four outputs are four rows m = 4 (l >> 4) + q of one n, whose scale is one register.
#pragma once

#include "exl3_grouped.h"

namespace exl3 {

struct G4Args {
    const uint16_t* x;
    int64_t x_ld;
    const uint8_t* codes;
    const uint16_t* scales;
    const uint8_t* zeros;              // or null
    const float* bias;                 // [n] or null
    void* out;
    int64_t out_ld;
    const int32_t* ends;               // or null: one matrix, all rows
    int E, T;
    int k, n;
    int groups, per;                   // scales of a row; chunks of 128 that share one (groups of 32 and 64: 1)
    int scale_bf16, out_dtype, vec, rest;
    int slots;                         // row blocks of the grid
    // The steps of 128 inputs of the tiles from `whole` on are split over workgroups, `splits` of `spc`. Their sums lie in
    // part [splits][tiles from whole on][part_rows][256].
    int whole, splits, spc, part_rows;
    float* part;
};

// 4 x 4 words of lane groups and blocks turned.
__device__ __forceinline__ void g4_turn(u32x4_t& w) {
    auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w = u32x4_t{c[0], c[1], d[0], d[1]};
}

// What takes a word's codes to q - z: fp16 as -(1024 + z) and -(64 + z); bf16 with zeros as bytes 128 - z.
template <int XT, bool Z>
__device__ __forceinline__ uint32_t g4_zero(int z) {
    if constexpr (XT == kRowF16) return 0xD400E400u + (uint32_t)z * 0x00100001u;
    else return Z ? (uint32_t)(128 - z) * 0x01010101u : 0u;
}
// The factor that g4_frag leaves out: the sums' (a scale's might leave its type).
template <int XT, bool Z>
constexpr float kG4Factor = XT == kRowBF16 && !Z ? 16.f : 1.f;

// The signed 4-bit number in the low bits of byte B, as sixteenths of 16 (the compiler shifts the byte down first, mostly).
template <int B>
__device__ __forceinline__ float g4_off(uint32_t w) {
    float f;
    if constexpr (B == 0) asm("v_cvt_off_f32_i4 %0, %1" : "=v"(f) : "v"(w));
    if constexpr (B == 1) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
    if constexpr (B == 2) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
    if constexpr (B == 3) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
    return f;
}

// x & mask | bits (of two constants the compiler makes two instructions).
__device__ __forceinline__ uint32_t g4_and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(mask), "v"(bits));
    return r;
}

// Eight q - z of a word, exact, in order. fp16: a byte in both halves, of which the lower keeps its low four bits below 1024 and the
// upper its high ones, so that they are 1024 + q and 1024 + 16 q; one multiply-add takes them to q - z. bf16 by way of fp32, where a
// conversion takes signed 4-bit numbers to sixteenths of them (z = 8), or signed bytes.
template <int XT, bool Z>
__device__ __forceinline__ u32x4_t g4_frag(uint32_t w, uint32_t zero) {
    u32x4_t r;
    if constexpr (XT == kRowF16) {
        const h2_t k = {(_Float16)1.f, (_Float16)0.0625f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t p = g4_and_or(__builtin_amdgcn_perm(w, w, 0x00000000u + 0x01010101u * i), 0x00F0000Fu, 0x64006400u);
            r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(h2_t, p), k, __builtin_bit_cast(h2_t, zero)));
        }
    } else if constexpr (!Z) {
        const uint32_t e = w ^ 0x88888888u, o = e >> 4;
        r[0] = __builtin_bit_cast(uint32_t, b2_t{(__bf16)g4_off<0>(e), (__bf16)g4_off<0>(o)});
        r[1] = __builtin_bit_cast(uint32_t, b2_t{(__bf16)g4_off<1>(e), (__bf16)g4_off<1>(o)});
        r[2] = __builtin_bit_cast(uint32_t, b2_t{(__bf16)g4_off<2>(e), (__bf16)g4_off<2>(o)});
        r[3] = __builtin_bit_cast(uint32_t, b2_t{(__bf16)g4_off<3>(e), (__bf16)g4_off<3>(o)});
    } else {
        const uint32_t e = ((w & 0x0F0F0F0Fu) + zero) ^ 0x80808080u, o = ((w >> 4 & 0x0F0F0F0Fu) + zero) ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = __builtin_bit_cast(uint32_t, b2_t{(__bf16)(float)(int8_t)(e >> (8 * i)), (__bf16)(float)(int8_t)(o >> (8 * i))});
    }
    return r;
}

// A scale of either type, or 0 where it is not there (masks: a choice that is alike in all lanes becomes a branch).
__device__ __forceinline__ float g4_scale(uint32_t v, int bf16, bool in = true) {
    const uint32_t m = -(uint32_t)bf16, k = -(uint32_t)in;
    return __builtin_bit_cast(float, ((v << 16 & m) | (__builtin_bit_cast(uint32_t, h2f((uint16_t)v)) & ~m)) & k);
}

// Values that lanes of a wave pass one another through LDS: what was stored or read before is so for all of them. A wave's LDS accesses
// are carried out in order, so this costs no instruction; it keeps the compiler from moving them past one another.
__device__ __forceinline__ void g4_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Block of rows, and its expert's first matrix row: slot s of blocks of BM rows.
template <int BM>
__device__ __forceinline__ GroupSlot g4_slot(const G4Args& g, unsigned slot) {
    if (g.ends) return group_slot<BM>(g.ends, g.E, g.T, slot);
    GroupSlot s;
    s.e = 0;
    s.row = (int64_t)slot * BM;
    s.rows = g.T - s.row < BM ? (int)(g.T - s.row) : BM;
    return s;
}

// Outputs n .. n + 3 of row m.
__device__ __forceinline__ void g4_store4(const G4Args& g, int64_t m, int64_t n, f4_t v) {
    if (n >= g.n) return;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (g.bias && n + q < g.n) v[q] += ldg(g.bias + n + q);
    if (g.vec) {
        store4_as(g.out, m * g.out_ld + n, v, g.out_dtype);
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (n + q < g.n) store_as(g.out, m * g.out_ld + n + q, v[q], g.out_dtype);
}

// tile: 0 few rows, 1, 2, 3 blocks of 32, 64, 128 rows
int g4_run_f16(const G4Args& g, int group, int tile, hipStream_t st);
int g4_run_bf16(const G4Args& g, int group, int tile, hipStream_t st);

}  // namespace exl3
