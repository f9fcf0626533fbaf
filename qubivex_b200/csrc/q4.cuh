// The 4-bit pool: what an element stands for, and where its bits lie.
//
// The d elements of a key or value row come in groups of 32.  A group holds two f16 values, an offset z and a step
// s >= 0, and a code c of 4 bits per element, which stands for z + s c: 5 bits an element.  From 32 f32 values:
//   z = the least of them rounded down to f16, s = (greatest - z) / 15 rounded up to f16, c = (x - z) / s rounded to
//   the nearest whole number (ties to even) and kept in 0..15; all codes are 0 where s is.
// Rounding z down and s up keeps the whole range within 0..15, so an element is off by at most s / 2.  A group that
// holds a NaN, an infinity or a value beyond f16's range (65504) stands for NaN throughout (z = NaN, s = 0).
//
// Layout: [block][kv head][tile][20 d bytes], a tile being 16 consecutive slots.  It is laid out for the attention
// kernel's lanes (lane 4 g + t of a warp): one bulk copy brings a tile, and every lane finds its matrix fragments'
// codes with one wide load per row and no bank conflicts.  G = d / 32 groups; in a tile:
//   0      keys' codes     [slot][t 0..3][group] words: code n of a word is dimension 32 group + 8 t + n, bits 4n..4n+3
//   8 d    values' codes   [row][unit][group] half words: dimensions 32 group + 4 g + 0..3, bits 4n..4n+3; slot r lies at
//                          row (r & 8) | (r & 1) << 2 | (r >> 1 & 3) and lane group g at unit g ^ q4_swap(row)
//   16 d   keys' steps     [slot pair][group][2] f16
//   17 d   values' steps   [slot pair][group][2] f16
//   18 d   keys' offsets   [slot][group] f16
//   19 d   values' offsets [slot pair][group][2] f16
#pragma once

#include <cuda_fp16.h>

#include "qvx_common.cuh"

namespace qvx {

QVX_HD uint32_t q4_row(uint32_t r) { return (r & 8u) | ((r & 1u) << 2) | ((r >> 1) & 3u); }
QVX_HD uint32_t q4_swap(uint32_t d, uint32_t row) { return d == 128 ? ((row >> 1) & 1u) << 2 : d == 256 ? (row & 3u) << 1 : 0u; }

// Byte offset in a tile of the 16-bit half that holds slot r's codes of dimensions 4 j .. 4 j + 3.
QVX_HD uint32_t q4_codes_at(uint32_t d, uint32_t r, uint32_t kv, uint32_t j) {
    const uint32_t ng = d / Q4_GROUP, grp = j >> 3, u = j & 7u;
    if (!kv) return r * (d / 2) + ((u >> 1) * ng + grp) * 4 + (u & 1u) * 2;
    const uint32_t row = q4_row(r);
    return 8 * d + row * (d / 2) + ((u ^ q4_swap(d, row)) * ng + grp) * 2;
}
#if defined(__CUDACC__)
// Four neighbouring lanes hold a group, eight elements each.  All 32 lanes call it.  Gives the lane's eight codes (code n
// in bits 4 n .. 4 n + 3) and the group's step and offset.
__device__ __forceinline__ uint32_t q4_quantise(const float (&x)[8], __half& step, __half& offset) {
    const uint32_t lane = threadIdx.x & 31u;
    float lo = x[0], hi = x[0], nan = 0.f * x[0];  // (fminf and fmaxf pass over a NaN; 0 x is NaN for one, and for an infinity)
#pragma unroll
    for (int n = 1; n < 8; n++) { lo = fminf(lo, x[n]); hi = fmaxf(hi, x[n]); nan = fmaf(0.f, x[n], nan); }
    const bool fits = nan == 0.f && fmaxf(fabsf(lo), fabsf(hi)) <= 65504.f;
#pragma unroll
    for (int w = 1; w < 4; w <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, w));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, w));
    }
    const uint32_t all = __ballot_sync(0xffffffffu, fits) >> (lane & 28u);
    if ((all & 15u) != 15u) {
        offset = __ushort_as_half(0x7e00); step = __ushort_as_half(0);
        return 0;
    }
    offset = __float2half_rd(lo);
    const float z = __half2float(offset);
    // (hi - z) / 15, rounded to nearest: a quotient within a unit of it, corrected by its exact remainder (Markstein).
    const float range = hi - z, q = range * (1.0f / 15.0f);
    step = __float2half_ru(fmaf(fmaf(-15.0f, q, range), 1.0f / 15.0f, q));
    const float s = __half2float(step);
    if (!(s > 0.0f)) return 0;
    // 0 <= x - z <= 15 s (1 + 2^-22), as z was rounded down and s up: the codes come out within 0..15 by themselves.
    // Adding 1.5 2^23 rounds to the nearest whole number, ties to even, and leaves it in the low bits.  The quotient by way
    // of a reciprocal is off by less than 2^-17; only beside a tie can that change a code, and then the division decides.
    float by, worst = 0.f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(by) : "f"(s));
    constexpr float MAGIC = 12582912.f;
    uint32_t c = 0;
#pragma unroll
    for (int n = 0; n < 8; n++) {
        const float t = (x[n] - z) * by, r = t + MAGIC;
        worst = fmaxf(worst, fabsf(t - (r - MAGIC)));
        c += __float_as_uint(r) << (4 * n);
    }
    if (worst > 0.4999f) {
        c = 0;
#pragma unroll
        for (int n = 0; n < 8; n++) c += __float_as_uint(__fdiv_rn(x[n] - z, s) + MAGIC) << (4 * n);
    }
    return c - 0x4b400000u * 0x11111111u;
}
// Where a lane's eight elements i .. i + 7 (i a multiple of 8) of a row of keys or values lie: what of it does not depend on
// the row, worked out once.  The first lane of a group has its step and offset as well.
template <int D>
struct Q4Place {
    static constexpr uint32_t NG = D / Q4_GROUP;
    uint32_t codes, unit, step, offset, kv;
    bool first;
    __device__ __forceinline__ Q4Place(uint32_t kv, uint32_t i) : kv(kv) {
        const uint32_t grp = i >> 5, u = (i >> 2) & 7u;
        first = (i & 31u) == 0u;
        codes = kv ? 8 * D + grp * 2 : ((u >> 1) * NG + grp) * 4;
        unit = u;
        step = (kv ? 17 : 16) * D + grp * 4;
        offset = kv ? 19 * D + grp * 4 : 18 * D + grp * 2;
    }
    // (values: the next unit of the row lies beside this one, as q4_swap is even)
    __device__ __forceinline__ uint32_t codes_at(uint32_t slot) const {
        if (!kv) return codes + slot * (D / 2);
        const uint32_t row = q4_row(slot);
        return codes + row * (D / 2) + (unit ^ q4_swap(D, row)) * (NG * 2);
    }
    __device__ __forceinline__ uint32_t step_at(uint32_t slot) const { return step + (slot >> 1) * (NG * 4) + (slot & 1u) * 2; }
    __device__ __forceinline__ uint32_t offset_at(uint32_t slot) const {
        return kv ? offset + (slot >> 1) * (NG * 4) + (slot & 1u) * 2 : offset + slot * (NG * 2);
    }
    __device__ __forceinline__ void store(uint8_t* tile, uint32_t slot, uint32_t c, __half s, __half z) const {
        uint8_t* at = tile + codes_at(slot);
        if (!kv) *reinterpret_cast<uint32_t*>(at) = c;
        else {
            *reinterpret_cast<uint16_t*>(at) = (uint16_t)c;
            *reinterpret_cast<uint16_t*>(at + NG * 2) = (uint16_t)(c >> 16);
        }
        if (first) {
            *reinterpret_cast<__half*>(tile + step_at(slot)) = s;
            *reinterpret_cast<__half*>(tile + offset_at(slot)) = z;
        }
    }
};
// 32 bytes at once.
__device__ __forceinline__ void ld_f32x8(float (&x)[8], const float* p) {
    asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "l"(p));
}
__device__ __forceinline__ void st_f32x8(float* p, const float (&x)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]),
                 "f"(x[5]), "f"(x[6]), "f"(x[7]) : "memory");
}
#endif

}  // namespace qvx
