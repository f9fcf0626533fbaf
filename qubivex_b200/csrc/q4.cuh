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

// Byte offsets in a tile of slot r (0..15): the 16-bit half holding codes of dimensions 4 j .. 4 j + 3, and the step
// and the offset of group `grp`.
QVX_HD uint32_t q4_codes_at(uint32_t d, uint32_t r, uint32_t kv, uint32_t j) {
    const uint32_t ng = d / Q4_GROUP, grp = j >> 3, u = j & 7u;
    if (!kv) return r * (d / 2) + ((u >> 1) * ng + grp) * 4 + (u & 1u) * 2;
    const uint32_t row = q4_row(r);
    return 8 * d + row * (d / 2) + ((u ^ q4_swap(d, row)) * ng + grp) * 2;
}
QVX_HD uint32_t q4_step_at(uint32_t d, uint32_t r, uint32_t kv, uint32_t grp) {
    return (kv ? 17 : 16) * d + ((r >> 1) * (d / Q4_GROUP) + grp) * 4 + (r & 1u) * 2;
}
QVX_HD uint32_t q4_offset_at(uint32_t d, uint32_t r, uint32_t kv, uint32_t grp) {
    const uint32_t ng = d / Q4_GROUP;
    return kv ? 19 * d + ((r >> 1) * ng + grp) * 4 + (r & 1u) * 2 : 18 * d + (r * ng + grp) * 2;
}

#if defined(__CUDACC__)
// Eight neighbouring lanes hold a group, four elements each (lane & 7 = the four's place).  All 32 lanes call it.
// Gives the lane's four codes (bits 0..15) and the group's step and offset.
__device__ __forceinline__ uint32_t q4_quantise(float4 x, __half& step, __half& offset) {
    const uint32_t lane = threadIdx.x & 31u;
    float lo = fminf(fminf(x.x, x.y), fminf(x.z, x.w)), hi = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
    // (fminf and fmaxf pass over a NaN; a comparison with one fails)
    const bool fits = fabsf(x.x) <= 65504.f && fabsf(x.y) <= 65504.f && fabsf(x.z) <= 65504.f && fabsf(x.w) <= 65504.f;
#pragma unroll
    for (int w = 1; w < 8; w <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, w));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, w));
    }
    const uint32_t all = __ballot_sync(0xffffffffu, fits) >> (lane & 24u);
    if ((all & 0xffu) != 0xffu) {
        offset = __ushort_as_half(0x7e00); step = __ushort_as_half(0);
        return 0;
    }
    offset = __float2half_rd(lo);
    const float z = __half2float(offset);
    step = __float2half_ru(__fdiv_rn(hi - z, 15.0f));
    const float s = __half2float(step);
    if (!(s > 0.0f)) return 0;
    uint32_t c = 0;
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int n = 0; n < 4; n++) c |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(v[n] - z, s)), 0.0f), 15.0f) << (4 * n);
    return c;
}
#endif

}  // namespace qvx
