// Decode attention over what a window and a few first positions ("sinks") leave visible, and over 4-bit pools.
//
// The token at position p sees the positions j <= p with j < sinks or j > p - window (window 0: all of them):
//   out_h = sum_j softmax_j(q_h . k_j / sqrt(d)) v_j
// computed in one pass with a running maximum m, sum l and weighted values per head (base 2: exp(x) = 2^(x log2 e)).
//
// Work split.  One (token, KV head, group of <= 8 query heads) is a thread-block cluster: its visible positions are cut
// into tiles (16 positions; 8 of an f32 pool), dealt in turn to the cluster's warps, each with a running state of its
// own; the states are joined through shared memory, then through the cluster's distributed shared memory.  So a launch
// takes nothing but its arguments: no work list, no scratch, no counters.  It can be captured while positions and tables
// change, and launches on several streams share nothing.
//
// Data path.  Every warp has a ring of tiles of its own that its first lane fills with bulk copies, completion on
// mbarriers; nobody waits for another warp until the states are joined.
//
// Arithmetic.  Scores S = Q K^T by mma.sync with the queries as A (8 heads padded to 16 rows: rows 0..7 hold the value
// rounded to the operand type, rows 8..15 the remainder, so one instruction carries both) and the keys as B.  A lane
// then holds head lane / 4 at positions 2 (lane & 3), +1 (and +8, +9), which is how B of O^T = V^T P^T wants the
// probabilities: they go in as value and remainder, in two passes, with no transposition.
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "attn_ptx.cuh"
#include "q4.cuh"

namespace qvx {

extern int* device_status_word(qvx_device* dev);

struct WindowArgs {
    const uint8_t* pool;
    const float* q;
    float* out;
    const uint32_t *pos, *blocks, *table_at;
    uint64_t n_blocks, block_bytes;
    uint32_t page_bytes;        // half of one (block, KV head)'s bytes
    uint32_t pool_blocks, max_pos, window, sinks;
    uint32_t heads, group, groups_per_kv, tiles_per_block;
    float scale_log2;
    int* status;
};

// ---- the cluster ------------------------------------------------------------------------------
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .u32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}" : "=f"(v) : "r"(addr), "r"(rank));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint4 lds128u(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64u(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
// N consecutive 32-bit words (N = 1, 2, 4 or 8).
template <int N>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[N]) {
    if constexpr (N == 1) w[0] = lds32(addr);
    if constexpr (N == 2) { const uint2 v = lds64u(addr); w[0] = v.x; w[1] = v.y; }
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = lds128u(addr + 16 * i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    }
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
// A power of two 2^e that brings values of magnitude up to `most` below 2^(e + 10); 1 for zero, infinities and NaN.
__device__ __forceinline__ int exponent_over(float most) {
    const int e = (int)((__float_as_uint(most) >> 23) & 255u) - 127;  // 2^e <= most < 2^(e + 1)
    return most > 0.f && e < 128 && e > -100 ? e - 9 : 0;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// ---- the tile arithmetic of each element type ----------------------------------------------------
// A Tile type: TP positions per tile; NTL n-tiles of 8 positions; STAGE bytes.  load_q: the lane's query fragments (head
// lane >> 2; zeros for a head the group lacks).  issue: the copies of one tile.  scores: s[2 NTL] of the lane's head at
// positions 2 t, 2 t + 1 (+ 8, + 9), base 2.  values: o += V^T P^T with `p` at the same places; `seen` masks of the
// lane's positions (bit i: p[i]'s position is visible) keep what lies in other slots out of the sums.
// finish: o's values in place, O^T of dimension dim(mt, i) and head 2 t + (i & 1).

// 16-bit pools: the native layout's rows by ldmatrix.
template <int DT, int D>
struct Tile16 {
    static constexpr uint32_t TP = 16, NTL = 2, STAGE = 2 * 16 * D * 2;
    uint32_t q[D / 16][4];
    float o[D / 16][4];
    float back;  // scores x back: undoes the power of two an f16 query row was scaled by

    __device__ __forceinline__ void load_q(const float* row, float scale, uint32_t lane) {
        const uint32_t t = lane & 3u;
        float2 x[D / 16][2];
        float most = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float2 v = row ? make_float2(row[16 * ks + 8 * h + 2 * t], row[16 * ks + 8 * h + 2 * t + 1]) : make_float2(0.f, 0.f);
                v.x *= scale; v.y *= scale;
                x[ks][h] = v;
                most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
        float down = 1.f;
        back = 1.f;
        if constexpr (DT == QVX_F16) {  // f16 overflows at 65504: bring the row's greatest value to 2^9 .. 2^10
            const int e = exponent_over(quad_max(most));
            down = pow2i(-e); back = pow2i(e);
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
            for (int h = 0; h < 2; h++) split16<DT>(x[ks][h].x * down, x[ks][h].y * down, q[ks][2 * h], q[ks][2 * h + 1]);
    }
    __device__ __forceinline__ static void issue(uint32_t stage, const uint8_t* head, uint32_t in_block, uint32_t page, uint32_t bar, uint64_t policy) {
        const uint8_t* k = head + in_block * (16 * D * 2);
        mbar_expect_tx(bar, STAGE);
        if (page == 16 * D * 2) bulk_g2s_hint(stage, k, STAGE, bar, policy);
        else {
            bulk_g2s_hint(stage, k, STAGE / 2, bar, policy);
            bulk_g2s_hint(stage + STAGE / 2, k + page, STAGE / 2, bar, policy);
        }
    }
    __device__ __forceinline__ void scores(uint32_t stage, uint32_t lane, float (&s)[4]) {
        const uint32_t r8 = lane & 7u, mid = lane >> 3, row = r8 + 8 * (mid >> 1), chunk = mid & 1u;
        float c[2][2][4];
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) c[a][b][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++) {
            uint32_t kf[4];
            ldmatrix_x4(stage + row * (D * 2) + (((2 * ks + chunk) ^ (row & 7u)) << 4), kf);
            mma_16816<DT>(c[ks & 1][0], q[ks], kf[0], kf[1]);
            mma_16816<DT>(c[ks & 1][1], q[ks], kf[2], kf[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                s[2 * n + i] = (c[0][n][i] + c[1][n][i]) + (c[0][n][i + 2] + c[1][n][i + 2]);
                if constexpr (DT == QVX_F16) s[2 * n + i] *= back;
            }
    }
    __device__ __forceinline__ void values(uint32_t stage, uint32_t lane, const float (&p)[4], uint32_t seen) {
        const uint32_t r8 = lane & 7u, mid = lane >> 3, row = r8 + 8 * (mid >> 1), chunk = mid & 1u;
        const uint32_t m0 = ((seen & 1u) ? 0xffffu : 0u) | ((seen & 2u) ? 0xffff0000u : 0u);
        const uint32_t m1 = ((seen & 4u) ? 0xffffu : 0u) | ((seen & 8u) ? 0xffff0000u : 0u);
        uint32_t h0, l0, h1, l1;
        split16<DT>(p[0], p[1], h0, l0);
        split16<DT>(p[2], p[3], h1, l1);
#pragma unroll
        for (int mt = 0; mt < D / 16; mt++) {
            uint32_t vf[4];
            ldmatrix_x4_trans(stage + STAGE / 2 + row * (D * 2) + (((2 * mt + chunk) ^ (row & 7u)) << 4), vf);
            vf[0] &= m0; vf[1] &= m0; vf[2] &= m1; vf[3] &= m1;
            mma_16816<DT>(o[mt], vf, h0, h1);
            mma_16816<DT>(o[mt], vf, l0, l1);
        }
    }
    __device__ __forceinline__ void finish(uint32_t) {}
    __device__ __forceinline__ static uint32_t dim(int mt, int i, uint32_t lane) { return 16 * mt + (lane >> 2) + ((i & 2) << 2); }
};

// f32 pools: both operands as a tf32 value and its tf32 remainder (22 bits together).  Tiles of 8 positions.
__device__ __forceinline__ void mma_1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
    // (an infinity or NaN: the remainder inf - inf is NaN, which is what the row's result is to be)
}
template <int D>
struct Tile32 {
    static constexpr uint32_t TP = 8, NTL = 1, STAGE = 2 * 8 * D * 4;
    // Dimensions 4 c .. 4 c + 3 with c = 8 (i >> 1) + 2 t + (i & 1) are the lane's k columns of steps 2 i and 2 i + 1:
    // the order of a product's columns is free, and this one lets a lane read its keys 16 bytes at a time, the eight
    // lanes of a phase on eight different chunks of the swizzled rows.
    float4 q[D / 16];
    float o[D / 16][4];

    __device__ __forceinline__ void load_q(const float* row, float scale, uint32_t lane) {
        const uint32_t t = lane & 3u;
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            const uint32_t at = 4 * (8 * (i >> 1) + 2 * t + (i & 1));
            q[i] = row ? make_float4(row[at] * scale, row[at + 1] * scale, row[at + 2] * scale, row[at + 3] * scale) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ static void issue(uint32_t stage, const uint8_t* head, uint32_t in_block, uint32_t page, uint32_t bar, uint64_t policy) {
        const uint8_t* k = head + in_block * (8 * D * 4);
        mbar_expect_tx(bar, STAGE);
        bulk_g2s_hint(stage, k, STAGE / 2, bar, policy);
        bulk_g2s_hint(stage + STAGE / 2, k + page, STAGE / 2, bar, policy);
    }
    __device__ __forceinline__ void scores(uint32_t stage, uint32_t lane, float (&s)[2]) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            const float4 k = lds128(stage + g * (D * 4) + (((8 * (i >> 1) + 2 * t + (i & 1)) ^ g) << 4));
            uint32_t kh[4], kl[4], a0[4], a1[4];
            split_tf32(k.x, kh[0], kl[0]); split_tf32(k.y, kh[1], kl[1]); split_tf32(k.z, kh[2], kl[2]); split_tf32(k.w, kh[3], kl[3]);
            split_tf32(q[i].x, a0[0], a0[1]); split_tf32(q[i].y, a0[2], a0[3]);
            split_tf32(q[i].z, a1[0], a1[1]); split_tf32(q[i].w, a1[2], a1[3]);
            mma_1688(c[0], a0, kh[0], kh[1]);
            mma_1688(c[1], a1, kh[2], kh[3]);
            mma_1688(c[0], a0, kl[0], kl[1]);
            mma_1688(c[1], a1, kl[2], kl[3]);
        }
        s[0] = (c[0][0] + c[1][0]) + (c[0][2] + c[1][2]);
        s[1] = (c[0][1] + c[1][1]) + (c[0][3] + c[1][3]);
    }
    __device__ __forceinline__ void values(uint32_t stage, uint32_t lane, const float (&p)[2], uint32_t seen) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        uint32_t ph[2], pl[2];
        split_tf32(p[0], ph[0], pl[0]);
        split_tf32(p[1], ph[1], pl[1]);
        const uint32_t m0 = (seen & 1u) ? 0xffffffffu : 0u, m1 = (seen & 2u) ? 0xffffffffu : 0u;
        const uint32_t v0 = stage + STAGE / 2 + 2 * t * (D * 4), v1 = v0 + D * 4;
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            const uint4 x = lds128u(v0 + (((8 * j + g) ^ (2 * t)) << 4)), y = lds128u(v1 + (((8 * j + g) ^ (2 * t + 1)) << 4));
            const float f[8] = {__uint_as_float(x.x & m0), __uint_as_float(x.y & m0), __uint_as_float(x.z & m0), __uint_as_float(x.w & m0),
                                __uint_as_float(y.x & m1), __uint_as_float(y.y & m1), __uint_as_float(y.z & m1), __uint_as_float(y.w & m1)};
            uint32_t h[8], l[8];
#pragma unroll
            for (int e = 0; e < 8; e++) split_tf32(f[e], h[e], l[e]);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t ah[4] = {h[2 * e], h[2 * e + 1], h[4 + 2 * e], h[5 + 2 * e]}, al[4] = {l[2 * e], l[2 * e + 1], l[4 + 2 * e], l[5 + 2 * e]};
                mma_1688(o[2 * j + e], ah, ph[0], ph[1]);
                mma_1688(o[2 * j + e], ah, pl[0], pl[1]);
                mma_1688(o[2 * j + e], al, ph[0], ph[1]);
            }
        }
    }
    __device__ __forceinline__ void finish(uint32_t) {}
    __device__ __forceinline__ static uint32_t dim(int mt, int i, uint32_t lane) { return 32 * (mt >> 1) + 4 * (lane >> 2) + 2 * (mt & 1) + (i >> 1); }
};

// 4-bit pools.  The group's step and offset stay outside the products, so that codes are operands, exactly:
//   score = sum_G s_G (q_G . c_G) + z_G sum(q_G),   out = sum_j p_j s_j (c_j - 8) + sum_j p_j (z_j + 8 s_j),
// the second sum of each a small product of its own; for the values P s_G takes the place of P, group by group, as f16
// value and remainder.  Keys: a code in the low bits of a 16-bit word IS the f16 number c 2^-24, in bits 4..7 it is c 2^-20
// (both subnormal, which the tensor cores multiply exactly): masking alone makes the operand.  Values: the tensor cores
// cut sums off instead of rounding them, and sums of codes that are all >= 0 would grow with the context and carry that
// loss into an output that is the small difference of two of them (1.9e-4 of the result at 20 000 positions); codes
// less 8 and offsets plus 8 steps have no such growth.  Bits 0..3 or 4..7 under f16's 1024 are 1024 + c or 1024 + 16 c,
// and one subtraction, or one multiply-add, makes them c - 8.
template <int D>
struct TileQ4 {
    static constexpr uint32_t TP = 16, NTL = 2, STAGE = 20 * D;
    static constexpr int NG = D / 32;
    uint32_t q[D / 16][4];   // queries x 2^4 in the columns whose codes lie in bits 0..3, as they are in the others
    uint32_t qs[2];          // sums over groups 2 t, 2 t + 1: value, remainder
    float o[D / 16][4];
    float z[4];              // sum p (z + 8 s): row g group g's f16 value, row g + 8 its remainder; heads as o's
    float back;              // undoes the power of two the query row was scaled by
    uint32_t se;             // the greatest step's f16 exponent so far (at least 1); o carries 2^(29 - se)

    __device__ __forceinline__ void load_q(const float* row, float scale, uint32_t lane) {
        const uint32_t t = lane & 3u;
        float x[NG][8], most = 0.f;
#pragma unroll
        for (int G = 0; G < NG; G++)
#pragma unroll
            for (int n = 0; n < 8; n++) {
                x[G][n] = row ? row[32 * G + 8 * t + n] * scale : 0.f;
                most = fmaxf(most, fabsf(x[G][n]));
            }
        const int e = exponent_over(quad_max(most));
        const float down = pow2i(-e);
        back = pow2i(e);
        float sum[NG];
#pragma unroll
        for (int G = 0; G < NG; G++) {
            sum[G] = 0.f;
#pragma unroll
            for (int n = 0; n < 8; n++) { x[G][n] *= down; sum[G] += x[G][n]; }
            sum[G] = quad_sum(sum[G]);
#pragma unroll
            for (int h = 0; h < 2; h++) {  // step 2 G + h: codes 2 h, 2 h + 4 (low nibbles of a byte), then 2 h + 1, 2 h + 5
                split16<QVX_F16>(x[G][2 * h] * 16.f, x[G][2 * h + 4] * 16.f, q[2 * G + h][0], q[2 * G + h][1]);
                split16<QVX_F16>(x[G][2 * h + 1], x[G][2 * h + 5], q[2 * G + h][2], q[2 * G + h][3]);
            }
        }
        qs[0] = qs[1] = 0;
#pragma unroll
        for (int G = 0; G < NG; G += 2)
            if (t == G / 2) split16<QVX_F16>(sum[G], sum[G + 1], qs[0], qs[1]);
#pragma unroll
        for (int i = 0; i < 4; i++) z[i] = 0.f;
        se = 1;
    }
    __device__ __forceinline__ static void issue(uint32_t stage, const uint8_t* head, uint32_t in_block, uint32_t, uint32_t bar, uint64_t policy) {
        mbar_expect_tx(bar, STAGE);
        bulk_g2s_hint(stage, head + in_block * STAGE, STAGE, bar, policy);
    }
    __device__ __forceinline__ void scores(uint32_t stage, uint32_t lane, float (&s)[4]) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        float total[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int n = 0; n < 2; n++) {
            uint32_t w[NG], st[NG];
            lds_words<NG>(stage + (g + 8 * n) * (D / 2) + t * (4 * NG), w);
            lds_words<NG>(stage + 16 * D + (t + 4 * n) * (4 * NG), st);
            float zc[4] = {0.f, 0.f, 0.f, 0.f};
            {
                const uint32_t zk = 2 * t < NG ? lds32(stage + 18 * D + (g + 8 * n) * (2 * NG) + 4 * t) : 0u;
                asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                             : "+f"(zc[0]), "+f"(zc[1]), "+f"(zc[2]), "+f"(zc[3]) : "r"(qs[0]), "r"(qs[1]), "r"(zk));
            }
#pragma unroll
            for (int G = 0; G < NG; G++) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                const uint32_t x = w[G], y = x >> 8;
                mma_16816<QVX_F16>(c, q[2 * G], x & 0x000f000fu, x & 0x00f000f0u);
                mma_16816<QVX_F16>(c, q[2 * G + 1], y & 0x000f000fu, y & 0x00f000f0u);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&st[G]));
                total[n][0] = fmaf(f.x, c[0] + c[2], total[n][0]);
                total[n][1] = fmaf(f.y, c[1] + c[3], total[n][1]);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) s[2 * n + i] = fmaf(total[n][i], 1048576.f, zc[i] + zc[i + 2]) * back;
        }
    }
    __device__ __forceinline__ void values(uint32_t stage, uint32_t lane, const float (&p)[4], uint32_t seen) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        const uint32_t m[2] = {((seen & 1u) ? 0xffffu : 0u) | ((seen & 2u) ? 0xffff0000u : 0u),
                               ((seen & 4u) ? 0xffffu : 0u) | ((seen & 8u) ? 0xffff0000u : 0u)};
        uint32_t st[2][NG], zh[2] = {0u, 0u}, zl[2] = {0u, 0u};
        __half2 top = __float2half2_rn(0.f);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            lds_words<NG>(stage + 17 * D + (t + 4 * n) * (4 * NG), st[n]);
            if (g < NG) {
                const uint32_t at = stage + 17 * D + (t + 4 * n) * (4 * NG) + 4 * g, s2 = lds32(at) & m[n], z2 = lds32(at + 2 * D) & m[n];
                const float2 fs = __half22float2(*reinterpret_cast<const __half2*>(&s2)), fz = __half22float2(*reinterpret_cast<const __half2*>(&z2));
                split16<QVX_F16>(fmaf(8.f, fs.x, fz.x), fmaf(8.f, fs.y, fz.y), zh[n], zl[n]);
            }
#pragma unroll
            for (int G = 0; G < NG; G++) {
                st[n][G] &= m[n];
                const uint32_t a = st[n][G] & 0x7fff7fffu;
                top = __hmax2(top, *reinterpret_cast<const __half2*>(&a));
            }
        }
        // The steps are brought to [.., 2) by the greatest exponent seen so far, so that P s, in f16, keeps 22 bits
        // relative to the greatest of them.
        const uint32_t bits = max((uint32_t)__half_as_ushort(__low2half(top)), (uint32_t)__half_as_ushort(__high2half(top)));
        const uint32_t e = min(__reduce_max_sync(0xffffffffu, bits) >> 10, 30u);
        if (e > se) {
            const float f = pow2i((int)se - (int)e);
#pragma unroll
            for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[mt][i] *= f;
            se = e;
        }
        const __half2 unit = __half2half2(__float2half_rn(pow2i(15 - (int)se)));
        uint32_t ph[2], pl[2];
        split16<QVX_F16>(p[0] * 16384.f, p[1] * 16384.f, ph[0], pl[0]);
        split16<QVX_F16>(p[2] * 16384.f, p[3] * 16384.f, ph[1], pl[1]);
        {
            const uint32_t za[4] = {zh[0], zl[0], zh[1], zl[1]};
            mma_16816<QVX_F16>(z, za, ph[0], ph[1]);
            mma_16816<QVX_F16>(z, za, pl[0], pl[1]);
        }
        // Codes: rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9, the lane's unit of each; a row's words hold two groups each.
        constexpr int NW = NG / 2;
        uint32_t c[4][NW];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t row = t + ((r & 1) << 2) + ((r & 2) << 2);
            lds_words<NW>(stage + 8 * D + row * (D / 2) + (g ^ q4_swap(D, row)) * (2 * NG), c[r]);
        }
#pragma unroll
        for (int G = 0; G < NG; G++) {
            uint32_t bh[2], bl[2];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                // P s = hi + lo: the product of the rounded halves, its error by a fused multiply-add, and the remainder's share.
                const __half2 sn = __hmul2(*reinterpret_cast<const __half2*>(&st[n][G]), unit);
                const __half2 h2 = *reinterpret_cast<const __half2*>(&ph[n]), l2 = *reinterpret_cast<const __half2*>(&pl[n]);
                const __half2 hi = __hmul2(h2, sn);
                const __half2 lo = __hfma2(l2, sn, __hfma2(h2, sn, __hneg2(hi)));
                bh[n] = *reinterpret_cast<const uint32_t*>(&hi);
                bl[n] = *reinterpret_cast<const uint32_t*>(&lo);
            }
            const uint32_t sel = G & 1 ? 0x7632u : 0x5410u;
            const uint32_t x = __byte_perm(c[0][G / 2], c[1][G / 2], sel), y = __byte_perm(c[2][G / 2], c[3][G / 2], sel);
            const uint32_t x8 = x >> 8, y8 = y >> 8;
            const uint32_t a0[4] = {low_code(x), high_code(x), low_code(y), high_code(y)};
            const uint32_t a1[4] = {low_code(x8), high_code(x8), low_code(y8), high_code(y8)};
            mma_16816<QVX_F16>(o[2 * G], a0, bh[0], bh[1]);
            mma_16816<QVX_F16>(o[2 * G], a0, bl[0], bl[1]);
            mma_16816<QVX_F16>(o[2 * G + 1], a1, bh[0], bh[1]);
            mma_16816<QVX_F16>(o[2 * G + 1], a1, bl[0], bl[1]);
        }
    }
    // Codes 0 and 4 (low) or 1 and 5 (high) of a word, less 8, as two f16.
    __device__ __forceinline__ static uint32_t low_code(uint32_t x) {
        const uint32_t h = (x & 0x000f000fu) | 0x64006400u;
        const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(1032.f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ static uint32_t high_code(uint32_t x) {
        const uint32_t h = (x & 0x00f000f0u) | 0x64006400u;
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ void finish(uint32_t lane) {
        // o: the steps came times 2^(15 - se), the probabilities times 2^14.  z: probabilities times 2^14; group G's sums
        // for heads 2 t, 2 t + 1 sit in lane 4 G + t.
        const float u = pow2i((int)se - 15 - 14);
#pragma unroll
        for (int G = 0; G < NG; G++) {
            const float z0 = __shfl_sync(0xffffffffu, z[0] + z[2], 4 * G + (lane & 3u)) * (1.f / 16384.f);
            const float z1 = __shfl_sync(0xffffffffu, z[1] + z[3], 4 * G + (lane & 3u)) * (1.f / 16384.f);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float(&x)[4] = o[2 * G + e];
                x[0] = fmaf(x[0], u, z0); x[1] = fmaf(x[1], u, z1);
                x[2] = fmaf(x[2], u, z0); x[3] = fmaf(x[3], u, z1);
            }
        }
    }
    __device__ __forceinline__ static uint32_t dim(int mt, int i, uint32_t lane) { return 32 * (mt >> 1) + 4 * (lane >> 2) + 2 * (mt & 1) + (i >> 1); }
};

// ---- the kernel ------------------------------------------------------------------------------------
template <class T, int D, int NW, int STAGES>
struct WindowSmem {
    static constexpr uint32_t ring = NW * STAGES * T::STAGE;        // each warp's ring; its state afterwards
    static constexpr uint32_t state = ring;                         // the CTA's joined state [8][D]
    static constexpr uint32_t ml = state + 8 * D * 4;               // [NW + 1][16]: each warp's m[8], l[8], then the CTA's
    static constexpr uint32_t bars = ml + (NW + 1) * 64;
    static constexpr uint32_t bytes = bars + NW * STAGES * 8;
    static_assert(STAGES * T::STAGE >= 8 * D * 4, "a warp's state fits its ring");
};

template <class T, int D, int NW, int STAGES>
__global__ void __launch_bounds__(NW * 32) attn_window_kernel(WindowArgs a) {
    using SM = WindowSmem<T, D, NW, STAGES>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t base = smem_u32(smem), warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t rank = blockIdx.x, ranks = gridDim.x;  // the cluster is the grid's whole x extent
    const uint32_t token = blockIdx.z, kv = blockIdx.y / a.groups_per_kv, sub = blockIdx.y % a.groups_per_kv;
    const uint32_t head0 = kv * a.group + 8 * sub, nheads = min(8u, a.group - 8 * sub);

    const uint32_t p = a.pos[token], ta = a.table_at[token];
    const bool over = p != 0xffffffffu && p > a.max_pos;
    const uint32_t len = p == 0xffffffffu || over ? 0u : p + 1u;
    if (over && rank == 0 && threadIdx.x == 0) atomicExch(a.status, STATUS_POSITION_BOUND);
    // Visible: [0, sink_end) and [win, len).
    uint32_t win = a.window && len > a.window ? len - a.window : 0u, sink_end = min(a.sinks, len);
    if (win <= sink_end) win = sink_end = 0;
    const uint32_t nt = len / T::TP + (len % T::TP != 0), ns = (sink_end + T::TP - 1) / T::TP, w0 = max(win / T::TP, ns);
    const uint32_t tiles = ns + nt - min(w0, nt);
    const uint32_t me = rank * NW + warp, step = ranks * NW;       // this warp takes tiles me, me + step, ...
    const uint32_t mine = tiles > me ? (tiles - me + step - 1) / step : 0u;

    const uint32_t ring = base + warp * (STAGES * T::STAGE), bar = base + SM::bars + warp * (STAGES * 8);
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < STAGES; i++) mbar_init(bar + 8 * i, 1);
        fence_barrier_init();
        fence_proxy_async();
    }
    __syncwarp();
    const uint64_t policy = l2_policy_evict_first();
    auto tile_of = [&](uint32_t i) { const uint32_t j = me + i * step; return j < ns ? j : w0 + (j - ns); };
    // Block ids of 32 of the warp's tiles, one per lane; the next 32 are fetched while these are used.
    auto fetch_id = [&](uint32_t i) {
        if (i >= mine) return 0u;
        const uint64_t at = (uint64_t)ta + tile_of(i) / a.tiles_per_block;
        const uint32_t id = at < a.n_blocks ? a.blocks[at] : 0xffffffffu;
        return id;
    };
    uint32_t ids = fetch_id(lane), ids_next = fetch_id(32 + lane);
    uint32_t bad = 0;  // bit `stage`: that tile's block is not the pool's
    auto issue = [&](uint32_t i, uint32_t stage) {
        if (i != 0 && (i & 31u) == 0) { ids = ids_next; ids_next = fetch_id(i + 32 + lane); }
        uint32_t id = __shfl_sync(0xffffffffu, ids, i & 31u);
        bad &= ~(1u << stage);
        if (id >= a.pool_blocks) { id = 0; bad |= 1u << stage; }  // (nothing of it will be seen; the copy keeps the ring in step)
        if (lane == 0) {
            if (bad >> stage & 1u) atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL);
            T::issue(ring + stage * T::STAGE, a.pool + (uint64_t)id * a.block_bytes + (uint64_t)kv * 2u * a.page_bytes,
                     tile_of(i) % a.tiles_per_block, a.page_bytes, bar + 8 * stage, policy);
        }
    };
    const uint32_t ahead = min((uint32_t)STAGES, mine);
    for (uint32_t i = 0; i < ahead; i++) issue(i, i);

    T w;
    const uint32_t g = lane >> 2, t = lane & 3u;
    w.load_q(g < nheads ? a.q + ((uint64_t)token * a.heads + head0 + g) * D : nullptr, a.scale_log2, lane);
#pragma unroll
    for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
        for (int i = 0; i < 4; i++) w.o[mt][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    uint32_t stage = 0, parity = 0, done = 0;
    for (; done < mine; done++) {
        if (!mbar_wait(bar + 8 * stage, parity)) {
            if (lane == 0) atomicExch(a.status, STATUS_WAIT_TIMEOUT);
            break;
        }
        const uint32_t at = ring + stage * T::STAGE, first = tile_of(done) * T::TP;
        float s[2 * T::NTL];
        w.scores(at, lane, s);
        uint32_t seen = (1u << (2 * T::NTL)) - 1u;
        const bool whole = first + T::TP <= len && (first >= win || first + T::TP <= sink_end) && !(bad >> stage & 1u);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 2 * (int)T::NTL; i++) {
                const uint32_t j = first + 2 * t + (i & 1) + 8 * (i >> 1);
                if (!(j < len && (j < sink_end || j >= win)) || (bad >> stage & 1u)) { s[i] = -INFINITY; seen &= ~(1u << i); }
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 2 * (int)T::NTL; i++) mx = fmaxf(mx, s[i]);
        const float mn = fmaxf(m, quad_max(mx)), ref = mn == -INFINITY ? 0.f : mn;  // (nothing seen yet: every p is 2^-inf = 0)
        const float al = ex2(m - ref);
        m = mn;
        float pr[2 * T::NTL], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * (int)T::NTL; i++) { pr[i] = ex2(s[i] - ref); sum += pr[i]; }
        l = fmaf(l, al, sum);
        if (__any_sync(0xffffffffu, al != 1.f)) {  // (the running maxima settle after the first tiles)
            const float a0 = __shfl_sync(0xffffffffu, al, 8 * t), a1 = __shfl_sync(0xffffffffu, al, 8 * t + 4);
#pragma unroll
            for (int mt = 0; mt < D / 16; mt++) { w.o[mt][0] *= a0; w.o[mt][1] *= a1; w.o[mt][2] *= a0; w.o[mt][3] *= a1; }
            if constexpr (std::is_same<T, TileQ4<D>>::value) { w.z[0] *= a0; w.z[1] *= a1; w.z[2] *= a0; w.z[3] *= a1; }
        }
        w.values(at, lane, pr, seen);
        __syncwarp();  // every lane has read the stage
        if (done + STAGES < mine) issue(done + STAGES, stage);
        if (++stage == STAGES) { stage = 0; parity ^= 1u; }
    }
    // After a wait that ran out: copies still in flight must land before this memory is used for anything else.
    for (uint32_t i = done; i < min(mine, done + STAGES); i++) {
        mbar_wait(bar + 8 * stage, parity);
        if (++stage == STAGES) { stage = 0; parity ^= 1u; }
    }
    w.finish(lane);
    l = quad_sum(l);

    // The warp's state into its own ring, m and l beside.
    float* own = reinterpret_cast<float*>(smem + warp * (STAGES * T::STAGE));
    float* ml = reinterpret_cast<float*>(smem + SM::ml);
    __syncwarp();
#pragma unroll
    for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
        for (int i = 0; i < 4; i++) own[(2 * t + (i & 1)) * D + T::dim(mt, i, lane)] = w.o[mt][i];
    if (t == 0) { ml[warp * 16 + g] = m; ml[warp * 16 + 8 + g] = l; }
    __syncthreads();
    // The CTA's state: its warps' in order.
    float* cta = reinterpret_cast<float*>(smem + SM::state);
    float* out = a.out + ((uint64_t)token * a.heads + head0) * D;
    for (uint32_t e = threadIdx.x; e < 8 * D; e += NW * 32) {
        const uint32_t h = e / D;
        float M = -INFINITY, L = 0.f, x = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) M = fmaxf(M, ml[i * 16 + h]);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const float f = ex2(ml[i * 16 + h] - ref);
            L = fmaf(f, ml[i * 16 + 8 + h], L);
            x = fmaf(f, reinterpret_cast<const float*>(smem + i * (STAGES * T::STAGE))[e], x);
        }
        if (ranks == 1) {
            if (h < nheads && !over) out[e] = len ? x / L : 0.f;
        } else {
            cta[e] = x;
            if (e % D == 0) { ml[NW * 16 + h] = M; ml[NW * 16 + 8 + h] = L; }
        }
    }
    if (ranks == 1) return;
    cluster_sync_all();
    // Every CTA joins its share of the elements over the cluster's states, in rank order.
    for (uint32_t e = rank * (NW * 32) + threadIdx.x; e < nheads * D; e += ranks * (NW * 32)) {
        const uint32_t h = e / D, m_at = base + SM::ml + NW * 64 + 4 * h, x_at = base + SM::state + 4 * e;
        float M = -INFINITY, L = 0.f, x = 0.f;
        for (uint32_t r = 0; r < ranks; r++) M = fmaxf(M, ld_cluster(m_at, r));
        const float ref = M == -INFINITY ? 0.f : M;
        for (uint32_t r = 0; r < ranks; r++) {
            const float f = ex2(ld_cluster(m_at, r) - ref);
            L = fmaf(f, ld_cluster(m_at + 32, r), L);
            x = fmaf(f, ld_cluster(x_at, r), x);
        }
        if (!over) out[e] = len ? x / L : 0.f;
    }
    cluster_sync_all();  // nobody leaves while its shared memory is being read
}

bool attn_window_supported(const Layout& L, size_t heads) {
    if (L.layout != QVX_LAYOUT_NATIVE || L.B % 16 != 0 || heads == 0 || heads % L.kvh != 0) return false;
    return L.d == 64 || L.d == 128 || L.d == 256;
}

template <class T, int D, int NW, int STAGES>
static cudaError_t launch_window(const WindowArgs& a, uint32_t ranks, dim3 grid, cudaStream_t s) {
    auto* kernel = attn_window_kernel<T, D, NW, STAGES>;
    using SM = WindowSmem<T, D, NW, STAGES>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SM::bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = SM::bytes;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

int32_t launch_attn_window(qvx_device* dev, const Layout& L, const void* pool, size_t pool_blocks, size_t heads, size_t s, const float* q,
                           const uint32_t* pos, const uint32_t* blocks, size_t n_blocks, const uint32_t* table_at, uint32_t max_pos,
                           uint32_t window, uint32_t sinks, float* out, cudaStream_t stream) {
    if (s == 0) return QVX_OK;
    const uint32_t tp = L.dtype == QVX_F32 ? 8 : 16;
    WindowArgs a{};
    a.pool = (const uint8_t*)pool; a.q = q; a.out = out; a.pos = pos; a.blocks = blocks; a.table_at = table_at;
    a.n_blocks = n_blocks; a.block_bytes = L.block_bytes; a.page_bytes = L.page_bytes;
    a.pool_blocks = (uint32_t)std::min<size_t>(pool_blocks, 0xffffffffu);
    a.max_pos = max_pos; a.window = window; a.sinks = sinks;
    a.heads = (uint32_t)heads; a.group = (uint32_t)(heads / L.kvh); a.groups_per_kv = (a.group + 7) / 8;
    a.tiles_per_block = L.B / tp;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)L.d));
    a.status = device_status_word(dev);
    // CTAs per cluster: from the most positions a token of this call can see, so that a token's result does not depend
    // on what else is in the batch.
    uint64_t most = (uint64_t)max_pos + 1;
    if (window) most = std::min(most, (uint64_t)window + sinks);
    uint32_t per_cta = 512;
#ifdef QVX_EXPERIMENTS
    if (const char* v = getenv("QVX_WINDOW_PER_CTA")) per_cta = (uint32_t)atol(v);
#endif
    uint32_t ranks = 1;
    while (ranks < 8 && (uint64_t)ranks * per_cta < most) ranks *= 2;
    const dim3 grid(ranks, L.kvh * a.groups_per_kv, (unsigned)s);
    LaunchTimer timer(dev, QVX_K_ATTN, stream);
    cudaError_t e = cudaErrorInvalidValue;
#define QVX_WINDOW(DD)                                                                                             \
    if (L.d == DD) {                                                                                               \
        if (L.dtype == QVX_BF16) e = launch_window<Tile16<QVX_BF16, DD>, DD, 4, DD == 256 ? 2 : 3>(a, ranks, grid, stream); \
        if (L.dtype == QVX_F16) e = launch_window<Tile16<QVX_F16, DD>, DD, 4, DD == 256 ? 2 : 3>(a, ranks, grid, stream);   \
        if (L.dtype == QVX_F32) e = launch_window<Tile32<DD>, DD, 4, DD == 256 ? 2 : 3>(a, ranks, grid, stream);   \
        if (L.dtype == QVX_Q4) e = launch_window<TileQ4<DD>, DD, 4, 4>(a, ranks, grid, stream);                    \
    }
    QVX_WINDOW(64)
    QVX_WINDOW(128)
    QVX_WINDOW(256)
#undef QVX_WINDOW
    return check_cuda(dev, e, "window attention launch");
}

}  // namespace qvx
