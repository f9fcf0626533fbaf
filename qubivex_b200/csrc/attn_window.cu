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
// Measured (B200, GPU time, of the measured copy bandwidth): bf16, 128 sequences, 64 query heads over 8 of 128, window 4096:
// 308 us, 99 %; bf16, 64 sequences, 32 over 4 of 128, window 1024: 26 us, 80 %; 4 bits, 16 x 32768 positions, 32 over 4 of
// 128: 107 us, 48 %; 4 bits, 64 x 1024-4096 positions: 54 us, 30 %.
//
// Data path.  Every warp has a ring of tiles of its own that its lanes fill in turn with bulk copies, completion on
// mbarriers; nobody waits for another warp until the states are joined.
//
// Arithmetic.  Scores S = Q K^T by mma.sync with the queries as A (8 heads padded to 16 rows: rows 0..7 hold the value
// rounded to the operand type, rows 8..15 the remainder, so one instruction carries both) and the keys as B.  A lane
// then holds head lane / 4 at positions 2 (lane & 3), +1 (and +8, +9), which is how B of O^T = V^T P^T wants the
// probabilities: they go in as value and remainder, in two passes, with no transposition.  (bf16: a third part of both.)
#include <stdlib.h>

#include <algorithm>
#include <mutex>

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
    uint32_t heads, group, groups_per_kv, tiles_per_block, tile_stride;
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
using P2 = unsigned long long;  // two floats in one 64-bit register
__device__ __forceinline__ P2 fma2(P2 a, P2 b, P2 c) {
    P2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ P2 pair_of(float x, float y) {
    P2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ float2 floats_of(P2 p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
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
// A Tile type: TP positions per tile, SUB tiles to a stage of the ring, BYTES per tile; a lane holds PER = TP / 4 scores
// of a tile.  load_q: the lane's query fragments (head lane >> 2; zeros for a head the group lacks).  issue: the copies of
// one tile.  scores: s of the lane's head at positions 2 t, 2 t + 1 (+ 8, + 9) of each tile, base 2.  values:
// o = o alpha + V^T P^T with `p` at the same places; bit i of `seen` says that p[i]'s position is visible: what lies in
// other slots is kept out of the sums.  A tile's products are summed by the tensor cores from zero and added to o in
// f32, rounded: the tensor cores cut sums off, and a long sum kept there would drift with every tile it takes in.
// finish: o's values in place, O^T of dimension dim(mt, i) and head 2 t + (i & 1).
// (No asm here is volatile: a product is a function of its registers, and the compiler may place it where it likes.)
template <int DT>
__device__ __forceinline__ void mma_more(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT == QVX_BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
template <int DT>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const float z = 0.f;
    if constexpr (DT == QVX_BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z));
    }
}
// o = o alpha + x, columns being heads 2 t (alpha a0) and 2 t + 1 (a1).
__device__ __forceinline__ void rescale_add(float (&o)[4], const float (&x)[4], float a0, float a1) {
    o[0] = fmaf(o[0], a0, x[0]); o[1] = fmaf(o[1], a1, x[1]);
    o[2] = fmaf(o[2], a0, x[2]); o[3] = fmaf(o[3], a1, x[3]);
}
// x = hi + lo + third, all bf16: 24 bits, where hi + lo (16 bits) would leave 3e-6 of the result.
__device__ __forceinline__ void split_bf16_3(float x0, float x1, uint32_t& hi, uint32_t& lo, uint32_t& third) {
    split16<QVX_BF16>(x0, x1, hi, lo);
    const float r0 = x0 - __uint_as_float(hi << 16) - __uint_as_float(lo << 16),
                r1 = x1 - __uint_as_float(hi & 0xffff0000u) - __uint_as_float(lo & 0xffff0000u);
    third = pack16<QVX_BF16>(r0, r1);
}

// 16-bit pools: the native layout's rows by ldmatrix.
template <int DT, int D>
struct Tile16 {
    static constexpr uint32_t TP = 16, SUB = 1, PER = 4, BYTES = 2 * 16 * D * 2, Q_SMEM = 0;
    static constexpr float P_LOG2 = 0.f;
    static constexpr bool THIRD = DT == QVX_BF16;
    uint32_t q[D / 16][4];
    uint32_t q3[THIRD ? D / 16 : 1][2];
    float o[D / 16][4];
    float back;  // scores x back: undoes the power of two an f16 query row was scaled by

    __device__ __forceinline__ void load_q(const float* row, float scale, uint32_t lane, uint32_t, uint32_t, uint32_t) {
        const uint32_t t = lane & 3u;
        float2 x[D / 16][2];
        float most = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float2 v = row ? *reinterpret_cast<const float2*>(row + 16 * ks + 8 * h + 2 * t) : make_float2(0.f, 0.f);
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
            for (int h = 0; h < 2; h++) {
                if constexpr (THIRD) split_bf16_3(x[ks][h].x, x[ks][h].y, q[ks][2 * h], q[ks][2 * h + 1], q3[ks][h]);
                else split16<DT>(x[ks][h].x * down, x[ks][h].y * down, q[ks][2 * h], q[ks][2 * h + 1]);
            }
#pragma unroll
        for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[mt][i] = 0.f;
    }
    __device__ __forceinline__ static void issue(uint32_t to, const uint8_t* k, uint32_t page, uint32_t bar, uint64_t policy) {
        if (page == 16 * D * 2) bulk_g2s_hint(to, k, BYTES, bar, policy);
        else {
            bulk_g2s_hint(to, k, BYTES / 2, bar, policy);
            bulk_g2s_hint(to + BYTES / 2, k + page, BYTES / 2, bar, policy);
        }
    }
    __device__ __forceinline__ void scores(uint32_t stage, uint32_t, uint32_t lane, float (&s)[4]) {
        const uint32_t r8 = lane & 7u, mid = lane >> 3, row = r8 + 8 * (mid >> 1), chunk = mid & 1u;
        float c[2][2][4], c3[2][4];
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++) {
            uint32_t kf[4];
            ldmatrix_x4(stage + row * (D * 2) + (((2 * ks + chunk) ^ (row & 7u)) << 4), kf);
            if (ks < 2) {
                mma_first<DT>(c[ks][0], q[ks], kf[0], kf[1]);
                mma_first<DT>(c[ks][1], q[ks], kf[2], kf[3]);
            } else {
                mma_more<DT>(c[ks & 1][0], q[ks], kf[0], kf[1]);
                mma_more<DT>(c[ks & 1][1], q[ks], kf[2], kf[3]);
            }
            if constexpr (THIRD) {
                const uint32_t a[4] = {q3[ks][0], 0u, q3[ks][1], 0u};
                if (ks == 0) { mma_first<DT>(c3[0], a, kf[0], kf[1]); mma_first<DT>(c3[1], a, kf[2], kf[3]); }
                else { mma_more<DT>(c3[0], a, kf[0], kf[1]); mma_more<DT>(c3[1], a, kf[2], kf[3]); }
            }
        }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float small = c[0][n][i + 2] + c[1][n][i + 2];
                if constexpr (THIRD) small += c3[n][i];
                s[2 * n + i] = (c[0][n][i] + c[1][n][i]) + small;
            }
    }
    __device__ __forceinline__ void values(uint32_t stage, uint32_t lane, const float (&p)[4], uint32_t seen, float a0, float a1) {
        const uint32_t r8 = lane & 7u, mid = lane >> 3, row = r8 + 8 * (mid >> 1), chunk = mid & 1u;
        const uint32_t m0 = ((seen & 1u) ? 0xffffu : 0u) | ((seen & 2u) ? 0xffff0000u : 0u);
        const uint32_t m1 = ((seen & 4u) ? 0xffffu : 0u) | ((seen & 8u) ? 0xffff0000u : 0u);
        uint32_t h0, l0, h1, l1, t0, t1;
        if constexpr (THIRD) { split_bf16_3(p[0], p[1], h0, l0, t0); split_bf16_3(p[2], p[3], h1, l1, t1); }
        else { split16<DT>(p[0], p[1], h0, l0); split16<DT>(p[2], p[3], h1, l1); }
#pragma unroll
        for (int mt = 0; mt < D / 16; mt++) {
            uint32_t vf[4];
            ldmatrix_x4_trans(stage + BYTES / 2 + row * (D * 2) + (((2 * mt + chunk) ^ (row & 7u)) << 4), vf);
            vf[0] &= m0; vf[1] &= m0; vf[2] &= m1; vf[3] &= m1;
            float x[4];
            if constexpr (THIRD) { mma_first<DT>(x, vf, t0, t1); mma_more<DT>(x, vf, l0, l1); }
            else mma_first<DT>(x, vf, l0, l1);
            mma_more<DT>(x, vf, h0, h1);
            rescale_add(o[mt], x, a0, a1);
        }
    }
    __device__ __forceinline__ void finish(uint32_t) {}
    __device__ __forceinline__ static uint32_t dim(int mt, int i, uint32_t lane) { return 16 * mt + (lane >> 2) + ((i & 2) << 2); }
};

// f32 pools: both operands as a tf32 value and its tf32 remainder (22 bits together).  Tiles of 8 positions.
__device__ __forceinline__ void mma_1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The value is rounded to tf32 (half a unit added below its 11 bits, the rest cut), so that the remainder takes either
// sign and what the products leave out does not add up.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
template <int D>
struct Tile32 {
    static constexpr uint32_t TP = 8, SUB = 1, PER = 2, BYTES = 2 * 8 * D * 4, Q_SMEM = 0;
    static constexpr float P_LOG2 = 0.f;
    // Dimensions 4 c .. 4 c + 3 with c = 8 (i >> 1) + 2 t + (i & 1) are the lane's k columns of steps 2 i and 2 i + 1:
    // the order of a product's columns is free, and this one lets a lane read its keys 16 bytes at a time, the eight
    // lanes of a phase on eight different chunks of the swizzled rows.
    float4 q[D / 16];
    float o[D / 16][4];
    static constexpr float back = 1.f;

    __device__ __forceinline__ void load_q(const float* row, float scale, uint32_t lane, uint32_t, uint32_t, uint32_t) {
        const uint32_t t = lane & 3u;
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            const uint32_t at = 4 * (8 * (i >> 1) + 2 * t + (i & 1));
            const float4 v = row ? *reinterpret_cast<const float4*>(row + at) : make_float4(0.f, 0.f, 0.f, 0.f);
            q[i] = make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
        }
#pragma unroll
        for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[mt][i] = 0.f;
    }
    __device__ __forceinline__ static void issue(uint32_t to, const uint8_t* k, uint32_t page, uint32_t bar, uint64_t policy) {
        bulk_g2s_hint(to, k, BYTES / 2, bar, policy);
        bulk_g2s_hint(to + BYTES / 2, k + page, BYTES / 2, bar, policy);
    }
    __device__ __forceinline__ void scores(uint32_t stage, uint32_t, uint32_t lane, float (&s)[2]) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            const float4 k = lds128(stage + g * (D * 4) + (((8 * (i >> 1) + 2 * t + (i & 1)) ^ g) << 4));
            uint32_t kh[4], kl[4], a0[4], a1[4];
            split_tf32(k.x, kh[0], kl[0]); split_tf32(k.y, kh[1], kl[1]); split_tf32(k.z, kh[2], kl[2]); split_tf32(k.w, kh[3], kl[3]);
            split_tf32(q[i].x, a0[0], a0[1]); split_tf32(q[i].y, a0[2], a0[3]);
            split_tf32(q[i].z, a1[0], a1[1]); split_tf32(q[i].w, a1[2], a1[3]);
            mma_1688(c[0], a0, kl[0], kl[1]);
            mma_1688(c[1], a1, kl[2], kl[3]);
            mma_1688(c[0], a0, kh[0], kh[1]);
            mma_1688(c[1], a1, kh[2], kh[3]);
        }
        s[0] = (c[0][0] + c[1][0]) + (c[0][2] + c[1][2]);
        s[1] = (c[0][1] + c[1][1]) + (c[0][3] + c[1][3]);
    }
    __device__ __forceinline__ void values(uint32_t stage, uint32_t lane, const float (&p)[2], uint32_t seen, float a0, float a1) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        uint32_t ph[2], pl[2];
        split_tf32(p[0], ph[0], pl[0]);
        split_tf32(p[1], ph[1], pl[1]);
        const uint32_t m0 = (seen & 1u) ? 0xffffffffu : 0u, m1 = (seen & 2u) ? 0xffffffffu : 0u;
        const uint32_t v0 = stage + BYTES / 2 + 2 * t * (D * 4), v1 = v0 + D * 4;
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
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
                mma_1688(acc, ah, pl[0], pl[1]);
                mma_1688(acc, al, ph[0], ph[1]);
                mma_1688(acc, ah, ph[0], ph[1]);
                rescale_add(o[2 * j + e], acc, a0, a1);
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
// (both subnormal, which the tensor cores multiply exactly): masking alone makes the operand.  Values: sums of codes that
// are all >= 0 would grow with the context and lose to f32's rounding what the output, the small difference of two of
// them, is made of (1.9e-4 of the result at 20 000 positions); codes less 8 and offsets plus 8 steps have no such
// growth.  Bits 0..3 or 4..7 under f16's 1024 are 1024 + c or 1024 + 16 c, and one subtraction, or one multiply-add, makes
// them c - 8.
// A stage is two tiles: what is done once per stage (maxima, the ring's upkeep) is shared, and two tiles' chains of
// dependent products run beside each other.  The queries' fragments stay in shared memory, 32 registers less.
// Bound by instructions, not by memory: about 480 a tile of 2560 bytes (d = 128), of which the masks and byte
// permutations and the half-precision arithmetic go at half rate and a 16 x 8 x 16 product takes 8 cycles beside which
// little else issues; 250 cycles a tile and SM where HBM asks for 111.  12 warps an SM without spills do more than 16 with
// 76 bytes of them (107 us against 117 for 16 x 32768 positions, 32 over 4 heads), and two stages a warp as much as three.
template <int D>
struct TileQ4 {
    static constexpr uint32_t TP = 16, SUB = 2, PER = 4, BYTES = 20 * D, Q_SMEM = D * 32;
    static constexpr float P_LOG2 = 14.f;
    static constexpr int NG = D / 32;
    uint32_t qs[2];          // query sums over groups 2 t, 2 t + 1: value, remainder
    float o[D / 16][4];
    float z[4];              // sum p (z + 8 s): row g group g's f16 value, row g + 8 its remainder; heads as o's
    float back;              // undoes the power of two the query row was scaled by
    uint32_t se;             // the greatest step's f16 exponent so far, 15 (steps below 2) or more; o carries 2^(15 - se)

    // Fragments at q_at + (step * 32 + lane) * 16, the steps shared out over the CTA's warps (a __syncthreads follows):
    // queries x 2^4 in the columns whose codes lie in bits 0..3, as they are in the others.
    __device__ __forceinline__ void load_q(const float* row, float scale, uint32_t lane, uint32_t q_at, uint32_t warp, uint32_t warps) {
        const uint32_t t = lane & 3u;
        float x[NG][8], most = 0.f;
#pragma unroll
        for (int G = 0; G < NG; G++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float4 v = row ? *reinterpret_cast<const float4*>(row + 32 * G + 8 * t + 4 * h) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[G][4 * h] = v.x * scale; x[G][4 * h + 1] = v.y * scale; x[G][4 * h + 2] = v.z * scale; x[G][4 * h + 3] = v.w * scale;
#pragma unroll
                for (int n = 0; n < 4; n++) most = fmaxf(most, fabsf(x[G][4 * h + n]));
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
            if (G % warps != warp) continue;
#pragma unroll
            for (int h = 0; h < 2; h++) {  // step 2 G + h: codes 2 h, 2 h + 4 (low nibbles of a byte), then 2 h + 1, 2 h + 5
                uint32_t f[4];
                split16<QVX_F16>(x[G][2 * h] * 16.f, x[G][2 * h + 4] * 16.f, f[0], f[1]);
                split16<QVX_F16>(x[G][2 * h + 1], x[G][2 * h + 5], f[2], f[3]);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_at + ((2 * G + h) * 32 + lane) * 16), "r"(f[0]), "r"(f[1]), "r"(f[2]), "r"(f[3]) : "memory");
            }
        }
        qs[0] = qs[1] = 0;
#pragma unroll
        for (int G = 0; G < NG; G += 2)
            if (t == G / 2) split16<QVX_F16>(sum[G], sum[G + 1], qs[0], qs[1]);
#pragma unroll
        for (int i = 0; i < 4; i++) z[i] = 0.f;
#pragma unroll
        for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[mt][i] = 0.f;
        se = 15;
    }
    __device__ __forceinline__ static void issue(uint32_t to, const uint8_t* tile, uint32_t, uint32_t bar, uint64_t policy) {
        bulk_g2s_hint(to, tile, BYTES, bar, policy);
    }
    __device__ __forceinline__ void scores(uint32_t stage, uint32_t q_at, uint32_t lane, float (&s)[8]) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        P2 total[4] = {0ull, 0ull, 0ull, 0ull};
        float zc[4][4];
        uint32_t w[4][NG], st[4][NG];
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const uint32_t tile = stage + (n >> 1) * BYTES, h = n & 1;
            lds_words<NG>(tile + (g + 8 * h) * (D / 2) + t * (4 * NG), w[n]);
            lds_words<NG>(tile + 16 * D + (t + 4 * h) * (4 * NG), st[n]);
            const uint32_t zk = 2 * t < NG ? lds32(tile + 18 * D + (g + 8 * h) * (2 * NG) + 4 * t) : 0u;
            asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                         : "=f"(zc[n][0]), "=f"(zc[n][1]), "=f"(zc[n][2]), "=f"(zc[n][3]) : "r"(qs[0]), "r"(qs[1]), "r"(zk), "f"(0.f));
        }
#pragma unroll
        for (int G = 0; G < NG; G++) {
            uint32_t q0[4], q1[4];
            lds_words<4>(q_at + (2 * G * 32 + lane) * 16, q0);
            lds_words<4>(q_at + ((2 * G + 1) * 32 + lane) * 16, q1);
#pragma unroll
            for (int n = 0; n < 4; n++) {
                float c[4];
                const uint32_t x = w[n][G], y = x >> 8;
                mma_first<QVX_F16>(c, q0, x & 0x000f000fu, x & 0x00f000f0u);
                mma_more<QVX_F16>(c, q1, y & 0x000f000fu, y & 0x00f000f0u);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&st[n][G]));
                const P2 step = pair_of(f.x, f.y);
                total[n] = fma2(step, pair_of(c[0], c[1]), total[n]);
                total[n] = fma2(step, pair_of(c[2], c[3]), total[n]);
            }
        }
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const float2 f = floats_of(total[n]);
            s[2 * n] = fmaf(f.x, 1048576.f, zc[n][0] + zc[n][2]);
            s[2 * n + 1] = fmaf(f.y, 1048576.f, zc[n][1] + zc[n][3]);
        }
    }
    __device__ __forceinline__ void values(uint32_t stage, uint32_t lane, const float (&p)[8], uint32_t seen, float a0, float a1) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        uint32_t st[4][NG], s2[4], z2[4];
        uint32_t any = 0;
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const uint32_t tile = stage + (n >> 1) * BYTES, pair = (t + 4 * (n & 1)) * (4 * NG);
            lds_words<NG>(tile + 17 * D + pair, st[n]);
            s2[n] = z2[n] = 0;
            if (g < NG) { s2[n] = lds32(tile + 17 * D + pair + 4 * g); z2[n] = lds32(tile + 19 * D + pair + 4 * g); }
            if (seen != 255u) {
                const uint32_t b = seen >> (2 * n), m = ((b & 1u) ? 0xffffu : 0u) | ((b & 2u) ? 0xffff0000u : 0u);
                s2[n] &= m; z2[n] &= m;
#pragma unroll
                for (int G = 0; G < NG; G++) st[n][G] &= m;
            }
#pragma unroll
            for (int G = 0; G < NG; G++) any |= st[n][G];
        }
        // P s in f16, the weights times 2^14: up to 2^15 while the steps are below 2, and 22 bits of the greatest of them are
        // kept down to steps of f16's least normal numbers.  Greater steps (bit 14, the exponent's highest, set) are brought
        // below 2 by a power of two of their own, that of the greatest seen so far.
        float b0 = a0, b1 = a1;
        const bool large = __any_sync(0xffffffffu, (any & 0x40004000u) != 0) || se > 15;
        if (large) {
            __half2 top = __float2half2_rn(0.f);
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int G = 0; G < NG; G++) { const uint32_t v = st[n][G] & 0x7fff7fffu; top = __hmax2(top, *reinterpret_cast<const __half2*>(&v)); }
            const uint32_t bits = max((uint32_t)__half_as_ushort(__low2half(top)), (uint32_t)__half_as_ushort(__high2half(top)));
            const uint32_t e = min(__reduce_max_sync(0xffffffffu, bits) >> 10, 30u);
            if (e > se) {
                const float f = pow2i((int)se - (int)e);
                b0 *= f; b1 *= f;
                se = e;
            }
        }
        // z + 8 s = zh + zl.
        uint32_t zh[4], zl[4];
        if (large) {
            const __half2 unit = __half2half2(__float2half_rn(pow2i(15 - (int)se)));
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float2 fs = __half22float2(*reinterpret_cast<const __half2*>(&s2[n])), fz = __half22float2(*reinterpret_cast<const __half2*>(&z2[n]));
                split16<QVX_F16>(fmaf(8.f, fs.x, fz.x), fmaf(8.f, fs.y, fz.y), zh[n], zl[n]);
#pragma unroll
                for (int G = 0; G < NG; G++) {
                    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&st[n][G]), unit);
                    st[n][G] = *reinterpret_cast<const uint32_t*>(&x);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < 4; n++) {  // (8 s stays in f16's range: the error of one addition, in f16, is exact)
                const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&s2[n]), __float2half2_rn(8.f)), y = *reinterpret_cast<const __half2*>(&z2[n]);
                const __half2 hi = __hadd2(x, y), v = __hsub2(hi, x);
                const __half2 lo = __hadd2(__hsub2(x, __hsub2(hi, v)), __hsub2(y, v));
                zh[n] = *reinterpret_cast<const uint32_t*>(&hi);
                zl[n] = *reinterpret_cast<const uint32_t*>(&lo);
            }
        }
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int n = 0; n < 4; n++) split16<QVX_F16>(p[2 * n], p[2 * n + 1], ph[n], pl[n]);
        {
            const uint32_t za[4] = {zh[0], zl[0], zh[1], zl[1]}, zb[4] = {zh[2], zl[2], zh[3], zl[3]};
            float x[4];
            mma_first<QVX_F16>(x, za, pl[0], pl[1]);
            mma_more<QVX_F16>(x, zb, pl[2], pl[3]);
            mma_more<QVX_F16>(x, za, ph[0], ph[1]);
            mma_more<QVX_F16>(x, zb, ph[2], ph[3]);
            rescale_add(z, x, a0, a1);
        }
        // Codes: rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of each tile, the lane's unit of each; a row's words hold two groups each.
        constexpr int NW = NG / 2;
        uint32_t c[2][4][NW];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t row = t + ((r & 1) << 2) + ((r & 2) << 2);
                lds_words<NW>(stage + i * BYTES + 8 * D + row * (D / 2) + (g ^ q4_swap(D, row)) * (2 * NG), c[i][r]);
            }
#pragma unroll
        for (int G = 0; G < NG; G++) {
            uint32_t bh[4], bl[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                // P s = hi + lo: the product of the rounded halves, its error by a fused multiply-add, and the remainder's share.
                const __half2 sn = *reinterpret_cast<const __half2*>(&st[n][G]), h2 = *reinterpret_cast<const __half2*>(&ph[n]), l2 = *reinterpret_cast<const __half2*>(&pl[n]);
                const __half2 hi = __hmul2(h2, sn);
                const __half2 lo = __hfma2(l2, sn, __hfma2(h2, sn, __hneg2(hi)));
                bh[n] = *reinterpret_cast<const uint32_t*>(&hi);
                bl[n] = *reinterpret_cast<const uint32_t*>(&lo);
            }
            const uint32_t sel = G & 1 ? 0x7632u : 0x5410u;
            float x0[4], x1[4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t x = __byte_perm(c[i][0][G / 2], c[i][1][G / 2], sel), y = __byte_perm(c[i][2][G / 2], c[i][3][G / 2], sel);
                const uint32_t x8 = x >> 8, y8 = y >> 8;
                const uint32_t v0[4] = {low_code(x), high_code(x), low_code(y), high_code(y)};
                const uint32_t v1[4] = {low_code(x8), high_code(x8), low_code(y8), high_code(y8)};
                if (i == 0) { mma_first<QVX_F16>(x0, v0, bl[0], bl[1]); mma_first<QVX_F16>(x1, v1, bl[0], bl[1]); }
                else { mma_more<QVX_F16>(x0, v0, bl[2], bl[3]); mma_more<QVX_F16>(x1, v1, bl[2], bl[3]); }
                mma_more<QVX_F16>(x0, v0, bh[2 * i], bh[2 * i + 1]);
                mma_more<QVX_F16>(x1, v1, bh[2 * i], bh[2 * i + 1]);
            }
            rescale_add(o[2 * G], x0, b0, b1);
            rescale_add(o[2 * G + 1], x1, b0, b1);
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
        // o: the steps came times 2^(15 - se).  z: group G's sums for heads 2 t, 2 t + 1 sit in lane 4 G + t.
        const float u = pow2i((int)se - 15);
#pragma unroll
        for (int G = 0; G < NG; G++) {
            const float z0 = __shfl_sync(0xffffffffu, z[0] + z[2], 4 * G + (lane & 3u));
            const float z1 = __shfl_sync(0xffffffffu, z[1] + z[3], 4 * G + (lane & 3u));
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
    static constexpr uint32_t stage = T::SUB * T::BYTES;
    static constexpr uint32_t ring = STAGES * stage;                // one warp's ring; its state afterwards
    static constexpr uint32_t state = NW * ring;                    // the CTA's joined state [8][D]
    static constexpr uint32_t q = state + 8 * D * 4;                // query fragments, where the type keeps them here
    static constexpr uint32_t ml = q + T::Q_SMEM;                   // [NW + 1][16]: each warp's m[8], l[8], then the CTA's
    static constexpr uint32_t bars = ml + (NW + 1) * 64;
    static constexpr uint32_t bytes = bars + NW * STAGES * 8;
    static_assert(ring >= 8 * D * 4, "a warp's state fits its ring");
};

template <class T, int D, int NW, int STAGES, int MIN_CTAS>
__global__ void __launch_bounds__(NW * 32, MIN_CTAS) attn_window_kernel(WindowArgs a) {
    using SM = WindowSmem<T, D, NW, STAGES>;
    constexpr uint32_t PER = T::PER, N = T::SUB * PER;
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
    const uint32_t rounds = (mine + T::SUB - 1) / T::SUB;

    const uint32_t ring = base + warp * SM::ring, bar = base + SM::bars + warp * (STAGES * 8);
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < STAGES; i++) mbar_init(bar + 8 * i, 1);
        fence_barrier_init();
        fence_proxy_async();
    }
    __syncwarp();
    const uint64_t policy = l2_policy_evict_first();
    // Of the warp's tiles, plain_from .. plain_upto - 1 are visible to the last position: those between the tile the window
    // begins in and the tile the sequence ends in (the sinks' are few and looked at).
    const uint32_t wide_from = ns + (win > w0 * T::TP ? 1u : 0u), wide_upto = tiles - (len % T::TP != 0 && tiles > 0 ? 1u : 0u);
    const uint32_t plain_from = wide_from > me ? (wide_from - me + step - 1) / step : 0u, plain_upto = wide_upto > me ? (wide_upto - me + step - 1) / step : 0u;
    auto tile_of = [&](uint32_t i) { const uint32_t j = me + i * step; return j < ns ? j : w0 + (j - ns); };
    // Lane i mod 32 looks up where the warp's i-th tile lies and issues its copy; the next 32 tiles' block ids are on their
    // way while these are in use.  An id that is not the pool's is noted in `foreign`: the copy then brings the pool's first
    // block in its place (it keeps the ring in step, and nothing of it will be seen).
    auto fetch_id = [&](uint32_t i) -> uint32_t {
        if (i >= mine) return 0u;
        const uint64_t at = (uint64_t)ta + tile_of(i) / a.tiles_per_block;
        return at < a.n_blocks ? a.blocks[at] : 0xffffffffu;
    };
    const uint8_t* src = nullptr;
    uint32_t ids_next = fetch_id(lane), foreign = 0, foreign_before = 0;
    auto next_batch = [&](uint32_t i0) {  // tiles i0 .. i0 + 31
        const uint32_t id = ids_next;
        ids_next = fetch_id(i0 + 32 + lane);
        foreign_before = foreign;
        foreign = __ballot_sync(0xffffffffu, id >= a.pool_blocks);
        if (id >= a.pool_blocks) atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL);
        src = a.pool + (uint64_t)(id < a.pool_blocks ? id : 0u) * a.block_bytes + (uint64_t)kv * 2u * a.page_bytes +
              (tile_of(i0 + lane) % a.tiles_per_block) * a.tile_stride;
    };
    // A stage's tiles: r * SUB .. (the last may lack some).
    auto issue = [&](uint32_t r, uint32_t stage) {
        const uint32_t i0 = r * T::SUB;
        if ((i0 & 31u) == 0) next_batch(i0);
        const uint32_t have = min((uint32_t)T::SUB, mine - i0), k = lane - (i0 & 31u);
        if (k == 0) mbar_expect_tx(bar + 8 * stage, have * T::BYTES);
        __syncwarp();
        if (k < have) T::issue(ring + stage * SM::stage + k * T::BYTES, src, a.page_bytes, bar + 8 * stage, policy);
    };
    const uint32_t ahead = min((uint32_t)STAGES, rounds);
    for (uint32_t i = 0; i < ahead; i++) issue(i, i);

    T w;
    const uint32_t g = lane >> 2, t = lane & 3u;
    w.load_q(g < nheads ? a.q + ((uint64_t)token * a.heads + head0 + g) * D : nullptr, a.scale_log2, lane, base + SM::q, warp, NW);
    if constexpr (T::Q_SMEM != 0) __syncthreads();
    float m = -INFINITY, l = 0.f;

    uint32_t stage = 0, parity = 0, done = 0;
    for (; done < rounds; done++) {
        if (!mbar_wait(bar + 8 * stage, parity)) {
            if (lane == 0) atomicExch(a.status, STATUS_WAIT_TIMEOUT);
            break;
        }
        const uint32_t at = ring + stage * SM::stage;
        float s[N];
        w.scores(at, base + SM::q, lane, s);
        uint32_t seen = (1u << N) - 1u;
        if (done * T::SUB < plain_from || (done + 1) * T::SUB > plain_upto || (foreign | foreign_before) != 0) {
            // (issuing runs at most one batch of 32 ids ahead of this)
            const uint32_t issued = min((done + STAGES) * T::SUB - 1u, (rounds - 1u) * T::SUB);
#pragma unroll
            for (int u = 0; u < (int)T::SUB; u++) {
                const uint32_t i = done * T::SUB + u, first = tile_of(i) * T::TP;
                const bool alien = ((i >> 5) == (issued >> 5) ? foreign : foreign_before) >> (i & 31u) & 1u;
#pragma unroll
                for (int k = 0; k < (int)PER; k++) {
                    const uint32_t j = first + 2 * t + (k & 1) + 8 * (k >> 1);
                    if (i >= mine || alien || !(j < len && (j < sink_end || j >= win))) { s[u * PER + k] = -INFINITY; seen &= ~(1u << (u * PER + k)); }
                }
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < (int)N; i++) mx = fmaxf(mx, s[i]);
        const float mn = fmaxf(m, quad_max(mx) * w.back), ref = mn == -INFINITY ? 0.f : mn;  // (nothing seen yet: every p is 2^-inf = 0)
        const float al = ex2(m - ref), from = T::P_LOG2 - ref;
        m = mn;
        float pr[N], sum = 0.f;
#pragma unroll
        for (int i = 0; i < (int)N; i++) { pr[i] = ex2(fmaf(s[i], w.back, from)); sum += pr[i]; }
        l = fmaf(l, al, sum);
        w.values(at, lane, pr, seen, __shfl_sync(0xffffffffu, al, 8 * t), __shfl_sync(0xffffffffu, al, 8 * t + 4));
        __syncwarp();  // every lane has read the stage
        if (done + STAGES < rounds) issue(done + STAGES, stage);
        if (++stage == STAGES) { stage = 0; parity ^= 1u; }
    }
    // After a wait that ran out: copies still in flight must land before this memory is used for anything else.
    for (uint32_t i = done; i < min(rounds, done + STAGES); i++) {
        mbar_wait(bar + 8 * stage, parity);
        if (++stage == STAGES) { stage = 0; parity ^= 1u; }
    }
    w.finish(lane);
    l = quad_sum(l);

    // The warp's state into its own ring, m and l beside.
    float* own = reinterpret_cast<float*>(smem + warp * SM::ring);
    float* ml = reinterpret_cast<float*>(smem + SM::ml);
    __syncwarp();
#pragma unroll
    for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
        for (int i = 0; i < 4; i++) own[(2 * t + (i & 1)) * D + T::dim(mt, i, lane)] = w.o[mt][i];
    if (t == 0) { ml[warp * 16 + g] = m; ml[warp * 16 + 8 + g] = l; }
    __syncthreads();
    // The CTA's state: its warps' in order, weighted by 2^(m - M).  Four elements a thread at a time.
    float* cta = reinterpret_cast<float*>(smem + SM::state);
    float* out = a.out + ((uint64_t)token * a.heads + head0) * D;
#pragma unroll
    for (uint32_t e = threadIdx.x * 4; e < 8 * D; e += NW * 128) {
        const uint32_t h = e / D;
        float M = -INFINITY, L = 0.f, f[NW];
#pragma unroll
        for (int i = 0; i < NW; i++) { f[i] = ml[i * 16 + h]; M = fmaxf(M, f[i]); }
        const float ref = M == -INFINITY ? 0.f : M;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NW; i++) {
            f[i] = ex2(f[i] - ref);
            L = fmaf(f[i], ml[i * 16 + 8 + h], L);
            const float4 y = *reinterpret_cast<const float4*>(smem + i * SM::ring + e * 4);
            x.x = fmaf(f[i], y.x, x.x); x.y = fmaf(f[i], y.y, x.y); x.z = fmaf(f[i], y.z, x.z); x.w = fmaf(f[i], y.w, x.w);
        }
        if (ranks == 1) {
            if (h < nheads && !over)
                *reinterpret_cast<float4*>(out + e) = L == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x / L, x.y / L, x.z / L, x.w / L);
        } else {
            *reinterpret_cast<float4*>(cta + e) = x;
            if (e % D == 0) { ml[NW * 16 + h] = M; ml[NW * 16 + 8 + h] = L; }
        }
    }
    if (ranks == 1) return;
    cluster_sync_all();
    // Every CTA joins its share of the elements over the cluster's states, in rank order.
    for (uint32_t e = rank * (NW * 32) + threadIdx.x; e < nheads * D; e += ranks * (NW * 32)) {
        const uint32_t h = e / D, m_at = base + SM::ml + NW * 64 + 4 * h, x_at = base + SM::state + 4 * e;
        float M = -INFINITY, L = 0.f, x = 0.f;
        for (uint32_t r0 = 0; r0 < ranks; r0 += 8) {  // (eight ranks' values in flight together)
            float rm[8], rl[8], rx[8];
#pragma unroll
            for (uint32_t r = 0; r < 8; r++) {
                const uint32_t from = min(r0 + r, ranks - 1);
                rm[r] = ld_cluster(m_at, from); rl[r] = ld_cluster(m_at + 32, from); rx[r] = ld_cluster(x_at, from);
            }
            float most = M;
#pragma unroll
            for (uint32_t r = 0; r < 8; r++) most = fmaxf(most, rm[r]);
            const float ref = most == -INFINITY ? 0.f : most, keep = ex2(M - ref);
            L *= keep; x *= keep; M = most;
#pragma unroll
            for (uint32_t r = 0; r < 8; r++) {
                const float f = r0 + r < ranks ? ex2(rm[r] - ref) : 0.f;
                L = fmaf(f, rl[r], L);
                x = fmaf(f, rx[r], x);
            }
        }
        if (!over) out[e] = L == 0.f ? 0.f : x / L;
    }
    cluster_sync_all();  // nobody leaves while its shared memory is being read
}

bool attn_window_supported(const Layout& L, size_t heads) {
    if (L.layout != QVX_LAYOUT_NATIVE || L.B % 16 != 0 || heads == 0 || heads % L.kvh != 0) return false;
    return L.d == 64 || L.d == 128 || L.d == 256;
}

// What one of the kernels is on one device: its attributes set, and how many clusters of each size the device holds at once
// (not its slots over the size: a cluster lies within one of the chip's groups of SMs).
struct WindowKernel {
    std::mutex mu;
    bool ready = false;
    uint32_t held[17] = {};
};

// `ranks` CTAs per cluster of a launch of `units` clusters: as many as leave every cluster resident at once (64 long 4-bit
// sequences: 107 us with clusters of 6, 115 with 4, 134 with 8, which come in two waves) and every second warp at least in
// work (4 x 37-512 positions: 4.4 us with half of 8 CTAs' warps idle, 5.0 with 4 CTAs).  With go: the launch as well.
template <class T, int D, int NW, int STAGES, int MIN_CTAS>
static cudaError_t window_ranks(const WindowArgs& a, uint64_t units, uint32_t tiles, int ordinal, uint32_t& ranks, bool go, dim3 grid, cudaStream_t s) {
    auto* kernel = attn_window_kernel<T, D, NW, STAGES, MIN_CTAS>;
    using SM = WindowSmem<T, D, NW, STAGES>;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = SM::bytes;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    static WindowKernel on[64];
    if (ordinal < 0 || ordinal >= 64) return cudaErrorInvalidDevice;
    WindowKernel& k = on[ordinal];
    {
        std::lock_guard<std::mutex> lk(k.mu);
        if (!k.ready) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SM::bytes);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            for (uint32_t r = 1; e == cudaSuccess && r <= 16; r = r < 8 ? r + 1 : r + 8) {
                int n = 0;
                cfg.gridDim = dim3(r, 1024); at[0].val.clusterDim.x = r;
                e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
                k.held[r] = n > 0 ? (uint32_t)n : 0u;
            }
            if (e != cudaSuccess) return e;
            k.ready = true;
        }
    }
    ranks = 1;
    for (uint32_t r = 2; r <= 16; r = r < 8 ? r + 1 : r + 8)
        if (units <= k.held[r] && r * NW <= 2 * tiles) ranks = r;
#ifdef QVX_EXPERIMENTS
    if (const char* v = getenv("QVX_WINDOW_RANKS")) ranks = (uint32_t)atol(v);
#endif
    if (!go) return cudaSuccess;
    grid.x = ranks;
    cfg.gridDim = grid;
    cfg.stream = s;
    at[0].val.clusterDim.x = ranks;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// CTAs of four warps; of eight where four would leave one CTA to an SM at most and every warp a few stages of work.
template <class T, int D, int STAGES, int MIN_CTAS, bool EIGHT>
static cudaError_t launch_window(const WindowArgs& a, uint64_t units, uint32_t tiles, uint32_t sms, int ordinal, dim3 grid, cudaStream_t s) {
    uint32_t ranks = 1;
    if constexpr (EIGHT) {
        cudaError_t e = window_ranks<T, D, 4, STAGES, MIN_CTAS>(a, units, tiles, ordinal, ranks, false, grid, s);
        if (e != cudaSuccess) return e;
        if (units * ranks <= sms && tiles >= ranks * 8 * T::SUB * 2) return window_ranks<T, D, 8, STAGES, 1>(a, units, tiles, ordinal, ranks, true, grid, s);
    }
    return window_ranks<T, D, 4, STAGES, MIN_CTAS>(a, units, tiles, ordinal, ranks, true, grid, s);
}

int32_t launch_attn_window(qvx_device* dev, const Layout& L, const void* pool, size_t pool_blocks, size_t heads, size_t s, const float* q,
                           const uint32_t* pos, const uint32_t* blocks, size_t n_blocks, const uint32_t* table_at, uint32_t max_pos,
                           uint32_t window, uint32_t sinks, float* out, cudaStream_t stream) {
    if (max_pos > 0x7fffffffu) return fail(dev, QVX_ERR_SHAPE, "shape mismatch in window attention: max_pos %u is past 2^31 - 1", max_pos);
    if (s == 0) return QVX_OK;
    if (((uintptr_t)pool | (uintptr_t)q | (uintptr_t)out) & 15u)
        return fail(dev, QVX_ERR_SHAPE, "shape mismatch in window attention: pool, q and out must be 16-byte aligned");
    const uint32_t tp = L.dtype == QVX_F32 ? 8 : 16;
    WindowArgs a{};
    a.pool = (const uint8_t*)pool; a.q = q; a.out = out; a.pos = pos; a.blocks = blocks; a.table_at = table_at;
    a.n_blocks = n_blocks; a.block_bytes = L.block_bytes; a.page_bytes = L.page_bytes;
    a.pool_blocks = (uint32_t)std::min<size_t>(pool_blocks, 0xffffffffu);
    a.max_pos = max_pos; a.window = window; a.sinks = sinks;
    a.heads = (uint32_t)heads; a.group = (uint32_t)(heads / L.kvh); a.groups_per_kv = (a.group + 7) / 8;
    a.tiles_per_block = L.B / tp;
    a.tile_stride = L.dtype == QVX_Q4 ? q4_tile_bytes(L.d) : tp * L.row_bytes;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)L.d));
    a.status = device_status_word(dev);
    uint64_t most = (uint64_t)max_pos + 1;  // positions a token of this call may see
    if (window) most = std::min(most, (uint64_t)window + sinks);
    const uint32_t tiles = (uint32_t)((most + tp - 1) / tp);
    const dim3 grid(1, L.kvh * a.groups_per_kv, (unsigned)s);
    const uint64_t units = (uint64_t)grid.y * grid.z;
    LaunchTimer timer(dev, QVX_K_ATTN, stream);
    cudaError_t e = cudaErrorInvalidValue;
    const uint32_t sms = (uint32_t)dev->prop.multiProcessorCount;
#define QVX_WINDOW(TYPE, TILE_T, DD, STG, CTAS, EIGHT) \
    if (L.dtype == TYPE && L.d == DD) e = launch_window<TILE_T, DD, STG, CTAS, EIGHT>(a, units, tiles, sms, dev->ordinal, grid, stream);
#define QVX_COMMA ,
    QVX_WINDOW(QVX_BF16, Tile16<QVX_BF16 QVX_COMMA 64>, 64, 3, 4, true)
    QVX_WINDOW(QVX_BF16, Tile16<QVX_BF16 QVX_COMMA 128>, 128, 3, 2, true)
    QVX_WINDOW(QVX_BF16, Tile16<QVX_BF16 QVX_COMMA 256>, 256, 3, 1, false)  // (eight warps' rings do not fit)
    QVX_WINDOW(QVX_F16, Tile16<QVX_F16 QVX_COMMA 64>, 64, 3, 4, true)
    QVX_WINDOW(QVX_F16, Tile16<QVX_F16 QVX_COMMA 128>, 128, 3, 2, true)
    QVX_WINDOW(QVX_F16, Tile16<QVX_F16 QVX_COMMA 256>, 256, 3, 1, false)
    QVX_WINDOW(QVX_F32, Tile32<64>, 64, 3, 4, true)
    QVX_WINDOW(QVX_F32, Tile32<128>, 128, 3, 2, true)
    QVX_WINDOW(QVX_F32, Tile32<256>, 256, 3, 1, false)
    QVX_WINDOW(QVX_Q4, TileQ4<64>, 64, 2, 4, true)
    QVX_WINDOW(QVX_Q4, TileQ4<128>, 128, 2, 3, true)
    QVX_WINDOW(QVX_Q4, TileQ4<256>, 256, 2, 2, true)
#undef QVX_COMMA
#undef QVX_WINDOW
    return check_cuda(dev, e, "window attention launch");
}

}  // namespace qvx
