// The prelude of decoders that norm every head by itself: RMS norm of each query and key head (d weights, one set for
// all heads), NeoX rotation by the token's position, and the store of the key and value rows into the pool, in one pass
// over the token's projections:
//   y = x * (1 / sqrt(sum(x^2) / d + eps)) * w,   z_i = y_i cos_i - y_{i+r/2} sin_i,  z_{i+r/2} = y_{i+r/2} cos_i + y_i sin_i
// for i < r/2 (r = rot_dim <= d, the rest of a head is not turned).  Values are not touched on their way to the pool.
//
// A warp takes a head: four consecutive elements per lane (two heads per warp at d = 64, two fours per lane at 256),
// the sum of squares by shuffles, the partner element of a rotation read again (it is in the L1: the other half of the
// same row).  Everything between load and store is f32; what is stored is rounded once to the pool's type.
// Bound by HBM at prompt lengths and by launch latency for a few tokens.
#include <algorithm>

#include "q4.cuh"

namespace qvx {

extern int* device_status_word(qvx_device* dev);

struct HeadPreludeArgs {
    Layout L;
    const uint8_t *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;  // elements between tokens
    const float *q_norm, *k_norm, *rope;
    const uint32_t *pos, *blocks, *table_at;
    float *q_out, *k_out, *v_out;
    uint8_t* pool;
    uint64_t n_blocks;
    uint32_t heads, s, dtype, rope_rows, rot, pool_blocks;
    float eps;
    int* status;
};

__device__ __forceinline__ float load_one(const uint8_t* p, uint32_t dtype, uint64_t i) {
    return dtype == QVX_F32 ? reinterpret_cast<const float*>(p)[i] : widen16(reinterpret_cast<const uint16_t*>(p)[i], dtype);
}
// Elements 4 j .. 4 j + 3 of a row.  VEC: the row starts at a multiple of four elements.
template <bool VEC>
__device__ __forceinline__ float4 load_four(const uint8_t* p, uint32_t dtype, uint64_t i) {
    if constexpr (VEC) {
        if (dtype == QVX_F32) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
        const uint2 h = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
        if (dtype == QVX_BF16)
            return make_float4(__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16),
                               __uint_as_float(h.y & 0xffff0000u));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
        return make_float4(a.x, a.y, b.x, b.y);
    } else {
        return make_float4(load_one(p, dtype, i), load_one(p, dtype, i + 1), load_one(p, dtype, i + 2), load_one(p, dtype, i + 3));
    }
}
template <bool VEC>
__device__ __forceinline__ void store_four(float* p, uint64_t i, float4 v) {
    if constexpr (VEC) { *reinterpret_cast<float4*>(p + i) = v; }
    else { p[i] = v.x; p[i + 1] = v.y; p[i + 2] = v.z; p[i + 3] = v.w; }
}

// Where token t's rows go: false when nothing is stored (no pool, or an entry that is not the pool's, which is reported).
__device__ __forceinline__ bool pool_target(const HeadPreludeArgs& a, uint32_t t, uint32_t p, uint32_t& block, uint32_t& slot) {
    if (!a.pool) return false;
    const uint64_t at = (uint64_t)a.table_at[t] + p / a.L.B;
    block = at < a.n_blocks ? a.blocks[at] : 0xffffffffu;
    slot = p % a.L.B;
    if (block < a.pool_blocks) return true;
    atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL);
    return false;
}

// Heads of a token in order: queries, keys, values.  A warp (half a warp at D = 64) takes one.
template <int D, bool VEC>
__global__ void __launch_bounds__(256) head_prelude_kernel(HeadPreludeArgs a) {
    constexpr uint32_t LPR = D == 64 ? 16 : 32, SEG = D == 256 ? 2 : 1;  // lanes per row, fours per lane
    const uint32_t sub = threadIdx.x / LPR, l = threadIdx.x % LPR, t = blockIdx.x;
    const uint32_t total = a.heads + 2u * a.L.kvh, h = blockIdx.y * (256u / LPR) + sub;
    const uint32_t p = a.pos[t];
    if (p == 0xffffffffu) return;  // padding of the batch
    if (a.rope && p >= a.rope_rows) {
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicExch(a.status, STATUS_POSITION_BOUND);
        return;
    }
    const bool live = h < total;  // (lanes of a row past the last keep their warp company in its shuffles)
    const uint32_t part = h < a.heads ? 0u : h < a.heads + a.L.kvh ? 1u : 2u;
    const uint32_t g = part == 0 ? h : part == 1 ? h - a.heads : h - a.heads - a.L.kvh;
    const uint8_t* src = part == 0 ? a.q : part == 1 ? a.k : a.v;
    const uint64_t row = (uint64_t)t * (part == 0 ? a.q_stride : part == 1 ? a.k_stride : a.v_stride) + (uint64_t)g * D;
    const float* w = part == 0 ? a.q_norm : a.k_norm;
    const bool norm = part < 2 && w != nullptr, turn = part < 2 && a.rope != nullptr;
    const uint32_t half = a.rot / 2;
    float4 x[SEG], y[SEG];  // own elements, and the ones they are turned with
    float ss = 0.f;
#pragma unroll
    for (uint32_t sg = 0; sg < SEG; sg++) {
        x[sg] = y[sg] = make_float4(0.f, 0.f, 0.f, 0.f);
        const uint32_t i = 4u * (l + 32u * sg);
        if (live) {
            x[sg] = load_four<VEC>(src, a.dtype, row + i);
            if (turn && i < a.rot) {
                float* yy = &y[sg].x;
                const uint32_t other = i < half ? i + half : i - half;
                if (half % 4 == 0) y[sg] = load_four<VEC>(src, a.dtype, row + other);
                else
                    for (uint32_t k = 0; k < 4 && i + k < a.rot; k++) yy[k] = load_one(src, a.dtype, row + (i + k < half ? i + k + half : i + k - half));
            }
        }
        ss = fmaf(x[sg].x, x[sg].x, fmaf(x[sg].y, x[sg].y, fmaf(x[sg].z, x[sg].z, fmaf(x[sg].w, x[sg].w, ss))));
    }
#pragma unroll
    for (uint32_t m = LPR / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    const float r = norm ? 1.0f / sqrtf(ss * (1.0f / D) + a.eps) : 1.0f;
    __syncwarp();  // the outputs may lie where the inputs do: every lane of the row has read what it needs
    uint32_t block = 0, slot = 0;
    const bool store = live && part > 0 && pool_target(a, t, p, block, slot);
    float* out = !live ? nullptr : part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;
    const uint64_t out_row = ((uint64_t)t * (part == 0 ? a.heads : a.L.kvh) + g) * D;
    uint8_t* dst = a.pool + (uint64_t)block * a.L.block_bytes + (uint64_t)g * 2u * a.L.page_bytes;
#pragma unroll
    for (uint32_t sg = 0; sg < SEG; sg++) {
        const uint32_t i = 4u * (l + 32u * sg);
        float v[4] = {x[sg].x, x[sg].y, x[sg].z, x[sg].w}, o[4] = {y[sg].x, y[sg].y, y[sg].z, y[sg].w};
        if (norm) {
            const float4 wv = make_float4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            v[0] = v[0] * r * wv.x; v[1] = v[1] * r * wv.y; v[2] = v[2] * r * wv.z; v[3] = v[3] * r * wv.w;
        }
        if (turn && i < a.rot) {
            const float* table = a.rope + (uint64_t)p * a.rot;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const uint32_t e = i + k;
                if (e < a.rot) {
                    const bool first = e < half;
                    const uint32_t c = first ? e : e - half;
                    const float other = norm ? o[k] * r * w[first ? e + half : e - half] : o[k];
                    const float cs = table[c], sn = table[half + c];
                    v[k] = first ? v[k] * cs - other * sn : v[k] * cs + other * sn;
                }
            }
        }
        const float4 z = make_float4(v[0], v[1], v[2], v[3]);
        if (out) store_four<true>(out, out_row + i, z);
        if (a.pool == nullptr) continue;
        if (a.L.dtype == QVX_Q4) {  // (all lanes of the warp: the groups' extremes go by shuffles)
            __half step, offset;
            const uint32_t codes = q4_quantise(z, step, offset);
            if (store) {
                const uint32_t kv = part - 1u, j = i >> 2, sl = slot % Q4_TILE;
                uint8_t* tile = dst + (uint64_t)(slot / Q4_TILE) * q4_tile_bytes(D);
                *reinterpret_cast<uint16_t*>(tile + q4_codes_at(D, sl, kv, j)) = (uint16_t)codes;
                if ((j & 7u) == 0u) {
                    *reinterpret_cast<__half*>(tile + q4_step_at(D, sl, kv, j >> 3)) = step;
                    *reinterpret_cast<__half*>(tile + q4_offset_at(D, sl, kv, j >> 3)) = offset;
                }
            }
        } else if (store) {
            if (a.L.layout == QVX_LAYOUT_NATIVE) {
                uint8_t* at = a.pool + (uint64_t)block * a.L.block_bytes + in_block_offset(a.L, slot, part - 1u, g, i);
                if (a.L.dtype == QVX_F32) *reinterpret_cast<float4*>(at) = z;
                else *reinterpret_cast<uint2*>(at) = make_uint2(narrow16x2(z.x, z.y, a.L.dtype), narrow16x2(z.z, z.w, a.L.dtype));
            } else {
                for (uint32_t k = 0; k < 4; k++) {
                    uint8_t* at = a.pool + (uint64_t)block * a.L.block_bytes + in_block_offset(a.L, slot, part - 1u, g, i + k);
                    if (a.L.dtype == QVX_F32) *reinterpret_cast<float*>(at) = v[k];
                    else *reinterpret_cast<uint16_t*>(at) = narrow16(v[k], a.L.dtype);
                }
            }
        }
    }
}

// Any other head size: one warp per head, a lane takes whole pairs, so that outputs may lie where the inputs do.
__global__ void __launch_bounds__(256) head_prelude_any_kernel(HeadPreludeArgs a) {
    const uint32_t l = threadIdx.x & 31u, t = blockIdx.x, d = a.L.d;
    const uint32_t total = a.heads + 2u * a.L.kvh, h = blockIdx.y * 8u + (threadIdx.x >> 5);
    const uint32_t p = a.pos[t];
    if (h >= total || p == 0xffffffffu) return;
    if (a.rope && p >= a.rope_rows) {
        if (l == 0) atomicExch(a.status, STATUS_POSITION_BOUND);
        return;
    }
    const uint32_t part = h < a.heads ? 0u : h < a.heads + a.L.kvh ? 1u : 2u;
    const uint32_t g = part == 0 ? h : part == 1 ? h - a.heads : h - a.heads - a.L.kvh;
    const uint8_t* src = part == 0 ? a.q : part == 1 ? a.k : a.v;
    const uint64_t row = (uint64_t)t * (part == 0 ? a.q_stride : part == 1 ? a.k_stride : a.v_stride) + (uint64_t)g * d;
    const float* w = part == 0 ? a.q_norm : a.k_norm;
    const bool norm = part < 2 && w != nullptr;
    float r = 1.0f;
    if (norm) {
        float ss = 0.f;
        for (uint32_t i = l; i < d; i += 32) { const float x = load_one(src, a.dtype, row + i); ss = fmaf(x, x, ss); }
#pragma unroll
        for (uint32_t m = 16; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        r = 1.0f / sqrtf(ss / (float)d + a.eps);
    }
    __syncwarp();
    uint32_t block = 0, slot = 0;
    const bool store = part > 0 && pool_target(a, t, p, block, slot);
    float* out = part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;
    const uint64_t out_row = ((uint64_t)t * (part == 0 ? a.heads : a.L.kvh) + g) * d;
    auto put = [&](uint32_t i, float z) {
        if (out) out[out_row + i] = z;
        if (!store) return;
        uint8_t* at = a.pool + (uint64_t)block * a.L.block_bytes + in_block_offset(a.L, slot, part - 1u, g, i);
        if (a.L.dtype == QVX_F32) *reinterpret_cast<float*>(at) = z;
        else *reinterpret_cast<uint16_t*>(at) = narrow16(z, a.L.dtype);
    };
    const uint32_t half = part < 2 && a.rope ? a.rot / 2 : 0u;
    const float* table = a.rope + (uint64_t)p * a.rot;
    for (uint32_t i = l; i < half; i += 32) {
        float x = load_one(src, a.dtype, row + i), y = load_one(src, a.dtype, row + half + i);
        if (norm) { x = x * r * w[i]; y = y * r * w[half + i]; }
        const float cs = table[i], sn = table[half + i];
        put(i, x * cs - y * sn);
        put(half + i, y * cs + x * sn);
    }
    for (uint32_t i = 2 * half + l; i < d; i += 32) {
        const float x = load_one(src, a.dtype, row + i);
        put(i, norm ? x * r * w[i] : x);
    }
}

int32_t launch_head_prelude(qvx_device* dev, const Layout& L, size_t heads, size_t s, const qvx_head_prelude* p, cudaStream_t stream) {
    if (s == 0) return QVX_OK;
    HeadPreludeArgs a{};
    a.L = L;
    a.q = (const uint8_t*)p->q; a.k = (const uint8_t*)p->k; a.v = (const uint8_t*)p->v;
    a.q_stride = p->q_stride; a.k_stride = p->k_stride; a.v_stride = p->v_stride;
    a.q_norm = p->q_norm; a.k_norm = p->k_norm; a.rope = p->rope;
    a.pos = p->pos; a.blocks = p->blocks; a.table_at = p->table_at;
    a.q_out = p->q_out; a.k_out = p->k_out; a.v_out = p->v_out;
    a.pool = (uint8_t*)p->pool; a.n_blocks = p->n_blocks;
    a.heads = (uint32_t)heads; a.s = (uint32_t)s; a.dtype = p->dtype;
    a.rope_rows = p->rope_rows; a.rot = p->rope ? p->rot_dim : 0u;
    a.pool_blocks = (uint32_t)std::min<size_t>(p->pool_blocks, 0xffffffffu);
    a.eps = (float)p->eps;
    a.status = device_status_word(dev);
    const uint32_t e = p->dtype == QVX_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v) % (4 * e)) == 0 &&
                     ((p->q_stride | p->k_stride | p->v_stride) % 4) == 0;
    const uint32_t rows = a.heads + 2u * L.kvh;
    LaunchTimer timer(dev, QVX_K_PRELUDE, stream);
    const bool sized = L.d == 64 || L.d == 128 || L.d == 256;
    const uint32_t per = sized && L.d == 64 ? 16 : 8;
    const dim3 grid((unsigned)s, (rows + per - 1) / per);
    if (!sized) head_prelude_any_kernel<<<grid, 256, 0, stream>>>(a);
    else if (L.d == 64) { if (vec) head_prelude_kernel<64, true><<<grid, 256, 0, stream>>>(a); else head_prelude_kernel<64, false><<<grid, 256, 0, stream>>>(a); }
    else if (L.d == 128) { if (vec) head_prelude_kernel<128, true><<<grid, 256, 0, stream>>>(a); else head_prelude_kernel<128, false><<<grid, 256, 0, stream>>>(a); }
    else { if (vec) head_prelude_kernel<256, true><<<grid, 256, 0, stream>>>(a); else head_prelude_kernel<256, false><<<grid, 256, 0, stream>>>(a); }
    return check_cuda(dev, cudaGetLastError(), "head prelude launch");
}

}  // namespace qvx
