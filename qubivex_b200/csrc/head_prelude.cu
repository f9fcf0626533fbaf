// The prelude of decoders that norm every head by itself: RMS norm of each query and key head (d weights, one set for
// all heads), NeoX rotation by the token's position, and the store of the key and value rows into the pool, in one pass
// over the token's projections:
//   y = x * (1 / sqrt(sum(x^2) / d + eps)) * w,   z_i = y_i cos_i - y_{i+r/2} sin_i,  z_{i+r/2} = y_{i+r/2} cos_i + y_i sin_i
// for i < r/2 (r = rot_dim <= d, the rest of a head is not turned).  Values are not touched on their way to the pool.
//
// Everything between load and store is f32; what is stored is rounded once to the pool's type.
// 8191 tokens of 32 + 8 + 8 bf16 heads of 128 into an f16 pool: 61 us for 268 MB, 68 % of the measured copy bandwidth (two
// thirds of the bytes are writes; f32 throughout: 85 %; norms left out: no faster).  64 tokens: 3.3 us.
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
    uint32_t heads, s, dtype, rope_rows, rot, pool_blocks, shift;
    uint32_t wide;  // outputs can be written 32 bytes at a time
    float eps;
    int* status;
};

__device__ __forceinline__ float load_one(const uint8_t* p, uint32_t dtype, uint64_t i) {
    return dtype == QVX_F32 ? reinterpret_cast<const float*>(p)[i] : widen16(reinterpret_cast<const uint16_t*>(p)[i], dtype);
}
// Eight consecutive elements, fetched (so that the next task's are on their way while this one's are worked on) and
// widened.  ACT: their type, read 16 bytes at a time, or ANY_ACT: the type as an argument, one by one.
constexpr int ANY_ACT = 3;
template <int ACT>
struct Eight {
    uint4 a, b;
    __device__ __forceinline__ void fetch(const uint8_t* p, uint32_t dtype, uint64_t i) {
        if constexpr (ACT == QVX_F32) {
            const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
            a = __ldcs(q); b = __ldcs(q + 1);
        } else if constexpr (ACT == ANY_ACT) {
            a.x = __float_as_uint(load_one(p, dtype, i)); a.y = __float_as_uint(load_one(p, dtype, i + 1));
            a.z = __float_as_uint(load_one(p, dtype, i + 2)); a.w = __float_as_uint(load_one(p, dtype, i + 3));
            b.x = __float_as_uint(load_one(p, dtype, i + 4)); b.y = __float_as_uint(load_one(p, dtype, i + 5));
            b.z = __float_as_uint(load_one(p, dtype, i + 6)); b.w = __float_as_uint(load_one(p, dtype, i + 7));
        } else {
            a = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i));
        }
    }
    __device__ __forceinline__ void clear() { a = b = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void widen(float (&x)[8]) const {
        if constexpr (ACT == QVX_F32 || ACT == ANY_ACT) {
            x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
            x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
        } else {
            const uint32_t h[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (ACT == QVX_BF16) { x[2 * k] = __uint_as_float(h[k] << 16); x[2 * k + 1] = __uint_as_float(h[k] & 0xffff0000u); }
                else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[k])); x[2 * k] = f.x; x[2 * k + 1] = f.y; }
            }
        }
    }
};

// Where token t's rows go: false when nothing is stored (no pool, or an entry that is not the pool's, which is reported).
__device__ __forceinline__ bool pool_target(const HeadPreludeArgs& a, uint32_t t, uint32_t p, uint32_t& block, uint32_t& slot) {
    if (!a.pool) return false;
    split_position(p, a.L.B, a.shift, block, slot);
    const uint64_t at = (uint64_t)a.table_at[t] + block;
    block = at < a.n_blocks ? a.blocks[at] : 0xffffffffu;
    if (block < a.pool_blocks) return true;
    atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL);
    return false;
}

// A task is ROWS passes of 256 / D consecutive heads of one token, all queries, all keys or all values: angles and the
// place in the pool are worked out once, and the rows' loads are in flight together.  A lane holds eight consecutive
// elements; rotating swaps them between lanes at a distance of half / 8 (shuffles) or, where rot_dim is not a multiple of
// 16, reads the partners again.  The grid is what the device holds at once, and its warps go through the queries' tasks,
// then the keys', then the values': one kind of code at a time (a warp per task spent a quarter of its time waiting for
// instructions), weights loaded once, the next task's position on its way.  PLAIN: norms, the exchange, no pool -- queries
// as they mostly are, with no decision left in the rows' code.
template <int D, int ROWS, int ACT, bool PLAIN>
__device__ __forceinline__ void prelude_tasks(const HeadPreludeArgs& a, const uint32_t part, uint32_t task, const uint32_t tasks, const uint32_t warps) {
    constexpr uint32_t LPR = D / 8, AT_ONCE = 32 / LPR, PER_WARP = ROWS * AT_ONCE;
    const uint32_t lane = threadIdx.x & 31u, i = lane % LPR * 8u;
    const uint32_t heads = part == 0 ? a.heads : a.L.kvh, pieces = (heads + PER_WARP - 1) / PER_WARP;
    const uint8_t* src = part == 0 ? a.q : part == 1 ? a.k : a.v;
    const uint64_t stride = part == 0 ? a.q_stride : part == 1 ? a.k_stride : a.v_stride;
    float* const out = part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;
    const float* w = part == 0 ? a.q_norm : a.k_norm;
    const bool norm = PLAIN || (part < 2 && w != nullptr), turn = PLAIN || (part < 2 && a.rot != 0);
    const uint32_t half = a.rot / 2;
    const bool exchange = PLAIN || half % 8 == 0;
    const uint32_t h8 = half / 8, at = i / 8, from = at < h8 ? lane + h8 : at < 2 * h8 ? lane - h8 : lane;
    if (task >= tasks) return;
    float wv[8];
#pragma unroll
    for (int k = 0; k < 8; k++) wv[k] = norm ? __ldg(w + i + k) : 1.f;
    Eight<ACT> ahead[ROWS];
    auto fetch = [&](uint32_t t, uint32_t g) {
#pragma unroll
        for (int u = 0; u < ROWS; u++) {
            // (lanes of a row past the last keep their warp company in its shuffles)
            if (g + u * AT_ONCE < heads) ahead[u].fetch(src, a.dtype, (uint64_t)t * stride + (uint64_t)(g + u * AT_ONCE) * D + i);
            else ahead[u].clear();
        }
    };
    // This lane's first head of a task; the next are AT_ONCE apart.
    uint32_t t = task / pieces, g0 = (task - t * pieces) * PER_WARP + lane / LPR, p = a.pos[t];
    fetch(t, g0);
    uint32_t t_next = t, g_next = g0, p_next = p;
    for (; task < tasks; task += warps, t = t_next, g0 = g_next, p = p_next) {
        const uint64_t row = (uint64_t)t * stride + (uint64_t)g0 * D + i;
        float x[ROWS][8];
#pragma unroll
        for (int u = 0; u < ROWS; u++) ahead[u].widen(x[u]);
        if (task + warps < tasks) {
            t_next = (task + warps) / pieces; g_next = (task + warps - t_next * pieces) * PER_WARP + lane / LPR;
            p_next = a.pos[t_next];
            // (outputs may lie where the inputs do, but a task's rows are read and written by this warp alone)
            fetch(t_next, g_next);
        }
        if (p == QVX_POS_NONE) continue;  // padding of the batch
        if (a.rope && p >= a.rope_rows) {
            if (part == 0 && g0 == 0) atomicExch(a.status, STATUS_POSITION_BOUND);
            continue;
        }
        float cs[8], sn[8];  // this lane's cosines and signed sines (1 and 0 past rot_dim)
#pragma unroll
        for (int k = 0; k < 8; k++) { cs[k] = 1.f; sn[k] = 0.f; }
        if (turn && i < a.rot) {
            const float* table = a.rope + (uint64_t)p * a.rot;
            if (exchange) {
                const uint32_t c = i < half ? i : i - half;
                const float sign = i < half ? -1.f : 1.f;
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const float4 cv = __ldg(reinterpret_cast<const float4*>(table + c + k)), sv = __ldg(reinterpret_cast<const float4*>(table + half + c + k));
                    cs[k] = cv.x; cs[k + 1] = cv.y; cs[k + 2] = cv.z; cs[k + 3] = cv.w;
                    sn[k] = sign * sv.x; sn[k + 1] = sign * sv.y; sn[k + 2] = sign * sv.z; sn[k + 3] = sign * sv.w;
                }
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 8; k++) {
                    const uint32_t e = i + k;
                    if (e < a.rot) {
                        cs[k] = table[e < half ? e : e - half];
                        sn[k] = e < half ? -table[half + e] : table[e];
                    }
                }
            }
        }
        uint32_t block = 0, slot = 0;
        const bool store = !PLAIN && part > 0 && pool_target(a, t, p, block, slot);
        uint8_t* at_block = a.pool + (uint64_t)block * a.L.block_bytes;
#pragma unroll
        for (int u = 0; u < ROWS; u++) {
            const uint32_t g = g0 + u * AT_ONCE;
            const bool live = g < heads;
            float(&v)[8] = x[u];
            float r = 1.f;
            if (norm) {
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int k = 0; k < 8; k += 2) { s0 = fmaf(v[k], v[k], s0); s1 = fmaf(v[k + 1], v[k + 1], s1); }
                float ss = s0 + s1;
#pragma unroll
                for (uint32_t m = LPR / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
                r = rsqrtf(fmaf(ss, 1.0f / D, a.eps));
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = v[k] * r * wv[k];
            }
            if (turn) {
                float o[8];  // the elements these are turned with, normed as well
                if (exchange) {
#pragma unroll
                    for (int k = 0; k < 8; k++) o[k] = __shfl_sync(0xffffffffu, v[k], from);
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 8; k++) {
                        const uint32_t e = i + k, other = e < half ? e + half : e - half;
                        o[k] = 0.f;
                        if (live && e < a.rot) {
                            o[k] = load_one(src, a.dtype, row - i + u * AT_ONCE * D + other);
                            if (norm) o[k] *= r * w[other];
                        }
                    }
                    __syncwarp();  // (outputs may lie where the inputs do: every lane has read what it needs)
                }
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = fmaf(v[k], cs[k], o[k] * sn[k]);
            }
            if ((PLAIN || out) && live) {
                float* to = out + ((uint64_t)t * heads + g) * D + i;
                if (a.wide) st_f32x8(to, v);
                else {
                    reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
            if (PLAIN || part == 0 || a.pool == nullptr) continue;
            if (a.L.dtype == QVX_Q4) {  // (all lanes of the warp: the groups' extremes go by shuffles)
                __half step, offset;
                const uint32_t codes = q4_quantise(v, step, offset);
                if (store && live)
                    Q4Place<D>(part - 1u, i).store(at_block + (uint64_t)g * 2u * a.L.page_bytes + slot / Q4_TILE * q4_tile_bytes(D), slot % Q4_TILE, codes, step, offset);
            } else if (store && live) {
                if (a.L.layout == QVX_LAYOUT_NATIVE) {
                    if (a.L.dtype == QVX_F32) {
                        *reinterpret_cast<float4*>(at_block + in_block_offset(a.L, slot, part - 1u, g, i)) = make_float4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<float4*>(at_block + in_block_offset(a.L, slot, part - 1u, g, i + 4)) = make_float4(v[4], v[5], v[6], v[7]);
                    } else {
                        *reinterpret_cast<uint4*>(at_block + in_block_offset(a.L, slot, part - 1u, g, i)) =
                            make_uint4(narrow16x2(v[0], v[1], a.L.dtype), narrow16x2(v[2], v[3], a.L.dtype), narrow16x2(v[4], v[5], a.L.dtype),
                                       narrow16x2(v[6], v[7], a.L.dtype));
                    }
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 8; k++) {
                        uint8_t* to = at_block + in_block_offset(a.L, slot, part - 1u, g, i + k);
                        if (a.L.dtype == QVX_F32) *reinterpret_cast<float*>(to) = v[k];
                        else *reinterpret_cast<uint16_t*>(to) = narrow16(v[k], a.L.dtype);
                    }
                }
            }
        }
    }
}

template <int D, int ROWS, int ACT>
__global__ void __launch_bounds__(256, 3) head_prelude_kernel(HeadPreludeArgs a) {
    constexpr uint32_t PER_WARP = ROWS * (256 / D);
    const uint32_t warps = gridDim.x * 8u, gw = blockIdx.x * 8u + (threadIdx.x >> 5);
    const uint32_t q_tasks = a.s * ((a.heads + PER_WARP - 1) / PER_WARP), kv_tasks = a.s * ((a.L.kvh + PER_WARP - 1) / PER_WARP);
    if (a.q_norm && a.rot && a.rot % 16 == 0) prelude_tasks<D, ROWS, ACT, true>(a, 0, gw, q_tasks, warps);
    else prelude_tasks<D, ROWS, ACT, false>(a, 0, gw, q_tasks, warps);
    // (the warps that the tasks before left out go first)
    prelude_tasks<D, ROWS, ACT, false>(a, 1, (gw + warps - q_tasks % warps) % warps, kv_tasks, warps);
    prelude_tasks<D, ROWS, ACT, false>(a, 2, (gw + warps - (q_tasks + kv_tasks) % warps) % warps, kv_tasks, warps);
}

template <int D, int ROWS>
static void launch_sized(const HeadPreludeArgs& a, uint64_t warps, bool vec, uint32_t sms, cudaStream_t s) {
    const unsigned grid = (unsigned)std::min<uint64_t>((warps + 7) / 8, 3ull * sms);
    if (!vec) head_prelude_kernel<D, ROWS, ANY_ACT><<<grid, 256, 0, s>>>(a);
    else if (a.dtype == QVX_F32) head_prelude_kernel<D, ROWS, QVX_F32><<<grid, 256, 0, s>>>(a);
    else if (a.dtype == QVX_BF16) head_prelude_kernel<D, ROWS, QVX_BF16><<<grid, 256, 0, s>>>(a);
    else head_prelude_kernel<D, ROWS, QVX_F16><<<grid, 256, 0, s>>>(a);
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
    a.shift = block_shift(L.B);
    a.eps = (float)p->eps;
    a.status = device_status_word(dev);
    const uint32_t e = p->dtype == QVX_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v) % 16) == 0 && ((p->q_stride | p->k_stride | p->v_stride) * e % 16) == 0;
    a.wide = (((uintptr_t)p->q_out | (uintptr_t)p->k_out | (uintptr_t)p->v_out) % 32) == 0 ? 1u : 0u;
    const uint32_t rows = a.heads + 2u * L.kvh;
    const bool sized = L.d == 64 || L.d == 128 || L.d == 256;
    // Fewer rows than warps the device holds: a warp each, for the least latency.
    const uint32_t sms = (uint32_t)dev->prop.multiProcessorCount;
    const bool few = (uint64_t)s * rows < (uint64_t)sms * 32;
    const uint32_t per = sized ? (few ? 1u : 2u) * (256u / L.d) : 1u;
    const uint64_t warps = (uint64_t)s * ((a.heads + per - 1) / per + 2 * ((L.kvh + per - 1) / per));
    if (warps > 0x7fffffffull) return fail(dev, QVX_ERR_CORE, "head prelude: %zu tokens are too many for one launch", s);
    LaunchTimer timer(dev, QVX_K_PRELUDE, stream);
    if (!sized) head_prelude_any_kernel<<<dim3((unsigned)s, (rows + 7) / 8), 256, 0, stream>>>(a);
    else if (L.d == 64) { if (few) launch_sized<64, 1>(a, warps, vec, sms, stream); else launch_sized<64, 2>(a, warps, vec, sms, stream); }
    else if (L.d == 128) { if (few) launch_sized<128, 1>(a, warps, vec, sms, stream); else launch_sized<128, 2>(a, warps, vec, sms, stream); }
    else { if (few) launch_sized<256, 1>(a, warps, vec, sms, stream); else launch_sized<256, 2>(a, warps, vec, sms, stream); }
    return check_cuda(dev, cudaGetLastError(), "head prelude launch");
}

}  // namespace qvx
