// KV sync and KV append of a 4-bit pool, and rows of any pool read back.
//
// Store: a thread takes eight consecutive elements of a row; four neighbouring lanes hold a group of 32, find its least
// and greatest value by shuffles, and each writes its eight codes; the first of the four writes the group's step and
// offset.  Every store is the group's own bytes, so rows of one tile may be written by any blocks in any order.  16383 rows
// of 8 x 128: about 36 us for 155 MB, bound by instructions (some 130 per 256 elements) before HBM.
// Bound by HBM: 4 + 5/8 bytes per element.
//
// Read: a thread takes eight consecutive elements (one word of codes, or two half words) and writes them in the type
// asked for.  5/8 + 2 bytes per element from a 4-bit pool to 16-bit rows.
//
// Block ids come from device memory: a row whose block lies at or past pool_blocks is neither written nor read and
// the status word says so, as in kv_rows.cu; 0xffffffff in place of a position is passed over in silence.
#include <algorithm>

#include "q4.cuh"

namespace qvx {

extern int* device_status_word(qvx_device* dev);

struct Q4RowArgs {
    Layout L;
    uint8_t* pool;
    const float *k_rows, *v_rows;
    size_t row_stride;
    const uint32_t *at_direct, *pos, *blocks, *table_at;
    uint32_t n, pool_blocks, shift;
    uint32_t aligned;  // bytes the rows can be read at a time: 32, 16, or 0 (one element)
    int* status;
};

// A warp keeps to one piece of 256 consecutive elements of the rows (`n_row` such pieces to a row, eight elements a lane)
// and goes through them ROWS at a time, the next ones on their way while these are worked on; the grid is what the device
// holds at once.  Two rows at a time; one where there are too few to give every warp two (100 rows: 2.4 us less latency
// for the store and the read together).
template <int D, int ROWS>
__global__ void __launch_bounds__(256, 4) kv_rows_q4_kernel(Q4RowArgs a, uint32_t n_row, uint32_t lines) {
    constexpr uint32_t d8 = D / 8;
    const uint32_t lane = threadIdx.x & 31u, half_row = a.L.kvh * d8;
    const uint32_t gw = blockIdx.x * 8u + (threadIdx.x >> 5), line = gw / n_row, w = (gw - line * n_row) * 32u + lane;
    if (line >= lines) return;
    const bool within = w < 2u * half_row;  // (a group's four lanes are in or out together)
    const uint32_t kv = w >= half_row ? 1u : 0u, e = w - kv * half_row, g = e / d8, i = e % d8 * 8u;
    const float* const src = (kv ? a.v_rows : a.k_rows) + 8u * e;
    const Q4Place<D> place(kv, i);
    uint8_t* const at_head = a.pool + (uint64_t)g * 2u * a.L.page_bytes;
    float next[ROWS][8];
    uint32_t p_next[ROWS];
    auto fetch = [&](uint32_t r0) {
#pragma unroll
        for (int u = 0; u < ROWS; u++) {
            const uint32_t r = r0 + u;
            p_next[u] = QVX_POS_NONE;
#pragma unroll
            for (int k = 0; k < 8; k++) next[u][k] = 0.f;
            if (!within || r >= a.n) continue;
            const float* at = src + (size_t)r * a.row_stride;
            if (a.aligned == 32) ld_f32x8(next[u], at);
            else if (a.aligned == 16) {
                const float4 v = reinterpret_cast<const float4*>(at)[0], y = reinterpret_cast<const float4*>(at)[1];
                next[u][0] = v.x; next[u][1] = v.y; next[u][2] = v.z; next[u][3] = v.w; next[u][4] = y.x; next[u][5] = y.y; next[u][6] = y.z; next[u][7] = y.w;
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) next[u][k] = at[k];
            }
            p_next[u] = a.at_direct ? a.at_direct[r] : a.pos[r];
        }
    };
    fetch(line * ROWS);
    for (uint32_t r0 = line * ROWS; r0 < a.n; r0 += lines * ROWS) {
        float x[ROWS][8];
        uint32_t block[ROWS], slot[ROWS];
        bool store[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; u++) {
#pragma unroll
            for (int k = 0; k < 8; k++) x[u][k] = next[u][k];
            store[u] = p_next[u] != QVX_POS_NONE;
            split_position(p_next[u], a.L.B, a.shift, block[u], slot[u]);
            if (store[u] && !a.at_direct) block[u] = a.blocks[a.table_at[r0 + u] + block[u]];
        }
        if (r0 + lines * ROWS < a.n) fetch(r0 + lines * ROWS);
#pragma unroll
        for (int u = 0; u < ROWS; u++) {
            __half step, offset;
            const uint32_t codes = q4_quantise(x[u], step, offset);
            if (store[u] && block[u] >= a.pool_blocks) { atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL); store[u] = false; }
            if (store[u]) place.store(at_head + (uint64_t)block[u] * a.L.block_bytes + slot[u] / Q4_TILE * q4_tile_bytes(D), slot[u] % Q4_TILE, codes, step, offset);
        }
    }
}

int32_t launch_kv_rows_q4(qvx_device* dev, const Layout& L, void* pool, const float* k_rows, const float* v_rows,
                          size_t row_stride_f32, const uint32_t* at_direct, const uint32_t* pos, const uint32_t* blocks,
                          const uint32_t* table_at, size_t n, size_t pool_blocks, int kind, cudaStream_t s) {
    if (n > 0x7fffffffu) return fail(dev, QVX_ERR_CORE, "kv rows: %zu rows do not fit 31 bits", n);
    if ((uintptr_t)pool & 15u) return fail(dev, QVX_ERR_SHAPE, "shape mismatch in kv rows: a 4-bit pool must be 16-byte aligned");
    const uint32_t n_row = (L.kvh * (L.d / 8) * 2u + 31u) / 32u;
    // Lines of warps, one per piece of a row: as many as there are rows for, or as the device holds (32 warps an SM).
    const uint64_t held = std::max<uint64_t>(1, 32ull * dev->prop.multiProcessorCount / n_row);
    const uint32_t each = n > held ? 2 : 1;
    const uint32_t lines = (uint32_t)std::min<uint64_t>((n + each - 1) / each, held);
    const uint64_t grid = ((uint64_t)lines * n_row + 7) / 8;
    if (grid > 0x7fffffffull) return fail(dev, QVX_ERR_CORE, "kv rows: rows of %zu elements are too long for one launch", (size_t)L.kvh * L.d);
    const uintptr_t ends = (uintptr_t)k_rows | (uintptr_t)v_rows | (uintptr_t)(row_stride_f32 * 4);
    Q4RowArgs a{L, (uint8_t*)pool, k_rows, v_rows, row_stride_f32, at_direct, pos, blocks, table_at, (uint32_t)n,
                (uint32_t)std::min<size_t>(pool_blocks, 0xffffffffu), block_shift(L.B), ends % 32 == 0 ? 32u : ends % 16 == 0 ? 16u : 0u, device_status_word(dev)};
    LaunchTimer timer(dev, kind, s);
#define QVX_ROWS(DD)                                                                                 \
    if (L.d == DD && each == 1) kv_rows_q4_kernel<DD, 1><<<(unsigned)grid, 256, 0, s>>>(a, n_row, lines); \
    if (L.d == DD && each == 2) kv_rows_q4_kernel<DD, 2><<<(unsigned)grid, 256, 0, s>>>(a, n_row, lines);
    QVX_ROWS(64)
    QVX_ROWS(128)
    QVX_ROWS(256)
#undef QVX_ROWS
    return check_cuda(dev, cudaGetLastError(), "4-bit kv rows launch");
}

struct ReadArgs {
    Layout L;
    const uint8_t* pool;
    const uint32_t* from;
    void* rows;
    uint32_t n, pool_blocks, shift, rows_dtype;
    uint32_t wide;  // bytes the rows can be written at a time: 32, 16, or 0 (one element)
    int* status;
};

// Other pools: `WIDTH` consecutive elements per thread, 8, or 1 where d is not a multiple of 8.
template <int WIDTH>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
    const uint32_t per_head = a.L.d / WIDTH, per_row = 2u * a.L.kvh * per_head;
    const uint64_t idx = (uint64_t)blockIdx.x * 256u + threadIdx.x, row = idx / per_row;
    if (row >= a.n) return;
    const uint32_t r = (uint32_t)row, w = (uint32_t)(idx - row * per_row);
    const uint32_t kv = w / (a.L.kvh * per_head), e = w % (a.L.kvh * per_head), g = e / per_head, i = e % per_head * WIDTH;
    const uint32_t p = a.from[r];
    if (p == QVX_POS_NONE) return;
    uint32_t block, slot;
    split_position(p, a.L.B, a.shift, block, slot);
    if (block >= a.pool_blocks) { atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL); return; }
    const uint8_t* b = a.pool + (uint64_t)block * a.L.block_bytes;
    float x[WIDTH];
#pragma unroll
    for (int k = 0; k < WIDTH; k++) {
        const uint8_t* at = b + in_block_offset(a.L, slot, kv, g, i + k);
        x[k] = a.L.dtype == QVX_F32 ? *reinterpret_cast<const float*>(at) : widen16(*reinterpret_cast<const uint16_t*>(at), a.L.dtype);
    }
    const uint64_t o = row * 2u * a.L.kvh * a.L.d + (uint64_t)(kv * a.L.kvh + g) * a.L.d + i;
    if (a.rows_dtype == QVX_F32) {
        float* out = (float*)a.rows + o;
        if constexpr (WIDTH == 8) {
            if (a.wide) {
                reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < WIDTH; k++) out[k] = x[k];
    } else {
        uint16_t* out = (uint16_t*)a.rows + o;
        if constexpr (WIDTH == 8) {
            if (a.wide) {
                uint4 v;
                v.x = narrow16x2(x[0], x[1], a.rows_dtype); v.y = narrow16x2(x[2], x[3], a.rows_dtype);
                v.z = narrow16x2(x[4], x[5], a.rows_dtype); v.w = narrow16x2(x[6], x[7], a.rows_dtype);
                *reinterpret_cast<uint4*>(out) = v;
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < WIDTH; k++) out[k] = narrow16(x[k], a.rows_dtype);
    }
}

// 4-bit pools: a warp takes 256 consecutive elements of ROWS consecutive rows (n_row: such pieces of a row): four, or one
// where there are too few rows.
template <int D, int ROWS>
__global__ void __launch_bounds__(256) kv_read_q4_kernel(ReadArgs a, uint32_t n_row) {
    constexpr uint32_t d8 = D / 8;
    const uint32_t lane = threadIdx.x & 31u, half_row = a.L.kvh * d8;
    const uint32_t gw = blockIdx.x * 8u + (threadIdx.x >> 5), r0 = gw / n_row * ROWS, w = gw % n_row * 32u + lane;
    if (r0 >= a.n || w >= 2u * half_row) return;
    const uint32_t kv = w >= half_row ? 1u : 0u, e = w - kv * half_row, g = e / d8;
    const Q4Place<D> place(kv, e % d8 * 8u);
    const uint8_t* const at_head = a.pool + (uint64_t)g * 2u * a.L.page_bytes;
    uint32_t p[ROWS], c[ROWS];
    __half step[ROWS], off[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; u++) p[u] = r0 + u < a.n ? a.from[r0 + u] : QVX_POS_NONE;
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        if (p[u] == QVX_POS_NONE) continue;
        uint32_t block, slot;
        split_position(p[u], a.L.B, a.shift, block, slot);
        if (block >= a.pool_blocks) { atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL); p[u] = QVX_POS_NONE; continue; }
        const uint8_t* tile = at_head + (uint64_t)block * a.L.block_bytes + slot / Q4_TILE * q4_tile_bytes(D);
        slot %= Q4_TILE;
        const uint8_t* at = tile + place.codes_at(slot);
        c[u] = kv ? *reinterpret_cast<const uint16_t*>(at) | (uint32_t)*reinterpret_cast<const uint16_t*>(at + D / 16) << 16
                  : *reinterpret_cast<const uint32_t*>(at);
        step[u] = *reinterpret_cast<const __half*>(tile + place.step_at(slot));
        off[u] = *reinterpret_cast<const __half*>(tile + place.offset_at(slot));
    }
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        if (p[u] == QVX_POS_NONE) continue;
        // A code in bits 0..3 of a half word is the f16 number c 2^-24, in bits 4..7 c 2^-20: converting those is exact.
        const float z = __half2float(off[u]), s0 = __half2float(step[u]) * 16777216.f, s1 = s0 * 0.0625f;
        float x[8];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t h = c[u] >> (8 * k), lo = h & 0x000f000fu, hi = h & 0x00f000f0u;
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            x[2 * k] = fmaf(f.x, s0, z); x[2 * k + 4] = fmaf(f.y, s0, z);
            x[2 * k + 1] = fmaf(y.x, s1, z); x[2 * k + 5] = fmaf(y.y, s1, z);
        }
        const uint64_t o = (uint64_t)(r0 + u) * 2u * a.L.kvh * D + (uint64_t)w * 8u;
        if (a.rows_dtype == QVX_F32) {
            float* out = (float*)a.rows + o;
            if (a.wide == 32) st_f32x8(out, x);
            else {
#pragma unroll
                for (int k = 0; k < 8; k++) out[k] = x[k];
            }
        } else {
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (a.rows_dtype == QVX_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
                else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
            }
            const uint4 v = make_uint4(h[0], h[1], h[2], h[3]);
            uint16_t* out = (uint16_t*)a.rows + o;
            if (a.wide) __stcs(reinterpret_cast<uint4*>(out), v);
            else {
#pragma unroll
                for (int k = 0; k < 8; k++) out[k] = (uint16_t)((k & 2 ? (k & 4 ? v.w : v.y) : (k & 4 ? v.z : v.x)) >> (16 * (k & 1)));
            }
        }
    }
}

int32_t launch_kv_read(qvx_device* dev, const Layout& L, const void* pool, size_t pool_blocks, const uint32_t* from, size_t n,
                       void* rows, uint32_t rows_dtype, cudaStream_t s) {
    if (n == 0) return QVX_OK;
    if (n > 0x7fffffffu) return fail(dev, QVX_ERR_CORE, "kv read: %zu rows do not fit 31 bits", n);
    const ReadArgs a{L, (const uint8_t*)pool, from, rows, (uint32_t)n, (uint32_t)std::min<size_t>(pool_blocks, 0xffffffffu), block_shift(L.B), rows_dtype,
                     (uintptr_t)rows % 32 == 0 ? 32u : (uintptr_t)rows % 16 == 0 ? 16u : 0u, device_status_word(dev)};
    if (L.dtype == QVX_Q4) {
        const uint32_t n_row = (L.kvh * (L.d / 8) * 2u + 31u) / 32u;
        const uint32_t each = (uint64_t)n * n_row > 32ull * dev->prop.multiProcessorCount ? 4 : 1;
        const uint64_t warps = (uint64_t)((n + each - 1) / each) * n_row;
        if (warps > 0x7fffffffull) return fail(dev, QVX_ERR_CORE, "kv read: %zu rows are too many for one launch", n);
        const unsigned grid = (unsigned)((warps + 7) / 8);
        LaunchTimer timer(dev, QVX_K_COPY, s);
#define QVX_READ(DD)                                                                     \
    if (L.d == DD && each == 1) kv_read_q4_kernel<DD, 1><<<grid, 256, 0, s>>>(a, n_row); \
    if (L.d == DD && each == 4) kv_read_q4_kernel<DD, 4><<<grid, 256, 0, s>>>(a, n_row);
        QVX_READ(64)
        QVX_READ(128)
        QVX_READ(256)
#undef QVX_READ
        return check_cuda(dev, cudaGetLastError(), "4-bit kv read launch");
    }
    const uint32_t width = L.d % 8 == 0 ? 8 : 1;
    const uint64_t threads = (uint64_t)n * 2u * L.kvh * (L.d / width), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffull) return fail(dev, QVX_ERR_CORE, "kv read: %zu rows are too many for one launch", n);
    LaunchTimer timer(dev, QVX_K_COPY, s);
    if (width == 8) kv_read_kernel<8><<<(unsigned)grid, 256, 0, s>>>(a);
    else kv_read_kernel<1><<<(unsigned)grid, 256, 0, s>>>(a);
    return check_cuda(dev, cudaGetLastError(), "kv read launch");
}

}  // namespace qvx
