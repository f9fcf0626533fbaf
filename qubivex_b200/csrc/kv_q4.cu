// KV sync and KV append of a 4-bit pool, and rows of any pool read back.
//
// Store: a thread takes four consecutive elements of a row; eight neighbouring lanes hold a group of 32, find its least
// and greatest value by shuffles, and each writes its four codes (16 bits); the first of the eight writes the group's
// step and offset.  Every store is the group's own bytes, so rows of one tile may be written by any blocks in any order.
// Bound by HBM: 4 + 5/8 bytes per element.
//
// Read: a thread takes eight consecutive elements (one word of codes, or two half words; one 16-byte chunk of a 16-bit
// row) and writes them in the type asked for.  5/8 + 2 bytes per element from a 4-bit pool to 16-bit rows.
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
    uint32_t n, pool_blocks;
    uint32_t aligned;  // the rows can be read 16 bytes at a time
    int* status;
};

__global__ void __launch_bounds__(256) kv_rows_q4_kernel(Q4RowArgs a) {
    const uint32_t d4 = a.L.d >> 2, per_row = 2u * a.L.kvh * d4;
    const uint64_t idx = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    // (per_row is a multiple of 32, so the eight lanes of a group are always in the same row)
    const uint64_t row = idx / per_row;
    const bool live = row < a.n;
    const uint32_t r = live ? (uint32_t)row : 0u, w = (uint32_t)(idx - row * per_row);
    const uint32_t kv = w / (a.L.kvh * d4), e = w % (a.L.kvh * d4), g = e / d4, j = e % d4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t block = 0, slot = 0;
    bool store = live;
    if (live) {
        const float* src = (kv ? a.v_rows : a.k_rows) + (size_t)r * a.row_stride + 4u * e;
        x = a.aligned ? *reinterpret_cast<const float4*>(src) : make_float4(src[0], src[1], src[2], src[3]);
        const uint32_t p = a.at_direct ? a.at_direct[r] : a.pos[r];
        if (p == 0xffffffffu) store = false;
        else if (a.at_direct) { block = p / a.L.B; slot = p % a.L.B; }
        else { block = a.blocks[a.table_at[r] + p / a.L.B]; slot = p % a.L.B; }
        if (store && block >= a.pool_blocks) { atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL); store = false; }
    }
    __half step, offset;
    const uint32_t codes = q4_quantise(x, step, offset);
    if (!store) return;
    uint8_t* tile = a.pool + (uint64_t)block * a.L.block_bytes + (uint64_t)g * 2u * a.L.page_bytes +
                    (uint64_t)(slot / Q4_TILE) * q4_tile_bytes(a.L.d);
    const uint32_t s = slot % Q4_TILE;
    *reinterpret_cast<uint16_t*>(tile + q4_codes_at(a.L.d, s, kv, j)) = (uint16_t)codes;
    if ((j & 7u) == 0u) {
        *reinterpret_cast<__half*>(tile + q4_step_at(a.L.d, s, kv, j >> 3)) = step;
        *reinterpret_cast<__half*>(tile + q4_offset_at(a.L.d, s, kv, j >> 3)) = offset;
    }
}

int32_t launch_kv_rows_q4(qvx_device* dev, const Layout& L, void* pool, const float* k_rows, const float* v_rows,
                          size_t row_stride_f32, const uint32_t* at_direct, const uint32_t* pos, const uint32_t* blocks,
                          const uint32_t* table_at, size_t n, size_t pool_blocks, int kind, cudaStream_t s) {
    if (n > 0x7fffffffu) return fail(dev, QVX_ERR_CORE, "kv rows: %zu rows do not fit 31 bits", n);
    const uint64_t threads = (uint64_t)n * 2u * L.kvh * (L.d / 4), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffull) return fail(dev, QVX_ERR_CORE, "kv rows: %zu rows are too many for one launch", n);
    const bool aligned = (((uintptr_t)k_rows | (uintptr_t)v_rows) & 15u) == 0 && row_stride_f32 % 4 == 0;
    Q4RowArgs a{L, (uint8_t*)pool, k_rows, v_rows, row_stride_f32, at_direct, pos, blocks, table_at, (uint32_t)n,
                (uint32_t)std::min<size_t>(pool_blocks, 0xffffffffu), aligned ? 1u : 0u, device_status_word(dev)};
    LaunchTimer timer(dev, kind, s);
    kv_rows_q4_kernel<<<(unsigned)grid, 256, 0, s>>>(a);
    return check_cuda(dev, cudaGetLastError(), "4-bit kv rows launch");
}

struct ReadArgs {
    Layout L;
    const uint8_t* pool;
    const uint32_t* from;
    void* rows;
    uint32_t n, pool_blocks, rows_dtype;
    uint32_t wide;  // rows can be written 16 bytes at a time
    int* status;
};

// `width` consecutive elements per thread: 8, or 1 where d is not a multiple of 8.
template <int WIDTH>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
    const uint32_t per_head = a.L.d / WIDTH, per_row = 2u * a.L.kvh * per_head;
    const uint64_t idx = (uint64_t)blockIdx.x * 256u + threadIdx.x, row = idx / per_row;
    if (row >= a.n) return;
    const uint32_t r = (uint32_t)row, w = (uint32_t)(idx - row * per_row);
    const uint32_t kv = w / (a.L.kvh * per_head), e = w % (a.L.kvh * per_head), g = e / per_head, i = e % per_head * WIDTH;
    const uint32_t p = a.from[r];
    if (p == 0xffffffffu) return;
    const uint32_t block = p / a.L.B, slot = p % a.L.B;
    if (block >= a.pool_blocks) { atomicExch(a.status, STATUS_BLOCK_OUT_OF_POOL); return; }
    const uint8_t* b = a.pool + (uint64_t)block * a.L.block_bytes;
    float x[WIDTH];
    if (a.L.dtype == QVX_Q4) {
        if constexpr (WIDTH == 8) {  // (d is a multiple of 8 in every 4-bit pool)
            const uint8_t* tile = b + (uint64_t)g * 2u * a.L.page_bytes + (uint64_t)(slot / Q4_TILE) * q4_tile_bytes(a.L.d);
            const uint32_t s = slot % Q4_TILE, d = a.L.d, j = i >> 2, grp = i / Q4_GROUP;
            const uint32_t c = *reinterpret_cast<const uint16_t*>(tile + q4_codes_at(d, s, kv, j)) |
                               (uint32_t)*reinterpret_cast<const uint16_t*>(tile + q4_codes_at(d, s, kv, j + 1)) << 16;
            const float step = __half2float(*reinterpret_cast<const __half*>(tile + q4_step_at(d, s, kv, grp)));
            const float off = __half2float(*reinterpret_cast<const __half*>(tile + q4_offset_at(d, s, kv, grp)));
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = fmaf(step, (float)((c >> (4 * k)) & 15u), off);
        }
    } else {
#pragma unroll
        for (int k = 0; k < WIDTH; k++) {
            const uint8_t* at = b + in_block_offset(a.L, slot, kv, g, i + k);
            x[k] = a.L.dtype == QVX_F32 ? *reinterpret_cast<const float*>(at) : widen16(*reinterpret_cast<const uint16_t*>(at), a.L.dtype);
        }
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

int32_t launch_kv_read(qvx_device* dev, const Layout& L, const void* pool, size_t pool_blocks, const uint32_t* from, size_t n,
                       void* rows, uint32_t rows_dtype, cudaStream_t s) {
    if (n == 0) return QVX_OK;
    if (n > 0x7fffffffu) return fail(dev, QVX_ERR_CORE, "kv read: %zu rows do not fit 31 bits", n);
    const uint32_t width = L.d % 8 == 0 ? 8 : 1;
    const uint64_t threads = (uint64_t)n * 2u * L.kvh * (L.d / width), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffull) return fail(dev, QVX_ERR_CORE, "kv read: %zu rows are too many for one launch", n);
    ReadArgs a{L, (const uint8_t*)pool, from, rows, (uint32_t)n, (uint32_t)std::min<size_t>(pool_blocks, 0xffffffffu), rows_dtype,
               ((uintptr_t)rows & 15u) == 0 ? 1u : 0u, device_status_word(dev)};
    LaunchTimer timer(dev, QVX_K_COPY, s);
    if (width == 8) kv_read_kernel<8><<<(unsigned)grid, 256, 0, s>>>(a);
    else kv_read_kernel<1><<<(unsigned)grid, 256, 0, s>>>(a);
    return check_cuda(dev, cudaGetLastError(), "kv read launch");
}

}  // namespace qvx
