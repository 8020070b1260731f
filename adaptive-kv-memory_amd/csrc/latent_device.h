// Device helpers shared by the kernels over the paged latent cache.
#pragma once

#include "akv_common.h"
#include "latent.h"
#include "paged_device.h"
#include "tile_common.h"

namespace akv {
namespace {

// p is held times 2^13 and the running maximum may lag behind by two log2 units: p in (0, 2^15] keeps
// 11 bits down to 2^-27 of the largest weight.
constexpr float kBias = 13.0f, kLagBy = 2.0f;

__device__ __forceinline__ float qmax(float x) {  // over the four lanes of a row
    x = __builtin_fmaxf(x, __shfl_xor(x, 16));
    return __builtin_fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float qsum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// LDS holds a cached row as it is, its 16-byte chunks in another order: chunk c lies at c ^ turn(row),
// so that eight rows read at one chunk (rows lie 64 or 128 bytes apart modulo the banks), and the
// transposed reads of four rows at two chunks, fall on different banks.
__device__ __forceinline__ int turn(int row) { return (row & 2) << 1 | (row & 4) >> 1; }

// 1 KiB: 16 bytes of each lane, from buffer offset voff, to LDS [lds, lds + 1024).
__device__ __forceinline__ void dma_kib(u4 rsrc, uint32_t lds, uint32_t voff) {
    uint32_t m0;
    asm volatile("s_mov_b32 %[m0], m0\n\ts_mov_b32 m0, %[lds]\n\ts_nop 3\n\t"
                 "buffer_load_dwordx4 %[v], %[r], 0 offen lds\n\ts_mov_b32 m0, %[m0]"
                 : [m0] "=&s"(m0) : [lds] "s"(lds), [r] "s"(rsrc), [v] "v"(voff) : "memory");
}
// A buffer of `bytes` at `at`, which are one for the whole wave.
__device__ __forceinline__ u4 wave_rsrc(const unsigned char *at, int bytes) {
    u4 r = rsrc4(at, (uint32_t)bytes);
#pragma unroll
    for (int i = 0; i < 3; ++i) r[i] = (uint32_t)__builtin_amdgcn_readfirstlane((int)r[i]);
    return r;
}

typedef short s4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u2 read_transposed(uint32_t lds) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)(size_t)lds));
}

// The parts of the cache that a wave loads: 1 KiB pieces of tiles of 16 rows.
template <int DC>
struct Rows16 {
    static constexpr int ROWB = 2 * (DC + kLatentRope), BYTES = 16 * ROWB, PIECES = BYTES / 1024;
    // Offset in the tile of what a lane loads of a piece: LDS takes the pieces in a row.
    static __device__ __forceinline__ uint32_t offset(int piece, int lane) {
        const int c = 64 * piece + lane, row = c / (ROWB / 16), at = c - row * (ROWB / 16);
        return row * ROWB + ((at ^ turn(row)) << 4);
    }
};

// Where the tiles of a sequence lie, 64 pages of its table in a wave's lanes.
struct Pages {
    const int32_t *table;
    int width, first, ids;
    __device__ __forceinline__ void fill(int page) {
        first = page;
        ids = page + (int)(threadIdx.x & 63) < width ? table[page + (threadIdx.x & 63)] : -1;
        asm volatile("" : "+v"(ids));  // waited for here
    }
    __device__ __forceinline__ uint32_t at(int page) {
        if (page - first >= 64 || page < first) fill(page);
        return (uint32_t)__builtin_amdgcn_readlane(ids, page - first);
    }
};
// The tile of 16 rows from token `k` of kv on as a buffer: slots that hold no token are past its end,
// and come as zeros whatever is in them (0 times what is not finite would be NaN in rows that do not
// see them).
struct Tile {
    const unsigned char *at;
    int rows;
    bool there;
};
__device__ __forceinline__ Tile tile_at(const LatentView &v, Pages &pages, int k, int kv) {
    uint32_t page = k < kv ? pages.at(k >> v.log_page) : ~0u;
    Tile t;
    t.there = page < v.n_pages;
    t.rows = t.there ? min(kv - k, 16) : 0;
    if (!t.there) page = 0;
    t.at = v.base + (int64_t)page * v.page_bytes + (int64_t)(k & ((1 << v.log_page) - 1)) * v.row_bytes;
    return t;
}

// Eight values of a query row as float.
__device__ __forceinline__ float query_value(u4 w, int e, bool bf16) {
    const uint32_t v = w[e >> 1];
    return bf16 ? __builtin_bit_cast(float, e & 1 ? v & 0xffff0000u : v << 16) : (float)as_h2(v)[e & 1];
}
// A row enters times 2^(14 - exponent), its largest then in [2^13, 2^14) (less where that is below
// 2^-60), and its scores times the factor are in the log2 domain.
__device__ __forceinline__ int row_exponent(float top) { return top > 0.0f ? max(__builtin_amdgcn_frexp_expf(top), -60) : 14; }
__device__ __forceinline__ float row_factor(float scale_log2, int ex) { return __builtin_fmaxf(__builtin_ldexpf(scale_log2, ex - 14), 0x1p-126f); }
template <int N, typename Value>
__device__ __forceinline__ float scaled_row(h8 (&op)[N], Value value, float scale_log2) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf(value(i, e)));
    const int ex = row_exponent(qmax(top));
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) op[i][e] = (_Float16)__builtin_ldexpf(value(i, e), 14 - ex);
    return row_factor(scale_log2, ex);
}

}  // namespace
}  // namespace akv
