// Device helpers shared by the kernels over the paged latent cache.
#pragma once

#include <type_traits>

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

// 1 KiB: 16 bytes of each lane, from buffer offset voff + soff, to LDS [lds, lds + 1024).
__device__ __forceinline__ void dma_kib(u4 rsrc, uint32_t lds, uint32_t voff, uint32_t soff = 0) {
    uint32_t m0;
    asm volatile("s_mov_b32 %[m0], m0\n\ts_mov_b32 m0, %[lds]\n\ts_nop 3\n\t"
                 "buffer_load_dwordx4 %[v], %[r], %[s] offen lds\n\ts_mov_b32 m0, %[m0]"
                 : [m0] "=&s"(m0) : [lds] "s"(lds), [r] "s"(rsrc), [v] "v"(voff), [s] "s"(soff) : "memory");
}
// A buffer of `bytes` at `at`, which are one for the whole wave.
__device__ __forceinline__ u4 wave_rsrc(const unsigned char *at, int bytes) {
    u4 r = rsrc4(at, (uint32_t)bytes);
#pragma unroll
    for (int i = 0; i < 3; ++i) r[i] = (uint32_t)__builtin_amdgcn_readfirstlane((int)r[i]);
    return r;
}

// The lane's number, computed where it is asked for: what follows from it is not kept in registers over a
// loop that has none left (a register that is spilled costs a wait for all loads in flight).
__device__ __forceinline__ int lane_again() {
    int x;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
    return x;
}
template <typename T>
__device__ __forceinline__ __attribute__((address_space(3))) T *lds_mut(uint32_t a) {
    return (__attribute__((address_space(3))) T *)(size_t)a;
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

// A tile of 16 rows to LDS: a loop, whose code is a tenth of its instructions.
template <int DC>
__device__ __forceinline__ void load_tile(u4 rsrc, uint32_t lds, int lane) {
    using T = Rows16<DC>;
    constexpr int CH = T::ROWB / 16;
    int row = lane / CH, at = lane - row * CH;  // of the lane's chunk
#pragma unroll 1
    for (int i = 0; i < T::PIECES; ++i) {
        dma_kib(rsrc, lds + i * 1024, row * T::ROWB + ((at ^ turn(row)) << 4));
        at += 64;
        if (at >= CH) at -= CH, ++row;
        if (CH < 64 && at >= CH) at -= CH, ++row;
    }
}

// Where the tiles of a sequence lie, 64 pages of its table in a wave's lanes.
struct Pages {
    const int32_t *table;
    int width, first, ids;
    __device__ __forceinline__ void fill(int page) {
        first = __builtin_amdgcn_readfirstlane(page);
        const int at = page + lane_again();
        ids = at < width ? table[at] : -1;
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
    k = __builtin_amdgcn_readfirstlane(k), kv = __builtin_amdgcn_readfirstlane(kv);
    uint32_t page = k < kv ? pages.at(k >> v.log_page) : ~0u;
    Tile t;
    t.there = page < v.n_pages;
    t.rows = t.there ? min(kv - k, 16) : 0;
    if (!t.there) page = 0;
    t.at = v.base + (int64_t)page * v.page_bytes + (int64_t)(k & ((1 << v.log_page) - 1)) * v.row_bytes;
    return t;
}

// Two outputs, rounded to the nearest.
__device__ __forceinline__ uint32_t out_pair(bool bf16, float a, float b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    return bf16 ? __builtin_bit_cast(uint32_t, (bf2){(__bf16)a, (__bf16)b}) : as_u32((h2){(_Float16)a, (_Float16)b});
}

// A query row as the operand of the first product, N pieces of eight channels a lane.  float16 enters as it
// is.  bfloat16 enters as float16 times 2^(14 - exponent), its largest then in [2^13, 2^14) (less where that
// is below 2^-60), which its scores' factor takes back.  Returns the factor that turns scores to the log2 domain.
__device__ __forceinline__ int row_exponent(uint32_t top_bf16) {  // of the largest's bits without its sign
    const float top = __builtin_bit_cast(float, top_bf16 << 16);
    return top > 0.0f ? max(__builtin_amdgcn_frexp_expf(top), -60) : 14;
}
__device__ __forceinline__ float row_factor(float scale_log2, int ex) { return __builtin_fmaxf(__builtin_ldexpf(scale_log2, ex - 14), 0x1p-126f); }
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
template <int N>
__device__ __forceinline__ us2 largest(const u4 (&w)[N]) {
    us2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, (uint32_t)w[i][e] & 0x7fff7fffu));
    return top;
}
// Two bfloat16 times x as float16.
__device__ __forceinline__ uint32_t scaled_pair(uint32_t w, float x) {
    const float lo = __builtin_fmaf(__builtin_bit_cast(float, w << 16), x, -0.0f), hi = __builtin_fmaf(__builtin_bit_cast(float, w & 0xffff0000u), x, -0.0f);
    return as_u32((h2){(_Float16)lo, (_Float16)hi});
}
template <int N>
__device__ __forceinline__ float query_operand(h8 (&op)[N], const u4 (&w)[N], int bf16, float scale_log2) {
    if (!bf16) {
#pragma unroll
        for (int i = 0; i < N; ++i) op[i] = __builtin_bit_cast(h8, w[i]);
        return __builtin_fmaxf(scale_log2, 0x1p-126f);
    }
    const us2 t = largest(w);
    uint32_t top = max(t[0], t[1]);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const int ex = row_exponent(top);
    const float x = __builtin_ldexpf(1.0f, 14 - ex);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        u4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = scaled_pair(w[i][e], x);
        op[i] = __builtin_bit_cast(h8, o);
    }
    return row_factor(scale_log2, ex);
}

}  // namespace
}  // namespace akv
