// The paged 4-bit cache's data movement: append (quantize into slots), read (values out of
// slots), copies of whole pages and the compaction of sequences to the tokens that stay.
// All of it is bound by memory; the tile layout is written out in akv_hip.h.
#include <algorithm>

#include "akv_common.h"
#include "paged.h"

namespace akv {
namespace {

constexpr float kTop = 61440.0f;  // appended values are clamped to this: 15 * scale + zero stays below 65504

// float64 -> float16, rounded once: the float32 between is rounded towards zero and its last
// bit set if anything was cut off, so that the second rounding sees on which side of a tie
// the value lies.
__device__ __forceinline__ _Float16 round16(double d) {
    float f = (float)d;
    uint32_t u = __builtin_bit_cast(uint32_t, f);
    if ((double)f != d) {
        if (__builtin_fabs((double)f) > __builtin_fabs(d)) --u;
        u |= 1u;
    }
    return (_Float16)__builtin_bit_cast(float, u);
}

// (hi - lo) / 15 as exact arithmetic rounds it to float16.  The float32 quotient is within four
// of its units of the true one; float64 decides where a float16 tie may lie between them, and
// below float16's normal range, where ties lie elsewhere.
__device__ __forceinline__ _Float16 scale_of(float hi, float lo) {
    const float f = (hi - lo) * (1.0f / 15.0f);
    const uint32_t from_tie = (__builtin_bit_cast(uint32_t, f) + 0x1000u + 4u) & 0x1fffu;
    // (asked of the whole wave: the compiler would compute both sides always)
    if (__builtin_amdgcn_ballot_w64(from_tie <= 8u || f < 0x1p-14f)) return round16(((double)hi - (double)lo) / 15.0);
    return (_Float16)f;
}

// Codes of eight values: (x - z) / s rounded to the nearest whole number, ties to even, as
// exact arithmetic has it, within 0..15.  The float32 quotient is within 8e-6 of the true one
// (below 16, four roundings); where that leaves the side of a border open float64 decides.
// Nibble e of the result is value e.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float z, float s) {
    const float inv = __builtin_amdgcn_rcpf(s);
    float c[8], far = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float r = (x[e] - z) * inv;
        c[e] = __builtin_rintf(r);
        far = __builtin_fmaxf(far, __builtin_fabsf(r - c[e]));
    }
    if (__builtin_amdgcn_ballot_w64(far > 0.5f - 2e-5f))
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = (float)__builtin_rint(((double)x[e] - (double)z) / (double)s);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = __builtin_amdgcn_fmed3f(c[e], 0.0f, 15.0f);
    // four digits to the base 16 are exact in float32
    const float a = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]);
    const float b = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]);
    return (uint32_t)a | ((uint32_t)b << 16);
}

// x combined with that of the lanes of its group (4, 8 or 16 of them) by DPP.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <bool MAX>
__device__ __forceinline__ float pick(float a, float b) {  // NaN stays
    return MAX ? __builtin_elementwise_maximum(a, b) : __builtin_elementwise_minimum(a, b);
}
template <bool MAX>
__device__ __forceinline__ float over_group(float x, int log_lanes) {
    x = pick<MAX>(x, dpp<0xB1>(x));                  // neighbours
    x = pick<MAX>(x, dpp<0x4E>(x));                  // pairs of a quad
    if (log_lanes >= 3) x = pick<MAX>(x, dpp<0x141>(x)); // quads of a half row (mirrored: a quad's lanes agree)
    if (log_lanes >= 4) x = pick<MAX>(x, dpp<0x140>(x));
    return x;
}

// Sequence of each lane's token t: the number of sequences that end at or before it.
__device__ __forceinline__ int seq_of(const PagedSeqs &q, int t, bool live) {
    const int lane = threadIdx.x & 63;
    const int first = __builtin_amdgcn_readfirstlane(t);
    const int last = __builtin_amdgcn_readlane(t, 63);
    int n = 0;
    for (int s0 = 0; s0 < q.n_seqs; s0 += 64) {
        const int end = s0 + lane < q.n_seqs ? q.q_starts[s0 + lane + 1] : 0x7fffffff;
        for (int tt = first; tt <= last; ++tt) {
            const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= tt));
            if (tt == t) n += c;
        }
    }
    return live && n < q.n_seqs ? n : -1;
}

// Where the rows of token t lie: the tile of head 0, the next head's distance, the token in it.
struct Slot {
    unsigned char *page;  // null: the token has no slot
    int64_t head_bytes;
    int tok;
};
__device__ __forceinline__ Slot slot_of(const PagedRowsParams &p, int t, bool live) {
    const int tile_bytes = paged_tile_bytes(p.D, p.ng), log_page = p.pool.log_tpp + 4;
    Slot at{nullptr, (int64_t)tile_bytes << p.pool.log_tpp, 0};
    const int s = seq_of(p.seqs, t, live);
    if (s < 0) return at;
    const SeqRows r = seq_rows(p.seqs, s, log_page);
    const int64_t pos = (int64_t)r.at + (t - r.begin);
    if (t < r.begin || t >= r.begin + r.n || pos < 0 || pos >> log_page >= p.seqs.width) return at;
    const uint32_t page = (uint32_t)p.seqs.table[s * p.seqs.table_stride + (pos >> log_page)];
    if (page >= p.pool.n_pages) return at;
    at.page = p.pool.base + page * p.pool.page_bytes + (int64_t)((int)(pos >> 4) & ((1 << p.pool.log_tpp) - 1)) * tile_bytes;
    at.tok = (int)(pos & 15);
    return at;
}

template <int DT>
struct Raw8 {  // eight values as they come
    u4 a, b;
    __device__ __forceinline__ void load(const unsigned char *p) {
        a = *(const u4 *)p;
        if constexpr (DT == AKV_DT_F32) b = ((const u4 *)p)[1];
    }
    __device__ __forceinline__ void to(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = a[i];
            if constexpr (DT == AKV_DT_F32) {
                x[i] = __builtin_bit_cast(float, w);
                x[4 + i] = __builtin_bit_cast(float, (uint32_t)b[i]);
            } else if constexpr (DT == AKV_DT_F16) {
                x[2 * i] = (float)as_h2(w)[0], x[2 * i + 1] = (float)as_h2(w)[1];
            } else {
                x[2 * i] = __builtin_bit_cast(float, w << 16);
                x[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
            }
        }
    }
};

template <int DT>
__device__ __forceinline__ void store8(unsigned char *p, const float *x) {
    if constexpr (DT == AKV_DT_F32) {
        ((f4 *)p)[0] = (f4){x[0], x[1], x[2], x[3]};
        ((f4 *)p)[1] = (f4){x[4], x[5], x[6], x[7]};
    } else {
        u4 a;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == AKV_DT_F16) a[i] = as_u32((h2){(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
            else a[i] = f32_to_bf16_rne(x[2 * i]) | ((uint32_t)f32_to_bf16_rne(x[2 * i + 1]) << 16);
        }
        *(u4 *)p = a;
    }
}

// Bytes (g of d[0], g of d[1], ...) of up to four dwords.
__device__ __forceinline__ uint32_t byte_of(uint32_t d, int g) { return (d >> (8 * g)) & 255u; }

// Byte offset in a tile of the 16-bit piece (quad, row, pair, half, parity) of the V codes.
template <int D>
__device__ __forceinline__ int v_piece(int tok, int r, int h) {
    return 8 * D + (((tok >> 2) * 16 + r) * 2 + ((tok >> 1) & 1)) * (D / 16) + h * 4 + (tok & 1) * 2;
}
template <int D>
__device__ __forceinline__ int v_meta(int tok, int grp, int ng) {
    return 16 * D + 64 * ng + (((tok >> 2) * ng + grp) * 4 + (tok & 3)) * 2;
}

}  // namespace

// Append and read.  A lane holds 8 channels 32 g + 8 i .. of one side of one (token, head); D / 8
// lanes a side, both sides next to each other, IT such sets of rows a wave: rows of one token
// look their slot up once.  Group minima and maxima by DPP.  A V row's bytes are dealt to 16
// places of its tile, so four lanes (i of every g) transpose their 4 x 4 bytes and move 16-bit
// pieces.  Bound by memory for prompts (IT = 4: 13800 tokens of 8 heads, float16, 74 MB: append 24 us,
// 3.1 TB/s, the rest the quantizer's vector instructions, read 19 us, 3.9 TB/s) and by latency for a
// decode step (IT = 1: 48 tokens, 2.8 us and 2.2 us).
template <int D, int DT, int IT>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedRowsParams p) {
    constexpr int LN = D / 8, PW = 32 / LN;  // lanes a side, rows of a wave's set
    const uint32_t lane = threadIdx.x & 63, H = p.pool.heads, n_pairs = (uint32_t)p.seqs.n_tokens * H;
    const uint32_t first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (PW * IT);
    if (first >= n_pairs) return;
    const int side = (lane / LN) & 1, b = lane & (LN - 1), g = b >> 2, i = b & 3;
    uint32_t pair = first + lane / (2 * LN);
    uint32_t t = pair / H, h = pair - t * H;
    const int ng = p.ng, ll = p.log_lanes, grp = b >> ll;
    const unsigned char *src = (side ? p.v : p.k) + b * (DT == AKV_DT_F32 ? 32 : 16);
    const int64_t st = side ? p.v_t : p.k_t, sh = side ? p.v_h : p.k_h;
    // the slot first: loads return in order, and its three would wait behind the rows
    Slot at = slot_of(p, t, pair < n_pairs);
    Raw8<DT> raw[IT];
    uint32_t tt = t, hh = h;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const bool live = pair + it * PW < n_pairs;  // others read the last row
        raw[it].load(src + (live ? tt : (uint32_t)p.seqs.n_tokens - 1) * st + (live ? hh : H - 1) * sh);
        hh += PW;
        while (hh >= H) hh -= H, ++tt;
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        if (it > 0) {
            const uint32_t was = t;
            pair += PW;
            h += PW;
            while (h >= H) h -= H, ++t;
            if (__builtin_amdgcn_ballot_w64(t != was)) at = slot_of(p, t, pair < n_pairs);
        }
        float x[8];
        raw[it].to(x);
        float lo = pick<false>(pick<false>(pick<false>(x[0], x[1]), pick<false>(x[2], x[3])),
                               pick<false>(pick<false>(x[4], x[5]), pick<false>(x[6], x[7])));
        float hi = pick<true>(pick<true>(pick<true>(x[0], x[1]), pick<true>(x[2], x[3])),
                              pick<true>(pick<true>(x[4], x[5]), pick<true>(x[6], x[7])));
        lo = over_group<false>(lo, ll);
        hi = over_group<true>(hi, ll);
        const bool bad = !(__builtin_fabsf(lo) < INFINITY && __builtin_fabsf(hi) < INFINITY);
        // values past the clamp get the end's code by themselves
        lo = __builtin_amdgcn_fmed3f(lo, -kTop, kTop);
        hi = __builtin_amdgcn_fmed3f(hi, -kTop, kTop);
        const _Float16 s16 = scale_of(hi, lo), z16 = (_Float16)lo;
        const float s = (float)s16, z = (float)z16;
        const uint32_t w = s == 0.0f || bad ? 0u : codes_of(x, z, s);
        const uint32_t sb = bad ? 0x7e00u : __builtin_bit_cast(uint16_t, s16);
        const uint32_t zb = bad ? 0x7e00u : __builtin_bit_cast(uint16_t, z16);
        uint32_t d[4];
#pragma unroll
        for (int q = 0; q < D / 32; ++q) d[q] = __shfl(w, (lane & ~(LN - 1)) + 4 * q + i);
        if (!at.page) continue;
        unsigned char *tile = at.page + h * at.head_bytes;
        const int tok = at.tok;
        const bool lead = (b & ((1 << ll) - 1)) == 0;
        if (side == 0) {
            *(uint32_t *)(tile + tok * (D / 2) + (i * (D / 32) + g) * 4) = w;
            if (lead) *(uint32_t *)(tile + 16 * D + (tok * ng + grp) * 4) = sb | (zb << 16);
        } else {
            if constexpr (D == 128) {
                const int r = 4 * i + g;
                *(uint16_t *)(tile + v_piece<D>(tok, r, 0)) = byte_of(d[0], g) | (byte_of(d[1], g) << 8);
                *(uint16_t *)(tile + v_piece<D>(tok, r, 1)) = byte_of(d[2], g) | (byte_of(d[3], g) << 8);
            } else {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const int k = 2 * g + m;
                    *(uint16_t *)(tile + v_piece<D>(tok, 4 * i + k, 0)) = byte_of(d[0], k) | (byte_of(d[1], k) << 8);
                }
            }
            if (lead) {
                *(uint16_t *)(tile + v_meta<D>(tok, grp, ng)) = sb;
                *(uint16_t *)(tile + v_meta<D>(tok, grp, ng) + 32 * ng) = zb;
            }
        }
    }
}

template <int D, int DT, int IT>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedRowsParams p) {
    constexpr int LN = D / 8, PW = 32 / LN;
    const uint32_t lane = threadIdx.x & 63, H = p.pool.heads, n_pairs = (uint32_t)p.seqs.n_tokens * H;
    const uint32_t first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (PW * IT);
    if (first >= n_pairs) return;
    const int side = (lane / LN) & 1, b = lane & (LN - 1), g = b >> 2, i = b & 3;
    uint32_t pair = first + lane / (2 * LN);
    uint32_t t = pair / H, h = pair - t * H;
    const int ng = p.ng, grp = b >> p.log_lanes;
    unsigned char *dst = side ? p.v : p.k;
    const int64_t st = side ? p.v_t : p.k_t, sh = side ? p.v_h : p.k_h;
    Slot at = slot_of(p, t, pair < n_pairs);
    uint32_t w[IT], sz[IT], row_t[IT], row_h[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        if (it > 0) {
            const uint32_t was = t;
            pair += PW;
            h += PW;
            while (h >= H) h -= H, ++t;
            if (__builtin_amdgcn_ballot_w64(t != was)) at = slot_of(p, t, pair < n_pairs);
        }
        row_t[it] = t;
        row_h[it] = h;
        w[it] = sz[it] = 0;
        if (at.page) {
            const unsigned char *tile = at.page + h * at.head_bytes;
            const int tok = at.tok;
            if (side == 0) {
                w[it] = *(const uint32_t *)(tile + tok * (D / 2) + (i * (D / 32) + g) * 4);
                sz[it] = *(const uint32_t *)(tile + 16 * D + (tok * ng + grp) * 4);
            } else {
                // bytes g of row r = 4 i + g (D = 128) or of rows 4 i + 2 g, + 1 (D = 64)
                const int r = D == 128 ? 4 * i + g : 4 * i + 2 * g;
                w[it] = *(const uint16_t *)(tile + v_piece<D>(tok, r, 0)) |
                        ((uint32_t)*(const uint16_t *)(tile + (D == 128 ? v_piece<D>(tok, r, 1) : v_piece<D>(tok, r + 1, 0))) << 16);
                sz[it] = *(const uint16_t *)(tile + v_meta<D>(tok, grp, ng)) |
                         ((uint32_t)*(const uint16_t *)(tile + v_meta<D>(tok, grp, ng) + 32 * ng) << 16);
            }
        }
    }
    pair -= (IT - 1) * PW;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        uint32_t d[4], c = w[it];
#pragma unroll
        for (int q = 0; q < D / 32; ++q) d[q] = __shfl(c, (lane & ~(LN - 1)) + 4 * q + i);
        if (side == 1) {
            if constexpr (D == 128)  // row 4 i + q has this lane's group in byte g
                c = byte_of(d[0], g) | (byte_of(d[1], g) << 8) | (byte_of(d[2], g) << 16) | (byte_of(d[3], g) << 24);
            else                     // rows 4 i + 2 q, + 1 of lane q: this lane's group in bytes g and 2 + g
                c = byte_of(d[0], g) | (byte_of(d[0], 2 + g) << 8) | (byte_of(d[1], g) << 16) | (byte_of(d[1], 2 + g) << 24);
        }
        const float s = (float)as_h2(sz[it])[0], z = (float)as_h2(sz[it])[1];
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf((float)((c >> (4 * e)) & 15u), s, z);
        if (pair + it * PW < n_pairs)
            store8<DT>(dst + row_t[it] * st + row_h[it] * sh + b * (DT == AKV_DT_F32 ? 32 : 16), x);
    }
}

// 16-byte pieces of the pages of all pairs and layers, four a thread; bound by memory (777 pages of
// 8 layers, read and written once each: 38 us, more than memory's rate, as the cache behind L2
// holds some of it; four pages of 28 layers, 3.5 us).
__global__ __launch_bounds__(256) void paged_copy_kernel(const PagedCopyParams p) {
    const int64_t per = p.page_bytes >> 4;  // pieces a page
    const int64_t total = per * p.n * p.layers;
    u4 v[4];
    u4 *to[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t u = ((int64_t)blockIdx.x * 4 + k) * 256 + threadIdx.x;
        to[k] = nullptr;
        if (u < total) {
            const int64_t page = u / per, off = u - page * per;
            const int64_t layer = page / p.n, i = page - layer * p.n;
            const uint32_t a = (uint32_t)p.src[i], b = (uint32_t)p.dst[i];
            if (a < p.n_pages && b < p.n_pages && a != b) {
                unsigned char *base = p.data + layer * p.n_pages * p.page_bytes;
                v[k] = ((const u4 *)(base + a * p.page_bytes))[off];
                to[k] = (u4 *)(base + b * p.page_bytes) + off;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (to[k]) *to[k] = v[k];
}

// One wave a tile of the destination: its 16 rows come from up to 16 tiles.  Lane (row t of
// the tile, i) of the K codes, lane (quad a, row r) of the V codes as they are stored; whole
// tiles leave in 16-byte stores, the last one of a sequence row by row.  Bound by memory: half of 16
// sequences of 1000 to 16384 tokens, 4 layers of 8 heads, 122 us, 3.9 TB/s read and written (tiles
// whose rows lie in two of the source read both whole); a quarter of 4095 tokens in 28 layers 5.4 us.
template <int D, int NG>
__global__ __launch_bounds__(256) void paged_compact_kernel(const PagedCompactParams p) {
    constexpr int TB = paged_tile_bytes(D, NG), VW = D / 64;  // dwords a token pair of a V row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int H = p.pool.heads;
    // z: layer, y: sequence, x: (tile of the longest row, head), heads next to each other
    const int layer = blockIdx.z, s = blockIdx.y;
    const int64_t x = (int64_t)blockIdx.x * 4 + wave;
    const int64_t tile_no = x / H;
    const int h = (int)(x - tile_no * H);
    const int log_page = p.pool.log_tpp + 4;
    int64_t n = p.n_keep[s];
    const int64_t cap = (int64_t)p.dst_width << log_page;
    n = n > p.max_keep ? p.max_keep : n;
    n = n > cap ? cap : n;
    const int64_t j0 = tile_no * 16;
    if (j0 >= n) return;
    unsigned char *base = p.pool.base + layer * p.layer_bytes;
    const uint32_t dpage = (uint32_t)p.dst_table[s * p.dst_stride + (j0 >> log_page)];
    if (dpage >= p.pool.n_pages) return;
    const int in_page = (1 << p.pool.log_tpp) - 1;
    unsigned char *dst = base + dpage * p.pool.page_bytes +
                         (((int64_t)h << p.pool.log_tpp) + ((int)tile_no & in_page)) * TB;
    // lane & 15: a row of the tile; its place in the source as a byte offset, -1 if it has none
    const int row = lane & 15;
    int64_t from = -1;
    if (j0 + row < n) {
        const int64_t pos = p.keep[s * p.keep_stride + j0 + row];
        if (pos >= 0 && pos < ((int64_t)p.src_width << log_page)) {
            const uint32_t page = (uint32_t)p.src_table[s * p.src_stride + (pos >> log_page)];
            if (page < p.pool.n_pages)
                from = (page * p.pool.page_bytes + (((int64_t)h << p.pool.log_tpp) + ((int)(pos >> 4) & in_page)) * TB) * 16 +
                       (pos & 15);
        }
    }
    const bool whole = __builtin_amdgcn_ballot_w64(from >= 0) == ~0ull;
    auto tile_of = [&](int t) { return base + (__shfl(from, t) >> 4); };
    auto tok_of = [&](int t) { return (int)(__shfl(from, t) & 15); };
    // every lane takes part in the shuffles; rows without a source read the tile they would go to
    if (from < 0) from = (int64_t)(dst - base) * 16 + row;
    const bool mine = !(from >= 0 && (base + (from >> 4)) == dst && (from & 15) == row);  // not in its place already
    if (!__builtin_amdgcn_ballot_w64(mine)) return;
    const int kt = lane >> 2, ki = lane & 3;  // K codes: token, quarter row
    const unsigned char *ksrc = tile_of(kt) + tok_of(kt) * (D / 2) + ki * (D / 8);
    const int a = lane >> 4, r = lane & 15;
    const unsigned char *vsrc[4];
    int par[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int tk = tok_of(4 * a + j);
        vsrc[j] = tile_of(4 * a + j) + 8 * D + (((tk >> 2) * 16 + r) * 2 + ((tk >> 1) & 1)) * (D / 16);
        par[j] = (tk & 1) * 16;
    }
    // meta: lane (token mt, group mg), NG groups a token
    const int mt = (lane / NG) & 15, mg = lane % NG;
    const unsigned char *mtile = tile_of(mt);
    const int mtok = tok_of(mt);
    const uint32_t km = *(const uint32_t *)(mtile + 16 * D + (mtok * NG + mg) * 4);
    const unsigned char *vm = mtile + 16 * D + 64 * NG + (((mtok >> 2) * NG + mg) * 4 + (mtok & 3)) * 2;
    const uint16_t vs = *(const uint16_t *)vm, vz = *(const uint16_t *)(vm + 32 * NG);
    uint32_t kc[D / 32];
    uint32_t vq[4][VW];
    if constexpr (D == 128) {
        const u4 x4 = *(const u4 *)ksrc;
#pragma unroll
        for (int e = 0; e < 4; ++e) kc[e] = x4[e];
    } else {
        const u2 x2 = *(const u2 *)ksrc;
        kc[0] = x2[0], kc[1] = x2[1];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (VW == 2) {
            const u2 x2 = *(const u2 *)vsrc[j];
            vq[j][0] = x2[0] >> par[j], vq[j][1] = x2[1] >> par[j];
        } else {
            vq[j][0] = *(const uint32_t *)vsrc[j] >> par[j];
        }
    }
    const bool meta_lane = lane < 16 * NG;
    if (whole) {
        if constexpr (D == 128) {
            *(u4 *)(dst + lane * 16) = (u4){kc[0], kc[1], kc[2], kc[3]};
            u4 o;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int w = 0; w < 2; ++w) o[2 * q + w] = (vq[2 * q][w] & 0xffffu) | (vq[2 * q + 1][w] << 16);
            *(u4 *)(dst + 8 * D + lane * 16) = o;
        } else {
            *(u2 *)(dst + lane * 8) = (u2){kc[0], kc[1]};
            *(u2 *)(dst + 8 * D + lane * 8) = (u2){(vq[0][0] & 0xffffu) | (vq[1][0] << 16), (vq[2][0] & 0xffffu) | (vq[3][0] << 16)};
        }
    } else {
        const uint64_t ok = __builtin_amdgcn_ballot_w64(mine);  // lanes 0-15: the rows to write
        if ((ok >> kt) & 1) {
            if constexpr (D == 128) *(u4 *)(dst + lane * 16) = (u4){kc[0], kc[1], kc[2], kc[3]};
            else *(u2 *)(dst + lane * 8) = (u2){kc[0], kc[1]};
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((ok >> (4 * a + j)) & 1) {
#pragma unroll
                for (int w = 0; w < VW; ++w)
                    *(uint16_t *)(dst + 8 * D + ((a * 16 + r) * 2 + (j >> 1)) * (D / 16) + w * 4 + (j & 1) * 2) = (uint16_t)vq[j][w];
            }
        if (!((ok >> mt) & 1)) return;
    }
    if (meta_lane) {
        *(uint32_t *)(dst + 16 * D + (mt * NG + mg) * 4) = km;
        unsigned char *o = dst + 16 * D + 64 * NG + (((mt >> 2) * NG + mg) * 4 + (mt & 3)) * 2;
        *(uint16_t *)o = vs;
        *(uint16_t *)(o + 32 * NG) = vz;
    }
}

namespace {

// Whether a call's waves take four sets of rows each: fewer waves, which have their loads in flight
// together, but leave compute units idle, and look up a slot for each of the `span` tokens in them.  By
// the waves of one set that the call has.  Append of one set a wave against four, us: head_dim 128, 8
// heads (one token): 8192, 12288, 16384 and 65536 rows 5.5, 7.0, 8.4, 22.1 and 6.5, 7.2, 7.5, 17.4; one
// head (eight): 32768, 49152, 65536 rows 11.1, 15.3, 19.8 and 12.3, 15.8, 19.4; head_dim 64, 8 heads (two):
// 24576, 32768, 49152 rows 5.8, 6.9, 9.5 and 6.7, 7.0, 8.2; 2 heads (eight): 65536, 131072 rows 10.9, 20.0
// and 11.9, 19.9.  The read crosses at the same sizes.
bool four_sets(int64_t rows, int64_t wave_rows, int64_t heads) {
    const int64_t span = std::max<int64_t>(1, 4 * wave_rows / heads);
    return rows >= 3000 * (1 + span) * wave_rows;
}

template <template <int, int, int> class K>
hipError_t rows_launch(const PagedRowsParams &p, hipStream_t s) {
    const int64_t rows = p.seqs.n_tokens * p.pool.heads;
    if (rows == 0) return hipSuccess;  // (rows of no sequence are read as 0)
    if (rows >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    const bool many = four_sets(rows, 256 / p.D, p.pool.heads);
    const int64_t wave_rows = (256 / p.D) * (many ? 4 : 1);
    const unsigned blocks = (unsigned)((rows + 4 * wave_rows - 1) / (4 * wave_rows));
    auto go = [&](auto one, auto four) {
        if (many) four<<<dim3(blocks), dim3(256), 0, s>>>(p);
        else one<<<dim3(blocks), dim3(256), 0, s>>>(p);
    };
    if (p.D == 128) {
        if (p.dt == AKV_DT_F16) go(K<128, AKV_DT_F16, 1>::fn, K<128, AKV_DT_F16, 4>::fn);
        else if (p.dt == AKV_DT_BF16) go(K<128, AKV_DT_BF16, 1>::fn, K<128, AKV_DT_BF16, 4>::fn);
        else go(K<128, AKV_DT_F32, 1>::fn, K<128, AKV_DT_F32, 4>::fn);
    } else {
        if (p.dt == AKV_DT_F16) go(K<64, AKV_DT_F16, 1>::fn, K<64, AKV_DT_F16, 4>::fn);
        else if (p.dt == AKV_DT_BF16) go(K<64, AKV_DT_BF16, 1>::fn, K<64, AKV_DT_BF16, 4>::fn);
        else go(K<64, AKV_DT_F32, 1>::fn, K<64, AKV_DT_F32, 4>::fn);
    }
    return hipGetLastError();
}
template <int D, int DT, int IT>
struct AppendK {
    static constexpr auto fn = paged_append_kernel<D, DT, IT>;
};
template <int D, int DT, int IT>
struct ReadK {
    static constexpr auto fn = paged_read_kernel<D, DT, IT>;
};

}  // namespace

hipError_t paged_append_launch(const PagedRowsParams &p, hipStream_t s) { return rows_launch<AppendK>(p, s); }
hipError_t paged_read_launch(const PagedRowsParams &p, hipStream_t s) { return rows_launch<ReadK>(p, s); }

hipError_t paged_copy_launch(const PagedCopyParams &p, hipStream_t s) {
    const int64_t pieces = (p.page_bytes >> 4) * p.n * p.layers;
    if (pieces == 0) return hipSuccess;
    const int64_t blocks = (pieces + 1023) / 1024;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    paged_copy_kernel<<<dim3((unsigned)blocks), dim3(256), 0, s>>>(p);
    return hipGetLastError();
}

hipError_t paged_compact_launch(const PagedCompactParams &p, hipStream_t s) {
    const int64_t tiles = (p.max_keep + 15) / 16;
    if (tiles == 0 || p.n_seqs == 0 || p.layers == 0) return hipSuccess;
    const int64_t bx = (tiles * p.pool.heads + 3) / 4;
    if (bx > 0x7fffffff) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)bx, (unsigned)p.n_seqs, (unsigned)p.layers), block(256);
    if (p.D == 128) {
        if (p.ng == 4) paged_compact_kernel<128, 4><<<grid, block, 0, s>>>(p);
        else if (p.ng == 2) paged_compact_kernel<128, 2><<<grid, block, 0, s>>>(p);
        else paged_compact_kernel<128, 1><<<grid, block, 0, s>>>(p);
    } else {
        if (p.ng == 2) paged_compact_kernel<64, 2><<<grid, block, 0, s>>>(p);
        else paged_compact_kernel<64, 1><<<grid, block, 0, s>>>(p);
    }
    return hipGetLastError();
}

}  // namespace akv
