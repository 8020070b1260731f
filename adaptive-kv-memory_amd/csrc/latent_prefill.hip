// Attention over the paged latent cache in its expanded form, for chunks of a prompt.
//
// The mathematics.  Head h's keys are k = [W_k,h c | r] and its values v = W_v,h c of a cached row
// (latent c, rotated key r).  A row and token cost 2 (Dn + Dr + Dv) operations a head once they are
// made, against 2 (2 Dc + Dr) where the latent itself is key and value; making them costs 2 Dc (Dn + Dv) a
// token and head, which some 170 query tokens outweigh.  Two kernels: the expansion is a matrix product
// whose left side stays in LDS for all heads, the attention streams its results.  Keys and values are
// float16 over a power of two for each channel (which goes to the queries and the outputs, so that small weights
// keep their bits), query rows float16 scaled by a power of two, p one float16; for float16 outputs keys, values and p are
// two float16 each.  Scores, sums and the softmax state are float32.
#include <algorithm>
#include <type_traits>

#include "akv_common.h"
#include "latent.h"
#include "latent_device.h"

namespace akv {
namespace {

constexpr int kD = kLatentHead;       // channels of a head's own keys, and of its values
constexpr int kThreads = 256;         // of the scan, the expansion and the merge
constexpr int kAttendThreads = 512;
constexpr int kExpandTok = 128;       // tokens of a workgroup of the expansion
constexpr int kSetupTok = 128;        // tokens that an item's start counts
constexpr int kGroups = 256;
// Tokens of a step of the attention: with two float16 each they are twice the bytes in LDS.
__host__ __device__ constexpr int step_tokens(bool two) { return two ? 32 : 64; }

struct TileScan {
    int64_t pre[kThreads + 1], wave_sum[kThreads / 64];
};
// What lies before each thread's sequences, of(s) for sequence s.
template <typename Of>
__device__ __forceinline__ void scan_sequences(int n_seqs, TileScan &sc, Of of) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, per = (n_seqs + kThreads - 1) / kThreads;
    int64_t mine = 0, inc = 0;
    if (t < kThreads) {
        for (int i = 0; i < per; ++i)
            if (t * per + i < n_seqs) mine += of(t * per + i);
        inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 63) sc.wave_sum[wave] = inc;
    }
    __syncthreads();
    if (t < kThreads) {
        int64_t before = 0;
        for (int w = 0; w < wave; ++w) before += sc.wave_sum[w];
        sc.pre[t] = before + inc - mine;
        if (t == kThreads - 1) sc.pre[kThreads] = before + inc;
    }
    __syncthreads();
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}
// The first sequence of the thread whose sequences hold x, and how much of x lies in them; returns how many
// sequences a thread has.
__device__ __forceinline__ int seq_of_first(const TileScan &sc, int64_t x, int n_seqs, int &s, int64_t &off) {
    const int per = (n_seqs + kThreads - 1) / kThreads;
    int k = 0;
    for (int i = 0; i < kThreads / 64; ++i) k += __builtin_popcountll(__builtin_amdgcn_ballot_w64(sc.pre[64 * i + (threadIdx.x & 63)] <= x));
    s = (k - 1) * per;
    off = x - uniform64(sc.pre[k - 1]);
    return per;
}

}  // namespace

// Expansion.  A workgroup holds 128 cached rows' latents in LDS and makes the 128 key and 128 value channels
// of one head after another; a wave makes 64 of them for all 128 tokens.  Its weights come straight from
// memory in operand order, a stream of 16-byte loads that runs half a head ahead and on over the heads.
// All workgroups are at the same heads at about the same time, so that a chiplet's L2 reads them once.
// Bound by the matrix cores at the clock that the card's power leaves them, and by the weights' way from L2: 64 heads and
// 2 sequences of up to 17408 tokens (0.5 TFLOP, 1 GB written) take 510 to 580 us; 16 heads and 1396 tokens, a head a
// workgroup, 20 us, most of it the first 128 KB of latents and 256 KB of weights of each.
template <int DC>
__global__ __launch_bounds__(kThreads, 1) void latent_expand_kernel(const LatentPrefillParams p) {
    constexpr int LROW = 2 * DC, KS = DC / 32, TILES = kExpandTok / 16, RING = KS / 2;
    constexpr int PIECES = 16 * LROW / 1024;  // KiB of a tile's latents
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ TileScan sc;
    // float16 results that overflow become the largest
    __builtin_amdgcn_s_setreg(1 | 23 << 6, 1);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    auto tiles_of = [&](int s) {
        const SeqRows r = seq_rows(p.seqs, s, p.pool.log_page);
        return r.n == 0 ? 0 : (r.kv + kExpandTok - 1) / kExpandTok;
    };
    scan_sequences(p.seqs.n_seqs, sc, tiles_of);
    const int tiles = __builtin_amdgcn_readfirstlane((int)sc.pre[kThreads]);
    if (tiles == 0) return;
    // The heads in blocks, as many as make the longest workgroup shortest.  A tile of latents costs about
    // as much as two heads.
    int blocks = 1;
    float least = INFINITY;
    for (int n = lane + 1; n <= p.heads; n += 64) {
        const float cost = (float)(((int64_t)tiles * n + (int)gridDim.x - 1) / (int)gridDim.x) * (2 + (p.heads + n - 1) / n);
        if (cost < least) least = cost, blocks = n;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float cost = __shfl_xor(least, d);
        const int n = __shfl_xor(blocks, d);
        if (cost < least || (cost == least && n < blocks)) least = cost, blocks = n;
    }
    blocks = __builtin_amdgcn_readfirstlane(blocks);
    const int each = (p.heads + blocks - 1) / blocks;
    for (int64_t item = blockIdx.x; item < (int64_t)tiles * blocks; item += gridDim.x) {
        const int block = (int)(item / tiles), tile = (int)(item - (int64_t)block * tiles);
        const int h0 = block * each, h1 = min(p.heads, h0 + each);
        if (h0 >= h1) break;
        int s, tok0;
        {
            int64_t off;
            const int per = seq_of_first(sc, tile, p.seqs.n_seqs, s, off);
            for (int i = 0; i < per; ++i) {
                const int n = tiles_of(s);
                if (off < n) break;
                off -= n, ++s;
            }
            s = __builtin_amdgcn_readfirstlane(s), tok0 = __builtin_amdgcn_readfirstlane((int)off * kExpandTok);
        }
        const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_page));
        const u4 *w = (const u4 *)p.w + ((int64_t)(p.head0 + h0) * KS * 16 + wave * 4) * 64 + lane;
        const int last = (h1 - h0) * KS - 1;  // step of the stream: the heads lie one after the other
        u4 W[RING][4];
#pragma unroll
        for (int u = 0; u < RING - 1; ++u)
#pragma unroll
            for (int b = 0; b < 4; ++b) W[u][b] = w[(u * 16 + b) * 64];
        Pages pages{p.seqs.table + s * p.seqs.table_stride, p.seqs.width, 0, 0};
        pages.fill(tok0 >> p.pool.log_page);
        __syncthreads();  // the tile before is read
        // chunk c of row t lies at c ^ t % 16, so that the sixteen chunks that a read takes at once differ
#pragma unroll 1
        for (int i = 0; i < TILES / 4; ++i) {
            const int t = wave + 4 * i;
            const Tile at = tile_at(p.pool, pages, tok0 + 16 * t, r.kv);
            const u4 rsrc = wave_rsrc(at.at, at.rows * p.pool.row_bytes);
#pragma unroll 1
            for (int n = 0; n < PIECES; ++n) {
                const int c = 64 * n + lane, row = c / (LROW / 16), in = c % (LROW / 16);
                dma_kib(rsrc, __builtin_amdgcn_readfirstlane(lds_addr(smem) + t * 16 * LROW + n * 1024),
                        row * p.pool.row_bytes + ((in ^ (row & 15)) << 4));
            }
        }
        wait_vm<0>();
        __syncthreads();
        const uint32_t at = lds_addr(smem) + col * LROW;
        for (int h = h0; h < h1; ++h) {
            f4 acc[TILES][4];
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) acc[t][b] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int k = 0; k < KS; k += RING)
#pragma unroll
                for (int u = 0; u < RING; ++u) {
                    const int64_t next = min((h - h0) * KS + k + u + RING - 1, last);
#pragma unroll
                    for (int b = 0; b < 4; ++b) W[(u + RING - 1) % RING][b] = w[(next * 16 + b) * 64];
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        const h8 c = __builtin_bit_cast(h8, *lds_ptr<u4>(at + t * 16 * LROW + (((4 * (k + u) + grp) ^ col) << 4)));
#pragma unroll
                        for (int b = 0; b < 4; ++b) acc[t][b] = mfma_k32(__builtin_bit_cast(h8, W[u][b]), c, acc[t][b]);
                    }
                }
            // a lane has 16 consecutive channels of token col of every tile
            unsigned char *to = (wave < 2 ? p.keys : p.values) +
                                (((int64_t)h * p.cap + s * p.seq_cap + tok0 + col) * kD + 64 * (wave & 1) + 16 * grp) * 2;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                if (tok0 + 16 * t + col >= p.seq_cap) continue;
                u4 o[2];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f4 v = acc[t][b];
                    o[b >> 1][2 * (b & 1)] = as_u32((h2){(_Float16)v[0], (_Float16)v[1]});
                    o[b >> 1][2 * (b & 1) + 1] = as_u32((h2){(_Float16)v[2], (_Float16)v[3]});
                }
                ((u4 *)(to + (int64_t)t * 16 * kD * 2))[0] = o[0];
                ((u4 *)(to + (int64_t)t * 16 * kD * 2))[1] = o[1];
                if (!p.rest) continue;
                u4 rest[2];
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const h2 high = as_h2(o[b >> 1][2 * (b & 1) + e]);
                        rest[b >> 1][2 * (b & 1) + e] = as_u32((h2){(_Float16)(acc[t][b][2 * e] - (float)high[0]), (_Float16)(acc[t][b][2 * e + 1] - (float)high[1])});
                    }
                ((u4 *)(to + p.rest + (int64_t)t * 16 * kD * 2))[0] = rest[0];
                ((u4 *)(to + p.rest + (int64_t)t * 16 * kD * 2))[1] = rest[1];
            }
        }
    }
}

namespace {

// The work of a sequence: tile t of a head's rows costs a + b t tokens.
struct TileWork {
    SeqRows r;
    int rows, tiles;
    int64_t a, b;
    __device__ __forceinline__ int64_t cost(int t) const { return a + b * t; }
    __device__ __forceinline__ int64_t before(int64_t t) const { return a * t + b * (t * (t - 1) / 2); }
};
template <int R>
__device__ __forceinline__ TileWork tile_work(const LatentPrefillParams &p, const SeqRows &r) {
    TileWork w;
    w.r = r;
    w.rows = min(r.n, p.seqs.max_q);
    w.tiles = (w.rows + R - 1) / R;
    const int64_t old = min(max(r.at, 0), r.kv);
    w.a = (p.causal ? old + R : r.kv) + kSetupTok;
    w.b = p.causal ? R : 0;
    return w;
}
// Steps of tile t, and how many of them lie before cost c of it.
template <int R, int ST>
__device__ __forceinline__ int steps_of(const LatentPrefillParams &p, const TileWork &w, int t) {
    return (w.r.sees(p.causal, min((t + 1) * R, w.rows) - 1) + ST - 1) / ST;
}
template <int ST>
__device__ __forceinline__ int steps_before(int64_t c, int64_t cost, int steps) {
    if (c >= cost) return steps;
    const int64_t x = (c - kSetupTok + ST - 1) / ST;
    return (int)(x < 0 ? 0 : x > steps ? steps : x);
}
template <int R>
__device__ __forceinline__ void scan_tiles(const LatentPrefillParams &p, TileScan &sc) {
    scan_sequences(p.seqs.n_seqs, sc, [&](int s) {
        const TileWork w = tile_work<R>(p, seq_rows(p.seqs, s, p.pool.log_page));
        return w.before(w.tiles) * p.heads;
    });
}
__device__ __forceinline__ int64_t share_of(int64_t total, int groups) { return max((total + groups - 1) / groups, (int64_t)(2 * kSetupTok)); }

// Value e of eight of a query row as float.
template <bool BF16>
__device__ __forceinline__ float query_value(u4 w, int e) {
    const uint32_t v = w[e >> 1];
    return BF16 ? __builtin_bit_cast(float, e & 1 ? v & 0xffff0000u : v << 16) : (float)as_h2(v)[e & 1];
}
// value(i, e) times a power of two that takes the row's largest to [2^13, 2^14) as float16; returns what
// turns its scores to the log2 domain.
template <int N, typename Value>
__device__ __forceinline__ float scaled_row(h8 (&op)[N], Value value, float scale_log2) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf(value(i, e)));
    top = qmax(top);
    const int ex = top > 0.0f ? max(__builtin_amdgcn_frexp_expf(top), -60) : 14;
    const float x = __builtin_ldexpf(1.0f, 14 - ex);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) op[i][e] = (_Float16)__builtin_fmaf(value(i, e), x, -0.0f);
    return row_factor(scale_log2, ex);
}

// 64 pages of a sequence's table in a wave's lanes, and which of them are pages of the pool.
struct StepPages {
    int first, ids;
    uint64_t valid;
    __device__ __forceinline__ void fill(const LatentPrefillParams &p, int s, int page) {
        first = __builtin_amdgcn_readfirstlane(page);
        const int at = page + lane_again();
        ids = at < p.seqs.width ? p.seqs.table[s * p.seqs.table_stride + at] : -1;
        valid = __builtin_amdgcn_ballot_w64((uint32_t)ids < p.pool.n_pages);  // waited for here
    }
};

}  // namespace

// Attention.  A workgroup of eight waves takes 128 RB query tokens of one head, each wave 16 RB of them, and
// walks the keys and values in steps of 64 tokens.  Buffer loads fill two rings of three steps in LDS: the keys'
// own channels with the shared rotated ones, straight from the cache's rows, and the values.
// S^T = K Q^T leaves a lane with its row's scores of the tokens that the second product's operand wants, so p
// stays in registers.  A SIMD has two waves, which take turns: while one multiplies (the values of its last step,
// then the keys of the next) the other turns scores into p.  The second four waves do so by standing at one barrier
// more before their first step.
// 2 chunks of up to 1024 tokens after up to 16384, 64 heads: 0.95 to 1.07 ms, 0.93 PFLOP/s with what the causal tiles'
// corners waste, at 1.7 GHz: the card's power holds the clock, and fewer cycles (17.5 to 14.3 million of all chiplets)
// gave little time.  5 prompts of up to 777 tokens, 16 heads: 28 us, most of it an item's start and end.
//
// TWO, for float16 outputs: keys, values and p enter their products as two float16 each (of p v without the product of
// both rests), or their roundings would be larger than the output's own, 2.1e-4 of the norm.  One float16 for the keys
// moves a score by 2^-12 of its size and more: with scores of standard deviation 1 and 4 outputs are 2.6e-4 and 4.4e-4 off,
// single rows 1.9e-3; with two all are 2.1e-4, rows 2.7e-4.  For bfloat16 outputs, which round to 1.7e-3, one is
// enough (1.68e-3 at deviation 1, 1.73e-3 at 4).  Steps have 32 tokens then, so that three slots fit LDS.  2 chunks of
// up to 1024 tokens, 64 heads: 2.67 ms, 2.18 with one float16 for the keys, 1.51 with one for all.
template <int DC, int RB, bool TWO>
__global__ __launch_bounds__(kAttendThreads, 2) void latent_prefill_kernel(const LatentPrefillParams p) {
    constexpr int NW = kAttendThreads / 64, R = 16 * RB * NW, SLOTS = 3, ST = step_tokens(TWO), TT = ST / 16;
    // a slot of keys: the heads' own channels, the rotated ones, the rest; of values: the values, the rest
    constexpr int OWN = ST * kD * 2, ROPE = ST * kLatentRope * 2, KB = OWN + ROPE + (TWO ? OWN : 0), VB = OWN + (TWO ? OWN : 0);
    constexpr int PIECES = OWN / 1024 / NW, V_LOADS = (TWO ? 2 : 1) * PIECES, K_LOADS = V_LOADS + 1;
    constexpr int CB = kD / 16, NI = (kD + kLatentRope) / 32, ROWB = 2 * (DC + kLatentRope);
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ TileScan sc;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4, second = wave / (NW / 2);
    const uint32_t ring = lds_addr(smem);
    // Rows' 16-byte chunks lie turned so that the sixteen slots of 256 bytes that a read takes at once differ:
    // chunk c of a row of keys at c ^ row % 16, of rotated keys at c ^ row / 2 % 8, of values at
    // c ^ 2 (row % 8).  A load of 1 KiB brings four rows of keys or values, eight of rotated keys.
    const uint32_t k_off = grp * kD * 2 + ((col ^ grp) << 4), v_off = grp * kD * 2 + ((col ^ 2 * grp) << 4);
    const uint32_t r_off = (lane >> 3) * ROWB + 2 * DC + (((lane & 7) ^ grp) << 4);
    const uint32_t k_at = col * kD * 2 + ((grp ^ col) << 4);
    const uint32_t r_at = OWN + col * kLatentRope * 2 + ((grp ^ col >> 1) << 4);
    const int vrow = 4 * grp + (col >> 2);
    const uint32_t v_at = vrow * kD * 2 + (((col & 3) >> 1 ^ 2 * (vrow & 7)) << 4) + 8 * (col & 1);

    scan_tiles<R>(p, sc);
    const int64_t total = uniform64(sc.pre[kThreads]);
    const int64_t share = share_of(total, p.groups);
    if (blockIdx.x == 0 && threadIdx.x < kThreads) {
        p.sums[threadIdx.x] = sc.pre[threadIdx.x];
        if (threadIdx.x == 0) p.sums[kThreads] = total;
    }
    int64_t x = min((int64_t)blockIdx.x * share, total);
    const int64_t x_end = min(x + share, total);
    if (x >= x_end) return;
    int s, h = 0, tile = 0;
    int64_t c0;  // where in the tile's cost the run stands
    TileWork w;
    {
        int64_t off;
        seq_of_first(sc, x, p.seqs.n_seqs, s, off);
        for (;;) {
            w = tile_work<R>(p, wave_uniform(seq_rows(p.seqs, s, p.pool.log_page)));
            const int64_t n = w.before(w.tiles) * p.heads;
            if (off < n) break;
            off -= n;
            ++s;
        }
        const int64_t one = w.before(w.tiles);
        h = (int)(off / one);
        off -= h * one;
        while (off >= w.cost(tile)) off -= w.cost(tile++);
        c0 = off;
    }
    while (x < x_end) {
        const int64_t cost = w.cost(tile), c1 = min(cost, c0 + (x_end - x));
        const int steps_all = steps_of<R, ST>(p, w, tile);
        const int j0 = steps_before<ST>(c0, cost, steps_all), j1 = steps_before<ST>(c1, cost, steps_all);
        const bool starts = c0 <= kSetupTok, ends = c1 == cost;
        x += c1 - c0;
        if (j1 > j0 || (starts && ends)) {
            const int row0 = tile * R, head = p.head0 + h;
            const int mine = row0 + 16 * RB * wave;
            int see[RB];
            float kx[RB];
            h8 Q[RB][NI];
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                const int row = min(mine + 16 * r + col, w.rows - 1);
                see[r] = w.r.sees(p.causal, row);
                const unsigned char *q = p.q + (w.r.begin + row) * p.q_t + head * p.q_h + 16 * grp;
                const f4 *ws = (const f4 *)(p.w_scale + (int64_t)head * 2 * kD + 8 * grp);  // of the keys' channels
                u4 raw[NI];
                f4 by[kD / 32][2];
#pragma unroll
                for (int i = 0; i < NI; ++i) raw[i] = *(const u4 *)(q + 64 * i);
#pragma unroll
                for (int i = 0; i < kD / 32; ++i) by[i][0] = ws[8 * i], by[i][1] = ws[8 * i + 1];
                auto make = [&](auto is_bf16) {
                    kx[r] = scaled_row(Q[r], [&](int i, int e) {
                        const float v = query_value<decltype(is_bf16)::value>(raw[i], e);
                        return i < kD / 32 ? v * by[i][e >> 2][e & 3] : v;
                    }, p.scale_log2);
                };
                if (p.q_bf16) make(std::true_type{});
                else make(std::false_type{});
            }
            const int see_all = w.r.sees(p.causal, min(mine, w.rows - 1));  // what all of the wave's rows see
            const int kv = w.r.kv;
            const int lp = p.pool.log_page;
            StepPages pages;
            const int64_t base = ((int64_t)h * p.cap + s * p.seq_cap) * kD * 2;
            uint32_t there = 0;  // bits TT slot ..
            auto load_own = [&](const unsigned char *from, int k, int end, uint32_t to, uint32_t off, int turns) {
                const u4 rsrc = wave_rsrc(from + base + (int64_t)k * kD * 2, max(0, min(end - k, ST)) * kD * 2);
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int n = PIECES * wave + i;
                    dma_kib(rsrc, to + n * 1024, (off ^ (turns == 4 ? (n & 3) << 6 : (n & 1) << 7)) + n * 1024);
                }
            };
            auto load_keys = [&](int j, int slot) {
                const int k = j * ST, end = j < j1 ? kv : 0;
                const uint32_t to = __builtin_amdgcn_readfirstlane(ring + slot * KB);
                load_own(p.keys, k, end, to, k_off, 4);
                if (TWO) load_own(p.keys + p.rest, k, end, to + OWN + ROPE, k_off, 4);
                const int page = k >> lp;
                if (page + ((ST - 16) >> lp) - pages.first >= 64) pages.fill(p, s, page);
                const uint64_t valid = pages.valid >> (page - pages.first);
                uint32_t bits = 0;
#pragma unroll
                for (int i = 0; i < TT; ++i) bits |= (uint32_t)(valid >> (16 * i >> lp) & 1) << i;
                // the rotated keys of eight tokens (of four waves the same as of the others where a step has 32)
                const int eight = wave & (ST / 8 - 1), tok = k + 8 * eight, in = (tok >> lp) - pages.first;
                const int rows = pages.valid >> in & 1 ? max(0, min(end - tok, 8)) : 0;
                const unsigned char *rows_at = p.pool.base + (int64_t)__builtin_amdgcn_readlane(pages.ids, in) * p.pool.page_bytes +
                                               (int64_t)(tok & ((1 << lp) - 1)) * ROWB;
                dma_kib(wave_rsrc(rows_at, rows * ROWB), to + OWN + eight * 1024, r_off ^ (eight & 1) << 6);
                there = (there & ~(((1u << TT) - 1) << TT * slot)) | bits << TT * slot;
            };
            auto load_values = [&](int j, int slot) {
                const int k = j * ST, end = j < j1 ? kv : 0;
                const uint32_t to = __builtin_amdgcn_readfirstlane(ring + SLOTS * KB + slot * VB);
                load_own(p.values, k, end, to, v_off, 2);
                if (TWO) load_own(p.values + p.rest, k, end, to + OWN, v_off, 2);
            };
            auto after = [](int slot) { return slot + 1 == SLOTS ? 0 : slot + 1; };
            float mx[RB], l[RB];
            f4 acc[CB][RB];
            u4 P[ST / 32][RB], P_rest[ST / 32][RB];  // of 32 tokens each
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                mx[r] = kMinMax, l[r] = 0.0f;
#pragma unroll
                for (int b = 0; b < CB; ++b) acc[b][r] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < ST / 32; ++i) P[i][r] = P_rest[i][r] = (u4){0, 0, 0, 0};
            }
            constexpr int V_AHEAD = TWO ? 3 : 6, K_AHEAD = 8;  // reads that are under way
            auto value = [&](uint32_t va, int n) {
                const uint32_t a = (va ^ (n % CB) << 5) + n / CB * 32 * kD * 2;
                const u2 lo = read_transposed(a), hi = read_transposed(a + 16 * kD * 2);
                return __builtin_bit_cast(h8, (u4){lo[0], lo[1], hi[0], hi[1]});
            };
            // p times the values; then(m) in the steps that read no more of them
            auto add_values = [&](uint32_t va, auto then) {
                constexpr int READS = ST / 32 * CB;
                h8 V[V_AHEAD], V_rest[V_AHEAD];
                auto read = [&](int n) {
                    V[n % V_AHEAD] = value(va, n);
                    if (TWO) V_rest[n % V_AHEAD] = value(va + OWN, n);
                };
#pragma unroll
                for (int n = 0; n < V_AHEAD; ++n) read(n);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < READS; ++n) {
                    if (TWO)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int r = 0; r < RB; ++r)
                                acc[n % CB][r] = mfma_k32(i ? V_rest[n % V_AHEAD] : V[n % V_AHEAD],
                                                          __builtin_bit_cast(h8, i ? P[n / CB][r] : P_rest[n / CB][r]), acc[n % CB][r]);
#pragma unroll
                    for (int r = 0; r < RB; ++r) acc[n % CB][r] = mfma_k32(V[n % V_AHEAD], __builtin_bit_cast(h8, P[n / CB][r]), acc[n % CB][r]);
                    if (n + V_AHEAD < READS) read(n + V_AHEAD);
                    else then(n + V_AHEAD - READS);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            const uint32_t values = ring + SLOTS * KB + v_at;
            auto meet = [&]() {
                wait_lgkm0();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            };
            pages.fill(p, s, (j0 * ST) >> lp);
            load_keys(j0, 0);
            load_keys(j0 + 1, 1);
            load_values(j0, 0);
            wait_vm<K_LOADS + V_LOADS>();
            int slot = 0;  // of step j, for keys and for values
            if (second) {
                meet();
                load_keys(j0 + 2, 2);
            }
            for (int j = j0; j < j1; ++j) {
                // done then: this step's keys, the last one's values, and in the second waves, whose next barrier is the
                // first ones', also the next keys and this step's values
                wait_vm<K_LOADS>();
                meet();
                const int next = after(slot), last = after(next);
                load_values(j + 1, next);
                const uint32_t ka = ring + slot * KB + k_at, ra = ring + slot * KB + r_at;
                auto key = [&](int n) {
                    const int c = n / TT, i = n % TT;
                    return __builtin_bit_cast(h8, *lds_ptr<u4>(c < kD / 32 ? (ka ^ c << 6) + i * 16 * kD * 2
                                                               : c < NI    ? (ra ^ (c - kD / 32) << 6) + i * 16 * kLatentRope * 2
                                                                           : (ka ^ (c - NI) << 6) + OWN + ROPE + i * 16 * kD * 2));
                };
                h8 K[K_AHEAD];
                auto read_keys = [&](int from, int to) {
#pragma unroll
                    for (int n = from; n < to; ++n) K[n] = key(n);
                };
                if (j > j0) add_values(values + last * VB, [&](int m) { read_keys(m * K_AHEAD / V_AHEAD, (m + 1) * K_AHEAD / V_AHEAD); });
                else read_keys(0, K_AHEAD);
                __builtin_amdgcn_sched_barrier(0);
                f4 S[TT][RB] = {};
                constexpr int READS = TT * (NI + (TWO ? kD / 32 : 0));  // the rest meets the same queries
#pragma unroll
                for (int n = 0; n < READS; ++n) {
#pragma unroll
                    for (int r = 0; r < RB; ++r) S[n % TT][r] = mfma_k32(K[n % K_AHEAD], Q[r][n / TT % NI], S[n % TT][r]);
                    if (n + K_AHEAD < READS) K[n % K_AHEAD] = key(n + K_AHEAD);
                    __builtin_amdgcn_sched_barrier(0);
                }
                const int first = j * ST;
                const uint32_t have = there >> TT * slot & ((1u << TT) - 1);
                meet();
                if (second) {
                    load_keys(j + 3, slot);
                } else {
                    load_keys(j + 2, last);
                }
                if (!(first + ST <= see_all && have == (1u << TT) - 1)) {
                    int at0 = first + 4 * grp;
                    asm volatile("" : "+v"(at0));  // (nothing of this is computed where nothing is masked)
#pragma unroll
                    for (int i = 0; i < TT; ++i)
#pragma unroll
                        for (int r = 0; r < RB; ++r)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (at0 + 16 * i + e >= see[r] || !(have >> i & 1)) S[i][r][e] = -INFINITY;
                }
                float top[RB];
                bool over = false;
#pragma unroll
                for (int r = 0; r < RB; ++r) {
                    top[r] = S[0][r][0];
#pragma unroll
                    for (int i = 1; i < 4 * TT; ++i) top[r] = __builtin_fmaxf(top[r], S[i >> 2][r][i & 3]);
                    over |= __builtin_fmaf(top[r], kx[r], kBias - mx[r]) > kBias + kLagBy;
                }
                if (__builtin_amdgcn_ballot_w64(over)) {
#pragma unroll
                    for (int r = 0; r < RB; ++r) {
                        const float most = qmax(top[r]);
                        const float mn = __builtin_fmaf(most, kx[r], kBias - mx[r]) > kBias ? running_max(most, kx[r], kBias) : mx[r];
                        const float alpha = __builtin_amdgcn_exp2f(mx[r] - mn);
                        l[r] *= alpha;
                        mx[r] = mn;
#pragma unroll
                        for (int b = 0; b < CB; ++b) acc[b][r] *= alpha;
                    }
                }
#pragma unroll
                for (int r = 0; r < RB; ++r)
#pragma unroll
                    for (int i = 0; i < TT; ++i) {
                        float e[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) e[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i][r][q], kx[r], kBias - mx[r]));
                        l[r] += (e[0] + e[1]) + (e[2] + e[3]);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const h2 high = {(_Float16)e[2 * q], (_Float16)e[2 * q + 1]};
                            P[i >> 1][r][2 * (i & 1) + q] = as_u32(high);
                            if (TWO) P_rest[i >> 1][r][2 * (i & 1) + q] = as_u32((h2){(_Float16)(e[2 * q] - (float)high[0]), (_Float16)(e[2 * q + 1] - (float)high[1])});
                        }
                    }
                slot = next;
            }
            wait_vm<0>();
            meet();
            if (j1 > j0) add_values(values + (slot == 0 ? SLOTS - 1 : slot - 1) * VB, [](int) {});
            if (!second) meet();
            float *e = p.part + ((int64_t)blockIdx.x * 2 + starts) * (R * (kD + 2));
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                l[r] = qsum(l[r]);
                const int row = mine + 16 * r + col;
                if (starts && ends) {
                    const float inv = row_inverse(l[r]);
                    if (row < w.rows) {
                        const f4 *vs = (const f4 *)(p.w_scale + ((int64_t)head * 2 + 1) * kD) + grp;
                        unsigned char *out = (unsigned char *)p.out + ((int64_t)(w.r.begin + row) * p.H + head) * (2 * kD) + 8 * grp;
#pragma unroll
                        for (int b = 0; b < CB; ++b) {
                            const f4 v = acc[b][r] * inv * vs[4 * b];
                            *(u2 *)(out + 32 * b) = (u2){out_pair(p.q_bf16, v[0], v[1]), out_pair(p.q_bf16, v[2], v[3])};
                        }
                    }
                } else {
                    const int at = RB * wave + r;
#pragma unroll
                    for (int b = 0; b < CB; ++b) *(f4 *)(e + (at * CB + b) * 256 + lane * 4) = acc[b][r];
                    if (grp == 0) e[R * kD + 16 * at + col] = mx[r], e[R * kD + R + 16 * at + col] = l[r];
                }
            }
            __syncthreads();
        }
        // the next item
        c0 = 0;
        if (x < x_end && ++tile == w.tiles) {
            tile = 0;
            if (++h == p.heads) {
                h = 0;
                do {
                    w = tile_work<R>(p, wave_uniform(seq_rows(p.seqs, ++s, p.pool.log_page)));
                } while (w.tiles == 0);
            }
        }
    }
}

// Joins the partial states of items that several workgroups share: a wave takes 16 rows of one.  Bound by the
// states' bytes: 10 us for 5 prompts of up to 777 tokens, 16 heads.
template <int R, int ST>
__global__ __launch_bounds__(kThreads) void latent_prefill_merge_kernel(const LatentPrefillParams p) {
    constexpr int CB = kD / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const int s = blockIdx.z, h = blockIdx.y;
    const int block = blockIdx.x * (kThreads / 64) + wave, tile = block / (R / 16), in = block % (R / 16);
    const int per = (p.seqs.n_seqs + kThreads - 1) / kThreads;
    const TileWork w = tile_work<R>(p, wave_uniform(seq_rows(p.seqs, s, p.pool.log_page)));
    const int row = tile * R + 16 * in + col;
    if (tile >= w.tiles || tile * R + 16 * in >= w.rows) return;
    int64_t start = p.sums[s / per] + h * w.before(w.tiles) + w.before(tile);
    for (int i = s / per * per; i < s; ++i) {
        const TileWork b = tile_work<R>(p, wave_uniform(seq_rows(p.seqs, i, p.pool.log_page)));
        start += b.before(b.tiles) * p.heads;
    }
    const int64_t share = share_of(p.sums[kThreads], p.groups), cost = w.cost(tile);
    // start / share and (start + cost - 1) / share: below 2^8, so that the product errs by less than one
    const float one = 1.0f / (float)share;
    auto run_of = [&](int64_t at) {
        int g = (int)((float)at * one);
        g -= g * share > at;
        return g + ((g + 1) * share <= at);
    };
    const int g0 = run_of(start), g1 = run_of(start + cost - 1);
    if (g0 == g1) return;
    const int steps = steps_of<R, ST>(p, w, tile);
    // the runs that hold steps of it, and whether a run's entry is the one whose item starts there
    auto part = [&](int g, int64_t &c0) {
        c0 = max((int64_t)0, g * share - start);
        const int64_t c1 = min(cost, (g + 1) * share - start);
        return steps_before<ST>(c1, cost, steps) > steps_before<ST>(c0, cost, steps);
    };
    auto entry = [&](int g, int64_t c0) { return p.part + ((int64_t)g * 2 + (c0 <= kSetupTok)) * (R * (kD + 2)); };
    float m = kMinMax, l = 0.0f;
    f4 acc[CB] = {};
    int n = 0;
    bool whole = false;
    for (int g = g0; g <= g1; ++g) {
        int64_t c0;
        if (!part(g, c0)) continue;
        ++n;
        whole = c0 <= kSetupTok && g == g1;
        if (whole && n == 1) return;  // one run held all of it and wrote the rows
        const float *e = entry(g, c0);
        const float m_e = e[R * kD + 16 * in + col], l_e = e[R * kD + R + 16 * in + col];
        f4 a_e[CB];
#pragma unroll
        for (int b = 0; b < CB; ++b) a_e[b] = *(const f4 *)(e + (in * CB + b) * 256 + lane * 4);
        const float most = __builtin_fmaxf(m, m_e), old = __builtin_amdgcn_exp2f(m - most), add = __builtin_amdgcn_exp2f(m_e - most);
        m = most;
        l = l * old + l_e * add;
#pragma unroll
        for (int b = 0; b < CB; ++b) acc[b] = acc[b] * old + a_e[b] * add;
    }
    if (row >= w.rows) return;
    const float inv = row_inverse(l);
    const f4 *vs = (const f4 *)(p.w_scale + ((int64_t)(p.head0 + h) * 2 + 1) * kD) + grp;
    unsigned char *out = (unsigned char *)p.out + ((int64_t)(w.r.begin + row) * p.H + p.head0 + h) * (2 * kD) + 8 * grp;
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        const f4 v = acc[b] * inv * vs[4 * b];
        *(u2 *)(out + 32 * b) = (u2){out_pair(p.q_bf16, v[0], v[1]), out_pair(p.q_bf16, v[2], v[3])};
    }
}

namespace {
constexpr int64_t kSumsBytes = 4096;
static_assert((kThreads + 1) * 8 <= kSumsBytes, "the sums fit");
constexpr int64_t kMostBytes = (int64_t)4 << 30;  // keys and values of a pass, where one head's are not more
int64_t part_bytes(const LatentPrefillParams &p) { return (int64_t)p.groups * 2 * p.rows * (kD + 2) * 4; }
}  // namespace

int64_t latent_prefill_plan(LatentPrefillParams *p) {
    p->seq_cap = (int64_t)p->seqs.width << p->pool.log_page;
    p->cap = p->seq_cap * p->seqs.n_seqs;
    const int64_t head = std::max<int64_t>(1, p->cap * (p->q_bf16 ? 2 : 4) * kD * 2);
    p->heads = (int)std::max<int64_t>(1, std::min<int64_t>(p->H, kMostBytes / head));
    // 256 query tokens a workgroup where there are tiles of them for all, else 128 (attention and merge of 5
    // prompts of up to 777, 16 heads: 48 us as 256, 39 as 128; 2 chunks of up to 1024, 64 heads: 1.08 and 1.40 ms)
    p->rows = p->seqs.max_q > 128 && p->H * ((p->seqs.n_tokens + 255) / 256) >= kGroups ? 256 : 128;
    p->groups = kGroups;
    return kSumsBytes + part_bytes(*p) + p->heads * head;
}

hipError_t latent_prefill_launch(const LatentPrefillParams &p0, hipStream_t st) {
    LatentPrefillParams p = p0;
    if (p.seqs.n_seqs == 0 || p.seqs.max_q == 0) return hipSuccess;
    unsigned char *at = (unsigned char *)p.sums + kSumsBytes;
    p.part = (float *)at;
    p.keys = at + part_bytes(p);
    p.values = p.keys + p.heads * p.cap * kD * 2;
    p.rest = p.q_bf16 ? 0 : p.heads * p.cap * 2 * kD * 2;
    const int most = p.heads;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    auto of = [&](auto dc, auto rb, auto two) {
        constexpr int DC = decltype(dc)::value, RB = decltype(rb)::value, R = 128 * RB;
        constexpr bool TWO = decltype(two)::value;
        constexpr int ST = step_tokens(TWO);
        auto expand = latent_expand_kernel<DC>;
        auto attend = latent_prefill_kernel<DC, RB, TWO>;
        const int lds_e = kExpandTok * 2 * DC, lds_a = 3 * ST * ((TWO ? 8 : 4) * kD + 2 * kLatentRope);
        (void)hipFuncSetAttribute((const void *)expand, hipFuncAttributeMaxDynamicSharedMemorySize, lds_e);
        (void)hipFuncSetAttribute((const void *)attend, hipFuncAttributeMaxDynamicSharedMemorySize, lds_a);
        for (p.head0 = 0; p.head0 < p.H; p.head0 += most) {
            p.heads = std::min(most, p.H - p.head0);
            expand<<<dim3(p.groups), dim3(kThreads), lds_e, st>>>(p);
            hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            attend<<<dim3(p.groups), dim3(kAttendThreads), lds_a, st>>>(p);
            e = hipGetLastError();
            if (e != hipSuccess) return e;
            const int64_t blocks = ((int64_t)p.seqs.max_q + R - 1) / R * (R / 64);
            latent_prefill_merge_kernel<R, ST><<<dim3((unsigned)blocks, p.heads, p.seqs.n_seqs), dim3(kThreads), 0, st>>>(p);
            e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    };
    auto by_type = [&](auto dc, auto rb) { return p.q_bf16 ? of(dc, rb, std::false_type{}) : of(dc, rb, std::true_type{}); };
    auto by_rows = [&](auto dc) { return p.rows == 128 ? by_type(dc, std::integral_constant<int, 1>{}) : by_type(dc, std::integral_constant<int, 2>{}); };
    return p.Dc == 512 ? by_rows(std::integral_constant<int, 512>{}) : by_rows(std::integral_constant<int, 256>{});
}

}  // namespace akv
