// Attention over the paged 4-bit cache for chunks of a prompt: many query rows a sequence.
// Bound by the matrix cores and the softmax around them.
//
// A workgroup of W waves takes 32 W rows (query token, head of the group) of one sequence and
// cached head, each wave 32 of them as the columns of 32x32x16 MFMAs, and walks the cache in
// steps of 64 tokens, two buffers in LDS: while the MFMAs read one step, the next step's tiles
// are in flight to registers, one wave a tile and side, and are then dequantized into the
// other buffer, once for all rows.  Scores, running maximum and sum are float32.  Keys are two float16
// that add up to c s + z, so that scores are exact to float32 sums; values are one float16, and p is one
// for bfloat16 outputs, two (PTWO) for float16.  The outputs' own rounding leaves 1.68e-3 (bfloat16) and
// 2.0e-4 (float16) of their norm, all together 1.70e-3 and 2.8e-4.  (Keys as one float16 took three
// chunks of 65 to 512 tokens on 64 heads after 2k to 32k from 900 to 710 us, but with a channel ten times
// the others bfloat16 outputs were 2.0e-3 off, and not those of a call that asks for log-sums.)
// Eight chunks of 512 tokens on 64 heads over 8 after 8k: bfloat16 1.57 ms, float16 2.1.
//   K  [64 tokens][D / 8 chunks] of 16 bytes, chunk c at place c ^ turn(token) of its row;
//   V  the PV operand: [tile][32 channels][lane] of 16 bytes, tokens 4 hi + 0..3, 8 + 4 hi + 0..3;
//      row 16 b + r of its MFMA is channel 2 r + b of the 32.
// Both keep the eight lanes that LDS serves at a time on different banks, written and read.
// S^T = K Q^T leaves a lane with 16 scores of its row for every 32 tokens, which are the PV
// operand's tokens in order, so p goes from registers to the second product.
//
// The rows' tiles of all sequences and heads form one list whose entries count the tokens they
// see; it is cut into equal runs, one a workgroup.  Entries that several share leave partial
// states for paged_tile_merge_kernel.
#include <algorithm>
#include <type_traits>

#include "akv_common.h"
#include "paged.h"
#include "paged_device.h"

namespace akv {
namespace {

constexpr int kStep = 64;               // tokens a step: a tile for each wave of a group
constexpr int kTileWaves = 8;
constexpr int kSetupTok = 2 * kStep;    // what an entry's start counts
// p is held times 2^13, and the running maximum may lag behind by two log2 units: p in (0, 2^15] keeps 11
// bits down to 2^-27 of the largest weight and something down to 2^-38.  (With 2^7 and a lag of eight, bfloat16
// outputs were 3.6e-3 of the norm off where 65535 tokens share 1e-4 of the weight.)
constexpr float kLag = 2.0f;
constexpr float kPBias = 13.0f;

typedef float f16v __attribute__((ext_vector_type(16)));

struct TileSeq {
    SeqRows r;
    int rows, tiles;
    int64_t a, b;                       // entry t counts a + b t
    __device__ __forceinline__ int64_t cost(int t) const { return a + b * t; }
    __device__ __forceinline__ int64_t before(int64_t t) const { return a * t + b * (t * (t - 1) / 2); }
};
template <int R>
__device__ __forceinline__ TileSeq tile_seq(const PagedAttnParams &p, int s, bool uniform = true) {
    TileSeq q;
    q.r = seq_rows(p.seqs, s, p.pool.log_tpp + 4);
    if (uniform) q.r = wave_uniform(q.r);
    q.rows = min(q.r.n, p.seqs.max_q) * p.g;
    q.tiles = q.rows > p.few_rows ? (q.rows + R - 1) / R : 0;
    const int64_t old = min(max(q.r.at, 0), q.r.kv);
    q.a = (int64_t)p.g * ((p.causal ? old : q.r.kv) + kSetupTok) + R;
    q.b = p.causal ? R : 0;
    return q;
}
// Tokens that row `row` sees.
__device__ __forceinline__ int sees(const PagedAttnParams &p, const TileSeq &q, int row) {
    return q.r.sees(p.causal, row / p.g);
}
template <int R>
__device__ __forceinline__ int steps_of(const PagedAttnParams &p, const TileSeq &q, int t) {
    return max(1, (sees(p, q, min((t + 1) * R, q.rows) - 1) + kStep - 1) / kStep);
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

template <int R>
__device__ __forceinline__ void scan_tiles(const PagedAttnParams &p, int64_t *pre, int64_t *wave_sum, int per) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int64_t mine = 0;
    for (int i = 0; i < per; ++i) {
        const int s = t * per + i;
        if (s < p.seqs.n_seqs) {
            const TileSeq q = tile_seq<R>(p, s, false);
            mine += q.before(q.tiles) * p.pool.heads;
        }
    }
    int64_t inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wave_sum[wave] = inc;
    __syncthreads();
    int64_t before = 0;
    for (int w = 0; w < wave; ++w) before += wave_sum[w];
    pre[t] = before + inc - mine;
    if (t == (int)blockDim.x - 1) pre[blockDim.x] = before + inc;
    __syncthreads();
}

__device__ __forceinline__ int64_t tile_share(const PagedAttnParams &p, int64_t total) {
    return max((total + p.tile_groups - 1) / p.tile_groups, (int64_t)4 * kStep * p.g);
}

// Neighbouring tokens, whose chunks are written together, differ in bit 2, and any eight in a row
// in all three.
__device__ __forceinline__ int turn(int token) { return (token & 1) << 2 | (token & 2) | (token >> 2 & 1); }

// The four pairs of a dword of codes (nibbles n and n + 4 of it) as two float16 that add up to c s + z
// (to 2^-22 of it).
__device__ __forceinline__ void dequant8_two(const Nibbles &nb, uint32_t w, h2 s, h2 z, uint32_t *o, uint32_t *lo) {
    const uint32_t v = w >> 8;
    const h2 c[4] = {nb.low(w), nb.high(w), nb.low(v), nb.high(v)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = __builtin_fmaf((float)c[i][0], (float)s[0], (float)z[0]);
        const float b = __builtin_fmaf((float)c[i][1], (float)s[1], (float)z[1]);
        const h2 hi = {(_Float16)a, (_Float16)b};
        o[i] = as_u32(hi);
        lo[i] = as_u32((h2){(_Float16)(a - (float)hi[0]), (_Float16)(b - (float)hi[1])});
    }
}

// N products of operands in LDS, AHEAD of them loaded before the first, one more behind each:
// read(i) loads operand i, mul(i, a) takes it.  (Left to itself the compiler loads an operand,
// waits and multiplies, 32 times a step.)
constexpr int kAhead = 4;
template <int N, typename Read, typename Mul>
__device__ __forceinline__ void products(Read read, Mul mul) {
    h8 a[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) a[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        mul(i, a[i % kAhead]);
        if (i + kAhead < N) a[i % kAhead] = read(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// One tile of K or V on its way from memory to LDS.  What a load brings stays as it is until it
// is staged: any use before would wait for it.
template <int N>
struct Words {  // N dwords of one load: 4, 2 or 1
    typedef uint32_t vec __attribute__((ext_vector_type(N)));
    vec v;
    __device__ __forceinline__ void load(const unsigned char *tile, uint32_t at) { v = *(const vec *)(tile + at); }
    __device__ __forceinline__ uint32_t operator[](int i) const { return v[i]; }
};
template <>
struct Words<1> {
    uint32_t v;
    __device__ __forceinline__ void load(const unsigned char *tile, uint32_t at) { v = *(const uint32_t *)(tile + at); }
    __device__ __forceinline__ uint32_t operator[](int) const { return v; }
};

template <int D, int NG>
struct KLoad {
    Words<D / 32> c;
    Words<NG> m;
    __device__ __forceinline__ void load(const unsigned char *tile, int lane) {
        c.load(tile, (uint32_t)lane * (D / 8));
        m.load(tile + 16 * D, (uint32_t)(lane >> 2) * (NG * 4));
    }
    // lane (token lane / 4, i = lane % 4): chunk 4 g + i
    __device__ __forceinline__ void stage(unsigned char *kt, int tile, int lane, const Nibbles &nb) const {
        const int tok = 16 * tile + (lane >> 2), i = lane & 3;
#pragma unroll
        for (int g = 0; g < D / 32; ++g) {
            const uint32_t w = m[g * NG / (D / 32)];
            const h2 s = as_h2((w & 0xffffu) | (w << 16)), z = as_h2((w >> 16) | (w & 0xffff0000u));
            uint32_t o[4], r[4];
            dequant8_two(nb, c[g], s, z, o, r);
            u4 *d = (u4 *)(kt + tok * (2 * D) + (((4 * g + i) ^ turn(tok)) << 4));
            *d = (u4){o[0], o[1], o[2], o[3]};
            d[kStep * 2 * D / 16] = (u4){r[0], r[1], r[2], r[3]};
        }
    }
};
template <int D, int NG>
struct VLoad {
    static constexpr int NL = NG == 4 ? 2 : 1;  // groups a lane's channels lie in
    Words<D / 32> c[2];                         // (quad a, a + 2): pairs (p, h) of row r
    Words<1> m;                                 // a dword of the tile's meta
    __device__ __forceinline__ void load(const unsigned char *tile, int lane) {
        m.load(tile + 16 * D + 64 * NG, (uint32_t)(lane & (16 * NG - 1)) * 4);
        const uint32_t r = lane & 15, a = (lane >> 4) & 1;
#pragma unroll
        for (int q = 0; q < 2; ++q) c[q].load(tile + 8 * D + q * 4 * D, (a * 16 + r) * (D / 8));
    }
    // The meta goes through LDS: a lane needs up to 16 dwords of it, which read from memory took
    // four loads more and 16 registers through the products (500 of a step's 4700 cycles).
    __device__ __forceinline__ void post(uint32_t *meta, int lane) const { meta[lane & (16 * NG - 1)] = m[0]; }
    // Where rows see different tokens, values that are not finite would reach those that do not
    // see them as 0 * NaN.  They become 0 in the lane's part of the staged tile, and word (h, a)
    // of the tile's four says which, for `poison`: bit 16 half + 4 l + 2 q + pr.
    static __device__ __forceinline__ void hide(unsigned char *vt, uint32_t *bad, int tile, int lane) {
        constexpr int L = D / 64;
        asm volatile("" : "+v"(lane));  // or what comes of it is kept in registers through the whole loop
        const int r = lane & 15, a = (lane >> 4) & 1, h = lane >> 5;
        unsigned char *at = vt + (tile * (D / 32) * 64 + a * 32 + r) * 16 + h * (L * 1024);
        uint32_t w = 0;
#pragma unroll
        for (int l = 0; l < L; ++l) {
            u4 *d = (u4 *)(at + l * 1024);
            u4 x = d[0], y = d[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t b = not_finite(x[i]);
                x[i] &= ~b, y[i] &= ~b;  // of one group, so both or none
                w |= (b & 0x10001u) << (4 * l + i);
            }
            d[0] = x, d[16] = y;
        }
        if (r == 0) bad[2 * h + a] = w;
    }
    // What `hide` left of a step, for a row that sees its first `see` tokens: the groups whose
    // values are not finite.
    static __device__ __forceinline__ uint32_t poison(const uint32_t *bad, int lane, int see) {
        asm volatile("" : "+v"(lane));
        const uint32_t mine = bad[lane & 15];
        uint32_t groups = 0;
        for (uint64_t left = __builtin_amdgcn_ballot_w64(mine != 0) & 0xffffu; left; left &= left - 1) {
            const int from = __builtin_ctzll(left), a = from & 1, h = from >> 1 & 1;
            for (uint32_t w = __builtin_amdgcn_readlane(mine, from); w; w &= w - 1) {
                const int bit = __builtin_ctz(w), half = bit >> 4, l = bit >> 2 & 1, q = bit >> 1 & 1, pr = bit & 1;
                const int tok = 16 * (from >> 2) + 4 * (a + 2 * q) + 2 * pr + half;
                if (tok < see) groups |= 1u << ((D == 128 ? 2 * h + l : h) / (D / 32 / NG));
            }
        }
        return groups;
    }
    // lane (row r of the codes, quads a and a + 2, h): the 16 bytes of channels 32 (2 h + l) + 2 r + b;
    // at D = 64 h says which l of the two.  Slots from token nv on become 0.
    __device__ __forceinline__ void stage(unsigned char *vt, const uint32_t *meta, int tile, int lane, const Nibbles &nb, int nv) const {
        constexpr int L = D / 64;
        const int r = lane & 15, a = (lane >> 4) & 1, h = lane >> 5;
        uint32_t s[2][2 * NL], z[2][2 * NL];    // the quads' pairs (group, p)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            typedef uint32_t vec __attribute__((ext_vector_type(2 * NL)));
            const uint32_t at = ((a + 2 * q) * NG + (NG == 4 ? 2 * h : NG == 2 ? h : 0)) * 2;
            const vec sv = *(const vec *)(meta + at), zv = *(const vec *)(meta + 8 * NG + at);
#pragma unroll
            for (int i = 0; i < 2 * NL; ++i) s[q][i] = sv[i], z[q][i] = zv[i];
        }
        uint32_t keep[2][2] = {{~0u, ~0u}, {~0u, ~0u}};
        if (nv < 16) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int pr = 0; pr < 2; ++pr) {
                    const int tok = 4 * (a + 2 * q) + 2 * pr;
                    keep[q][pr] = (tok < nv ? 0xffffu : 0u) | (tok + 1 < nv ? 0xffff0000u : 0u);
                }
        }
        uint32_t w[2][2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int pr = 0; pr < 2; ++pr) {
                if constexpr (D == 128) w[q][pr] = h ? c[q][2 * pr + 1] : c[q][2 * pr];
                else w[q][pr] = c[q][pr] >> (8 * h);
            }
        unsigned char *at = vt + (tile * (D / 32) * 64 + a * 32 + r) * 16 + h * (L * 1024);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            u4 o[2];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int pr = 0; pr < 2; ++pr) {
                    const uint32_t v = w[q][pr] >> (8 * l);
                    const int mi = (NL == 2 ? 2 * l : 0) + pr;
                    const h2 sv = as_h2(s[q][mi] & keep[q][pr]), zv = as_h2(z[q][mi] & keep[q][pr]);
                    o[0][2 * q + pr] = as_u32(__builtin_elementwise_fma(nb.low(v), sv, zv));
                    o[1][2 * q + pr] = as_u32(__builtin_elementwise_fma(nb.high(v), sv, zv));
                }
            u4 *d = (u4 *)(at + l * 1024);
            d[0] = o[0], d[16] = o[1];
        }
    }
};

// The operand of 32 query rows: lane (row col, hi) has channels 8 c + (0, 4, 1, 5, 2, 6, 3, 7) of
// chunk c = 2 st + hi, the row divided by 2^ex so that its maximum lies in [1/2, 1).  Returns ex.
template <int D>
__device__ __forceinline__ int tile_query(h8 (&op)[D / 16], const u4 (&w)[D / 16], bool bf16) {
    if (bf16) {
        float y[D / 16][8], top = 0.0f;
#pragma unroll
        for (int st = 0; st < D / 16; ++st)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[st][i] = __builtin_bit_cast(float, i & 1 ? w[st][i >> 1] & 0xffff0000u : w[st][i >> 1] << 16);
                top = __builtin_fmaxf(top, __builtin_fabsf(y[st][i]));
            }
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const int ex = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
        for (int st = 0; st < D / 16; ++st) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[st][i] = __builtin_ldexpf(y[st][i], -ex);
            op[st] = (h8){(_Float16)y[st][0], (_Float16)y[st][4], (_Float16)y[st][1], (_Float16)y[st][5],
                          (_Float16)y[st][2], (_Float16)y[st][6], (_Float16)y[st][3], (_Float16)y[st][7]};
        }
        return ex;
    }
    typedef uint16_t s2 __attribute__((ext_vector_type(2)));
    s2 most = {0, 0};
#pragma unroll
    for (int st = 0; st < D / 16; ++st)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            most = __builtin_elementwise_max(most, __builtin_bit_cast(s2, (uint32_t)w[st][i] & 0x7fff7fffu));
    float top = (float)__builtin_bit_cast(_Float16, most[0] > most[1] ? most[0] : most[1]);
    top = __builtin_fmaxf(top, __shfl_xor(top, 32));
    const int ex = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 0;
    const int e1 = min(-ex, 15);  // 2^15 is float16's largest: small rows go in two steps
    const _Float16 a = (_Float16)__builtin_ldexpf(1.0f, e1), c = (_Float16)__builtin_ldexpf(1.0f, -ex - e1);
#pragma unroll
    for (int st = 0; st < D / 16; ++st) {
        u4 y;
#pragma unroll
        for (int n = 0; n < 4; ++n)  // channels n and n + 4
            y[n] = as_u32(as_h2(__builtin_amdgcn_perm((uint32_t)w[st][2 + (n >> 1)], (uint32_t)w[st][n >> 1],
                                                      n & 1 ? 0x07060302u : 0x05040100u)) * (h2){a, a} * (h2){c, c});
        op[st] = __builtin_bit_cast(h8, y);
    }
    return ex;
}

}  // namespace

template <int D, int NG, int W, bool PTWO>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_tile_kernel(const PagedAttnParams p) {
    constexpr int R = 32 * W, NB = D / 32, TB = paged_tile_bytes(D, NG), EROW = D + 4;
    constexpr int KT = 2 * kStep * 2 * D, BUF = KT + kStep * 2 * D;
    extern __shared__ __align__(16) unsigned char smem[];
    int64_t *pre = (int64_t *)smem, *wave_sum = pre + 64 * W + 1;  // before the first step only
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, hi = lane >> 5;

    const int per = (p.seqs.n_seqs + 64 * W - 1) / (64 * W);
    scan_tiles<R>(p, pre, wave_sum, per);
    const int64_t total = uniform64(pre[64 * W]);
    const int64_t share = tile_share(p, total);
    if (blockIdx.x == 0) {  // for the merge
        int64_t *sums = (int64_t *)p.sums;
        sums[threadIdx.x] = pre[threadIdx.x];
        if (threadIdx.x == 0) sums[64 * W] = total;
    }
    int64_t x = min((int64_t)blockIdx.x * share, total);
    const int64_t x_end = min(x + share, total);
    if (x >= x_end) return;
    int at = 0;  // the last sum at or below x
    for (int step = 32 * W; step > 0; step >>= 1)
        if (pre[at + step] <= x) at += step;
    int s = __builtin_amdgcn_readfirstlane(at * per);
    int64_t off = uniform64(x - pre[at]);
    __syncthreads();  // pre is done with
    TileSeq q = tile_seq<R>(p, s);
    while (off >= q.before(q.tiles) * p.pool.heads) {
        off -= q.before(q.tiles) * p.pool.heads;
        q = tile_seq<R>(p, ++s);
    }

    while (x < x_end) {
        const int64_t head_cost = q.before(q.tiles);
        const int h = __builtin_amdgcn_readfirstlane((int)(off / head_cost));
        const int64_t in_head = off - h * head_cost;
        int t = 0;
        for (int step = 1 << (31 - __builtin_clz(q.tiles)); step > 0; step >>= 1)
            if (t + step < q.tiles && q.before(t + step) <= in_head) t += step;
        t = __builtin_amdgcn_readfirstlane(t);
        const int64_t c0 = in_head - q.before(t), cost = q.cost(t);
        const int64_t c1 = min(cost, c0 + (x_end - x));
        const int n_steps = steps_of<R>(p, q, t);
        const int f0 = __builtin_amdgcn_readfirstlane((int)(c0 * n_steps / cost));
        const int f1 = __builtin_amdgcn_readfirstlane((int)(c1 * n_steps / cost));
        x += c1 - c0;
        off += c1 - c0;
        if (f0 < f1) {
            const int row0 = t * R + 32 * wave;
            const int row = min(row0 + col, q.rows - 1);
            const int head = h * p.g + row % p.g;
            const bool idle = row0 >= q.rows;
            const int see = sees(p, q, row);
            const int see_all = idle ? 0 : sees(p, q, row0), see_any = idle ? 0 : sees(p, q, min(row0 + 31, q.rows - 1));

            // steps that have tokens: a tile of rows that see nothing has none
            const int f2 = min(f1, (sees(p, q, min((t + 1) * R, q.rows) - 1) + kStep - 1) / kStep);
            const int32_t *table = p.seqs.table + s * p.seqs.table_stride;
            float mx = kMinMax, l = 0.0f;
            uint32_t poisoned = 0;  // groups of channels in which the row sees a value that is not finite
            f16v acc[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[b][i] = 0.0f;

            // Waves 0-3 stage K, waves 4-7 V, a tile each, and run half a step behind: one group's
            // products meet the other's softmax and staging on each SIMD (keys as one float16, chunks of
            // 65 to 512 tokens on 64 heads after 2k to 32k: 0.80 ms without the offset, 0.74 with it).
            // Slots between barriers, t a step:
            //   2 t      K group's products (t), V group's softmax (t - 1)
            //   2 t + 1  K group's softmax (t), V group's products (t)
            // where products (t) are P V of step t - 1 and Q K of step t.  K (t + 1) is staged after
            // the K group's softmax (t), V (t + 1) after the V group's, each into the buffer whose
            // last reader was a slot before.  Each group has its own copy of the loop, and its loads
            // are not conditional (the last step's again at the end): registers that a branch may or
            // may not load are copied behind it, which waits for the load.
            auto walk = [&](auto is_late) {
                constexpr bool late = decltype(is_late)::value;
                const int log_tpp = p.pool.log_tpp, tl = wave & 3;
                // lane i: the address of this head's tiles in the page at entry pb + i of the table
                // (of page 0 where that is no page of the pool), and which entries are pages
                int pb;
                uint32_t page_lo, page_hi;
                uint64_t valid;
                auto pages = [&](int step) {
                    pb = (4 * step) >> log_tpp;
                    uint32_t id = pb + lane < p.seqs.width ? (uint32_t)table[pb + lane] : ~0u;
                    valid = __builtin_amdgcn_ballot_w64(id < p.pool.n_pages);
                    if (id >= p.pool.n_pages) id = 0;
                    const uint64_t at = (uint64_t)p.pool.base + id * (uint64_t)p.pool.page_bytes + ((uint64_t)(h * TB) << log_tpp);
                    page_lo = (uint32_t)at;
                    page_hi = (uint32_t)(at >> 32);
                };
                pages(f0);
                std::conditional_t<late, VLoad<D, NG>, KLoad<D, NG>> raw;
                Nibbles nb;
                nb.init();
                int nv = 0;         // tokens of the wave's tile of the step that was loaded last
                uint32_t have = 0;  // and which of the step's four tiles have a page
                auto load = [&](int step) {
                    const int t0 = 4 * step, mine = t0 + tl, last = (t0 + 3) >> log_tpp;
                    if (last - pb >= 64) pages(step);
                    const int e0 = (t0 >> log_tpp) - pb, e1 = (mine >> log_tpp) - pb;
                    const uint32_t all = (2u << (last - pb - e0)) - 1;
                    have = 15;
                    if (((uint32_t)(valid >> e0) & all) != all) {
                        have = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) have |= (uint32_t)(valid >> (((t0 + i) >> log_tpp) - pb) & 1) << i;
                    }
                    nv = have >> tl & 1 ? min(max(q.r.kv - 16 * mine, 0), 16) : 0;
                    const uint64_t at = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane(page_hi, e1) << 32 |
                                         (uint32_t)__builtin_amdgcn_readlane(page_lo, e1)) +
                                        (uint32_t)((mine & ((1 << log_tpp) - 1)) * TB);
                    raw.load((const unsigned char *)at, lane);
                };
                const int all_see = sees(p, q, t * R);
                auto apart = [&](int step) { return kStep * (step + 1) > all_see; };  // rows see different tokens of it
                uint32_t *meta = (uint32_t *)(smem + 2 * BUF) + 2 * 16 + 16 * NG * tl;
                auto post = [&] {
                    if constexpr (late) raw.post(meta, lane);
                };
                auto stage = [&](unsigned char *buf, int step) {
                    if constexpr (late) {
                        raw.stage(buf + KT, meta, tl, lane, nb, nv);
                        if (apart(step)) raw.hide(buf + KT, (uint32_t *)(smem + 2 * BUF) + 16 * ((step - f0) & 1) + 4 * tl, tl, lane);
                    } else {
                        raw.stage(buf, tl, lane, nb);
                    }
                };
                load(f0);

                // ---- the query operand: chunk c = 2 st + hi, channels 8 c + (0, 4, 1, 5, 2, 6, 3, 7)
                h8 qop[D / 16];
                float kx;
                {
                    const unsigned char *qr = p.q + (q.r.begin + row / p.g) * p.q_t + head * p.q_h;
                    u4 w[D / 16];
#pragma unroll
                    for (int st = 0; st < D / 16; ++st) w[st] = *(const u4 *)(qr + (2 * st + hi) * 16);
                    const int ex = tile_query<D>(qop, w, p.q_bf16);
                    kx = __builtin_ldexpf(p.scale_log2, ex);
                }

                f16v sc[2];
                h8 pop[4];
                auto scores = [&](const unsigned char *buf) {  // operand: (chunk pair, half of K, 32 tokens)
#pragma unroll
                    for (int i = 0; i < 32; ++i) sc[i >> 4][i & 15] = 0.0f;
                    products<4 * (D / 16)>(
                        [&](int i) {
                            const int st = i / 4, part = i / 2 % 2, b = i & 1;
                            return *(const h8 *)(buf + part * (kStep * 2 * D) + (32 * b + col) * (2 * D) + (((2 * st + hi) ^ turn(col)) << 4));
                        },
                        [&](int i, h8 a) { sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qop[i / 4], sc[i & 1], 0, 0, 0); });
                };
                auto softmax = [&](int step, uint32_t here) {
                    if (kStep * (step + 1) > see_all || here != 15u) {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int tok = 32 * b + 8 * (i >> 2) + 4 * hi + (i & 3);
                                if (kStep * step + tok >= see || !(here >> (tok >> 4) & 1)) sc[b][i] = -INFINITY;
                            }
                    }
                    if (apart(step))
                        poisoned |= VLoad<D, NG>::poison((uint32_t *)(smem + 2 * BUF) + 16 * ((step - f0) & 1), lane, see - kStep * step);
                    float top = sc[0][0];
#pragma unroll
                    for (int i = 1; i < 32; ++i) top = __builtin_fmaxf(top, sc[i >> 4][i & 15]);
                    if (__builtin_amdgcn_ballot_w64(__builtin_fmaf(top, kx, kPBias - mx) > kPBias + kLag)) {
                        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                        const float mn = top * kx > mx ? running_max(top, kx, kPBias) : mx;
                        const float alpha = __builtin_amdgcn_exp2f(mx - mn);
                        l *= alpha;
#pragma unroll
                        for (int b = 0; b < NB; ++b) acc[b] *= alpha;
                        mx = mn;
                    }
                    const float bias = kPBias - mx;
#pragma unroll
                    for (int tile = 0; tile < 4; ++tile) {
                        float pr[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            pr[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[tile >> 1][8 * (tile & 1) + i], kx, bias));
                        if constexpr (PTWO)
#pragma unroll
                            for (int i = 0; i < 8; ++i) sc[tile >> 1][8 * (tile & 1) + i] = pr[i];
                        else
                            pop[tile] = (h8){(_Float16)pr[0], (_Float16)pr[1], (_Float16)pr[2], (_Float16)pr[3],
                                             (_Float16)pr[4], (_Float16)pr[5], (_Float16)pr[6], (_Float16)pr[7]};
                        l += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
                    }
                };
                auto outputs = [&](const unsigned char *buf) {
                    auto read = [&](int i) { return *(const h8 *)(buf + KT + (i * 64 + lane) * 16); };
                    if constexpr (PTWO) {  // p waits in the scores' registers; an operand's second product
                                           // comes behind the next one's first, or it would wait for its own
                        h8 ph[4], pl[4], was;
                        products<4 * NB>(read, [&](int i, h8 a) {
                            const int t4 = i / NB;
                            if (i % NB == 0)
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const float x = sc[t4 >> 1][8 * (t4 & 1) + j];
                                    ph[t4][j] = (_Float16)x;
                                    pl[t4][j] = (_Float16)(x - (float)ph[t4][j]);
                                }
                            acc[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[t4], acc[i % NB], 0, 0, 0);
                            if (i > 0) acc[(i - 1) % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(was, pl[(i - 1) / NB], acc[(i - 1) % NB], 0, 0, 0);
                            was = a;
                        });
                        acc[NB - 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(was, pl[3], acc[NB - 1], 0, 0, 0);
                    } else {
                        products<4 * NB>(read, [&](int i, h8 a) {
                            acc[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pop[i / NB], acc[i % NB], 0, 0, 0);
                        });
                    }
                };

                post();
                stage(smem, f0);
                __syncthreads();
                if (late) __syncthreads();
                for (int step = f0; step < f2; ++step) {
                    unsigned char *buf = smem + ((step - f0) & 1) * BUF, *other = smem + ((step - f0 + 1) & 1) * BUF;
                    const uint32_t here = have;
                    const bool seen = kStep * step < see_any;
                    load(min(step + 1, f2 - 1));
                    if (step > f0 && kStep * (step - 1) < see_any) outputs(other);
                    if (seen) scores(buf);
                    post();
                    __syncthreads();
                    if (seen) softmax(step, here);
                    if (step + 1 < f2) stage(other, step + 1);
                    __syncthreads();
                }
                if (!late) __syncthreads();
                if (kStep * (f2 - 1) < see_any) outputs(smem + ((f2 - 1 - f0) & 1) * BUF);
                __syncthreads();
            };
            if (f0 < f2) {
                if (wave < W / 2) walk(std::false_type{});
                else walk(std::true_type{});
            }

            l += __shfl_xor(l, 32);
            if (__builtin_amdgcn_ballot_w64(poisoned != 0))
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    if (poisoned >> (b / (NB / NG)) & 1) acc[b] += NAN;
            if (row0 + col < q.rows) {
                if (f0 == 0 && f1 == n_steps) {
                    const int64_t o = (q.r.begin + row / p.g) * p.Hq + head;
                    const float inv = row_inverse(l);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {  // channels 32 b + 16 k + 8 hi ..: pairs of rows r, 16 + r
                            u4 v;
#pragma unroll
                            for (int j = 0; j < 4; ++j) v[j] = to_pair(p.q_bf16, acc[b][4 * k + j] * inv, acc[b][8 + 4 * k + j] * inv);
                            *(u4 *)((unsigned char *)p.out + (o * D + 32 * b + 16 * k + 8 * hi) * 2) = v;
                        }
                    if (p.lse && hi == 0) p.lse[o] = row_lse(mx, l, kPBias);
                } else {
                    float *pr = p.tile_part + ((int64_t)(2 * blockIdx.x + (f0 == 0 ? 1 : 0)) * R + 32 * wave + col) * EROW;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            *(f4 *)(pr + 32 * b + 16 * (k >> 1) + 8 * hi + 4 * (k & 1)) =
                                (f4){acc[b][4 * (k >> 1) + 2 * (k & 1)], acc[b][8 + 4 * (k >> 1) + 2 * (k & 1)],
                                     acc[b][4 * (k >> 1) + 2 * (k & 1) + 1], acc[b][8 + 4 * (k >> 1) + 2 * (k & 1) + 1]};
                    if (hi == 0) pr[D] = mx, pr[D + 1] = l;
                }
            }
        }
        if (x < x_end && off >= head_cost * p.pool.heads) {
            do q = tile_seq<R>(p, ++s);
            while (q.tiles == 0);
            off = 0;
        }
    }
}

constexpr int kMergeRows = 64;
// Entries that several workgroups share, joined in order: kMergeRows rows of the entry that holds
// the start of a run, a workgroup, by the first start in it.  Bound by the states' bytes and the search's latency (255
// starts, 69 MB at D = 128: 18 us; 16 rows a workgroup 24, 32 rows 20).
template <int D, int W>
__global__ __launch_bounds__(256) void paged_tile_merge_kernel(const PagedAttnParams p) {
    constexpr int R = 32 * W, EROW = D + 4, CH = D / 16, B = 2, J = kMergeRows / 16;
    static_assert(64 * W % 256 == 0, "whole rounds of sums");
    const int64_t *sums = (const int64_t *)p.sums;
    const int64_t total = sums[64 * W], share = tile_share(p, total);
    const int64_t x = (blockIdx.x + 1) * share;
    if (x >= total) return;
    int at = -1;  // the last sum at or below x
    for (int i = threadIdx.x; i < 64 * W; i += 256) at += __syncthreads_count(sums[i] <= x);
    const int per = (p.seqs.n_seqs + 64 * W - 1) / (64 * W);
    int s = at * per;
    int64_t off = x - sums[at];
    TileSeq q = tile_seq<R>(p, s);
    while (off >= q.before(q.tiles) * p.pool.heads) {
        off -= q.before(q.tiles) * p.pool.heads;
        q = tile_seq<R>(p, ++s);
    }
    const int h = (int)(off / q.before(q.tiles));
    const int64_t in_head = off - h * q.before(q.tiles);
    int t = 0;
    for (int step = 1 << (31 - __builtin_clz(q.tiles)); step > 0; step >>= 1)
        if (t + step < q.tiles && q.before(t + step) <= in_head) t += step;
    const int64_t u0 = x - (in_head - q.before(t)), cost = q.cost(t);
    const int64_t g0 = u0 / share, g1 = (u0 + cost - 1) / share;
    const int in = kMergeRows * blockIdx.y + (threadIdx.x >> 4), ch = (threadIdx.x & 15) * CH;
    const int row0 = t * R + in;
    if (g0 != blockIdx.x || row0 >= q.rows) return;
    const int n_steps = steps_of<R>(p, q, t);
    float o[J][CH];
    float M[J], L[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        M[j] = kMinMax, L[j] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) o[j][c] = 0.f;
    }
    int f1 = 0;  // steps before run g
    for (int64_t g = g0; g <= g1; g += B) {
        f4 v[B][J][CH / 4];
        f2 ml[B][J];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int f0 = f1;
            f1 = g + i < g1 ? (int)(((g + i + 1) * share - u0) * n_steps / cost) : n_steps;
            if (f0 == 0 && f1 == n_steps) return;  // one workgroup had every step of it, and wrote
            const float *pr = p.tile_part + ((2 * (g + i) + (f0 == 0 ? 1 : 0)) * R + in) * EROW;
#pragma unroll
            for (int j = 0; j < J; ++j) {  // rows past the last are of the tile too
#pragma unroll
                for (int c = 0; c < CH / 4; ++c) v[i][j][c] = f0 < f1 ? ((const f4 *)(pr + 16 * j * EROW + ch))[c] : (f4){0.f, 0.f, 0.f, 0.f};
                ml[i][j] = f0 < f1 ? *(const f2 *)(pr + 16 * j * EROW + D) : (f2){kMinMax, 0.f};
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float mn = M[j];
#pragma unroll
            for (int i = 0; i < B; ++i) mn = __builtin_fmaxf(mn, ml[i][j][0]);
            const float a = __builtin_amdgcn_exp2f(M[j] - mn);
            L[j] *= a;
#pragma unroll
            for (int c = 0; c < CH; ++c) o[j][c] *= a;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const float b = __builtin_amdgcn_exp2f(ml[i][j][0] - mn);
                L[j] = __builtin_fmaf(ml[i][j][1], b, L[j]);
#pragma unroll
                for (int c = 0; c < CH; ++c) o[j][c] = __builtin_fmaf(v[i][j][c >> 2][c & 3], b, o[j][c]);
            }
            M[j] = mn;
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int row = row0 + 16 * j;
        if (row >= q.rows) break;
        const int head = h * p.g + row % p.g;
        const int64_t ro = (q.r.begin + row / p.g) * p.Hq + head;
        const float inv = row_inverse(L[j]);
#pragma unroll
        for (int c = 0; c < CH / 4; ++c)
            *(u2 *)((unsigned char *)p.out + (ro * D + ch + 4 * c) * 2) =
                (u2){to_pair(p.q_bf16, o[j][4 * c] * inv, o[j][4 * c + 1] * inv), to_pair(p.q_bf16, o[j][4 * c + 2] * inv, o[j][4 * c + 3] * inv)};
        if (p.lse && ch == 0) p.lse[ro] = row_lse(M[j], L[j], kPBias);
    }
}

// The importance from many rows.  A workgroup takes 64 tokens of a sequence and all its heads: each
// of four waves stages a tile of the next head's keys (two float16 that add up to them, so that scores
// stay exact to float32) while the products read this one's, and takes 32 rows of every 128.  A
// lane sums its row's p of 32 tokens over heads and rows in registers; rows and waves are joined
// at the end, in a fixed order.  Bound by vector instructions (the query operand, again for every 64
// tokens, and the exponentials) and their latency, two waves a SIMD: 2048 rows a head on 8
// heads, two sequences of 12000 tokens: 0.36 ms; 278 TFLOP/s.
template <int D, int NG>
__global__ __launch_bounds__(256, 2) void paged_importance_tile_kernel(const PagedImportanceParams p) {
    constexpr int TB = paged_tile_bytes(D, NG), BUF = 2 * kStep * 2 * D;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float sums[4][kStep];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, hi = lane >> 5, s = blockIdx.y;
    const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_tpp + 4));
    const int n = min(r.n, p.seqs.max_q);
    const int64_t kv = n > 0 ? min((int64_t)r.kv, p.n_scores) : 0;  // tokens whose score changes
    const int tok0 = blockIdx.x * kStep;
    f16v sum[2];
#pragma unroll
    for (int i = 0; i < 32; ++i) sum[i >> 4][i & 15] = 0.0f;
    if (tok0 < kv) {
        const int first = p.q_window > 0 && p.q_window < n ? n - p.q_window : 0, rows = (n - first) * p.g;
        const int log_tpp = p.pool.log_tpp, mine = tok0 / 16 + wave;
        const int32_t *table = p.seqs.table + s * p.seqs.table_stride;
        // lane i < 4: the page of tile i; tiles past the end or outside the pool read page 0 and count nothing
        uint32_t id = lane < 4 && tok0 + 16 * lane < r.kv ? (uint32_t)table[(tok0 / 16 + lane) >> log_tpp] : ~0u;
        const uint32_t have = (uint32_t)__builtin_amdgcn_ballot_w64(id < p.pool.n_pages) & 15u;
        if (id >= p.pool.n_pages) id = 0;
        const unsigned char *tile = p.pool.base + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(id, wave) * p.pool.page_bytes +
                                    (uint32_t)((mine & ((1 << log_tpp) - 1)) * TB);
        const int64_t head_bytes = (int64_t)TB << log_tpp;
        KLoad<D, NG> raw;
        Nibbles nb;
        nb.init();
        u4 w[D / 16];  // the next rows' queries and log-sums, in flight
        float lse;
        auto fetch = [&](int h, int row0) {
            const int row = min(row0 + 32 * wave + col, rows - 1), head = h * p.g + row % p.g;
            const int64_t t = r.begin + first + row / p.g;
            const unsigned char *qr = p.q + t * p.q_t + head * p.q_h;
#pragma unroll
            for (int st = 0; st < D / 16; ++st) w[st] = *(const u4 *)(qr + (2 * st + hi) * 16);
            lse = p.lse[t * p.Hq + head];
        };
        raw.load(tile, lane);
        fetch(0, 0);
        raw.stage(smem, wave, lane, nb);
        __syncthreads();
        const int last = p.pool.heads - 1;
        for (int h = 0, row0 = 0;;) {
            const unsigned char *buf = smem + (h & 1) * BUF;
            const bool live = row0 + 32 * wave + col < rows;
            const int row = min(row0 + 32 * wave + col, rows - 1);
            const int see = live ? r.sees(p.causal, first + row / p.g) : 0;
            h8 op[D / 16];
            const float kx = __builtin_ldexpf(p.scale_log2, tile_query<D>(op, w, p.q_bf16));
            float bias = lse * -1.4426950408889634f;
            asm volatile("" : "+v"(bias));  // before the next log-sum's load: else that is copied, and waited for, at the end
            const bool more = row0 + 128 < rows;
            raw.load(tile + min(h + 1, last) * head_bytes, lane);  // (again for every 128 rows: not conditional, as above)
            fetch(more ? h : min(h + 1, last), more ? row0 + 128 : 0);
            if (row0 + 32 * wave < rows) {
                f16v sc[2];
#pragma unroll
                for (int i = 0; i < 32; ++i) sc[i >> 4][i & 15] = 0.0f;
                products<4 * (D / 16)>(
                    [&](int i) {
                        const int st = i / 4, part = i / 2 % 2, b = i & 1;
                        return *(const h8 *)(buf + part * (kStep * 2 * D) + (32 * b + col) * (2 * D) + (((2 * st + hi) ^ turn(col)) << 4));
                    },
                    [&](int i, h8 a) { sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, op[i / 4], sc[i & 1], 0, 0, 0); });
                const bool clean = have == 15u && __builtin_amdgcn_ballot_w64(tok0 + kStep <= see) == ~0ull;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][i], kx, bias));
                        if (!clean) {
                            const int tok = 32 * b + 8 * (i >> 2) + 4 * hi + (i & 3);
                            pr = tok0 + tok < see && (have >> (tok >> 4) & 1) ? pr : 0.0f;
                        }
                        sum[b][i] += pr;
                    }
            }
            row0 += 128;
            if (more) continue;
            if (h < last) raw.stage(smem + ((h + 1) & 1) * BUF, wave, lane, nb);
            __syncthreads();
            if (h == last) break;
            ++h;
            row0 = 0;
        }
    }
    // over the 32 rows: each step halves what a lane holds; lane col ends with value col of its 32
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = sum[i >> 4][i & 15];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < d; ++i) {
            float a = v[i], b = v[i + d];
            asm("" : "+v"(a), "+v"(b));  // or a choice of values becomes one of indexes, 32 selects long
            v[i] = (col & d ? b : a) + __shfl_xor(col & d ? a : b, d);
        }
    sums[wave][32 * (col >> 4) + 8 * ((col >> 2) & 3) + 4 * hi + (col & 3)] = v[0];
    __syncthreads();
    const int64_t j = (int64_t)tok0 + threadIdx.x;
    if (threadIdx.x >= kStep || j >= p.n_scores) return;
    const float *old = p.scores + s * p.score_stride + j;
    float *out = p.out + s * p.out_stride + j;
    if (j < kv) {
        const float x = ((sums[0][threadIdx.x] + sums[1][threadIdx.x]) + sums[2][threadIdx.x]) + sums[3][threadIdx.x];
        *out = __builtin_fmaf(*old, p.decay, x / (float)p.Hq);
    } else if (out != old) {
        *out = *old;
    }
}

namespace {
constexpr int kTileGroups = 256;  // one workgroup a compute unit
constexpr int64_t kTileSums = 8192;               // scan_tiles' sums at the start of the workspace
static_assert((64 * kTileWaves + 1) * 8 <= kTileSums, "the sums fit");

template <int D, int NG, bool PTWO>
hipError_t tile_go_as(const PagedAttnParams &p, hipStream_t st) {
    constexpr int W = kTileWaves;
    constexpr int LDS = 2 * 3 * kStep * 2 * D + (2 * 16 + 4 * 16 * NG) * 4;  // two buffers, what `hide` writes of each, V meta
    static_assert((64 * W + 1 + W) * 8 <= LDS, "the sums fit the buffers");
    auto kern = paged_tile_kernel<D, NG, W, PTWO>;
    if (LDS > 48 * 1024) (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    kern<<<dim3(p.tile_groups), dim3(64 * W), LDS, st>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.tile_groups == 1) return hipSuccess;
    paged_tile_merge_kernel<D, W><<<dim3(p.tile_groups - 1, 32 * W / kMergeRows), dim3(256), 0, st>>>(p);
    return hipGetLastError();
}
template <int D, int NG>
hipError_t tile_go(const PagedAttnParams &p, hipStream_t st) {
    return p.q_bf16 ? tile_go_as<D, NG, false>(p, st) : tile_go_as<D, NG, true>(p, st);
}
}  // namespace

int64_t paged_tile_plan(PagedAttnParams *p) {
    const int64_t rows = (int64_t)p->seqs.max_q * p->g;
    p->tile_groups = 0;
    if (rows <= kFewRows) return 0;
    p->few_rows = p->groups ? kFewRows : 0;
    // steps that there can be: a workgroup has four at least
    const int64_t steps = std::max<int64_t>(1, (((int64_t)p->seqs.width << (p->pool.log_tpp + 4)) + kStep - 1) / kStep);
    const int64_t items = (rows + 32 * kTileWaves - 1) / (32 * kTileWaves) * p->pool.heads * p->seqs.n_seqs;
    p->tile_groups = (int)std::max<int64_t>(1, std::min<int64_t>(kTileGroups, items * steps));
    return kTileSums + (int64_t)p->tile_groups * 2 * 32 * kTileWaves * (p->D + 4) * 4;
}

hipError_t paged_tile_launch(const PagedAttnParams &p0, hipStream_t st) {
    PagedAttnParams p = p0;
    p.sums = (int *)p.tile_part;
    p.tile_part += kTileSums / 4;
    if (p.D == 128) {
        if (p.ng == 4) return tile_go<128, 4>(p, st);
        if (p.ng == 2) return tile_go<128, 2>(p, st);
        return tile_go<128, 1>(p, st);
    }
    if (p.ng == 2) return tile_go<64, 2>(p, st);
    return tile_go<64, 1>(p, st);
}

hipError_t paged_importance_tile_launch(const PagedImportanceParams &p, hipStream_t st) {
    const dim3 grid((unsigned)((p.n_scores + kStep - 1) / kStep), p.seqs.n_seqs);
    auto go = [&](auto kern) {
        const int lds = 2 * 2 * kStep * 2 * p.D;
        if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        kern<<<grid, dim3(256), lds, st>>>(p);
    };
    if (p.D == 128) {
        if (p.ng == 4) go(paged_importance_tile_kernel<128, 4>);
        else if (p.ng == 2) go(paged_importance_tile_kernel<128, 2>);
        else go(paged_importance_tile_kernel<128, 1>);
    } else {
        if (p.ng == 2) go(paged_importance_tile_kernel<64, 2>);
        else go(paged_importance_tile_kernel<64, 1>);
    }
    return hipGetLastError();
}

}  // namespace akv
