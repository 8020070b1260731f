// Attention over the paged 4-bit cache, its merge, and the importance of cached tokens.
//
// The mathematics.  A key is c s + z with whole codes c and one float16 (s, z) per token and
// channel group, so q.k = sum over groups of s (q.(c - 7)) + (z + 7 s) (sum of q): the matrix cores
// take the codes themselves, and scale and zero enter once per score in float32.  The query's
// rows are scaled to a maximum in [2^13, 2^14), which leaves with the softmax scale.  Scores are
// thus exact to float32 rounding, whatever the cache's widths.  Values: o = sum of p (c s + z) is the
// product of the codes with p s plus sum of p z, one more MFMA row per channel group; p and p s enter
// as two float16 each, for bfloat16 outputs as one.  Both lie high in float16's range (kFewBias), so
// that light tokens keep their part beside one that has nearly all of a row's weight.  Softmax
// state: running maximum and sum per row in float32.
#include <algorithm>
#include <type_traits>

#include "akv_common.h"
#include "paged.h"
#include "paged_device.h"

namespace akv {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kImpTiles = 4;          // tiles of a wave's run in the importance
constexpr int kImpBlocks = 4;         // most runs of a wave in a decode step's
constexpr int kImpHeads = 3;          // most heads of a wave there
// LDS of one head's query operand of 16 rows, its groups' sums, factor and log-sum.
__host__ __device__ constexpr int paged_query_bytes(int D, int ng) { return 32 * D + 64 * (ng + 2); }
// The few-rows kernel holds p times 2^14, in (0, 2^14], and V scales over a power of two that they stay
// below (at kHighExp below twice it: the append's largest is 2^13): p times a scale keeps 11 bits down
// to 2^-28 of the largest, and something down to 2^-38 (less by what scales lie below 2^-12).  (With p in (0, 4] and scales as they are, a
// token of 0.999 of the weight and a value near 0 took 2e-3 to 1e-1 of an output with it, by the size
// of the values and the length of a wave's run.)
constexpr float kFewBias = 14.0f;
constexpr int kLowExp = -12, kHighExp = 12;  // of that power, which goes in steps of 2^4: 2^12 and 7 2^12 are float16
constexpr int kMaxGroups = 512;       // two workgroups a compute unit: what registers allow at head_dim 128

__device__ __forceinline__ float xmax(float x) {
    x = __builtin_fmaxf(x, __shfl_xor(x, 16));
    return __builtin_fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float xsum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
// Codes enter as c - 7: around zero the sums stay of the size of their result, and zeros are those of
// such codes, z + 7 s.  (The MFMA cuts terms off below its largest, always downwards, and holds
// subnormals at their exponent: codes of one sign left float16 outputs of 60000 tokens 6e-4 of
// their norm off, subnormal ones the log-sums 1.5e-6.)
constexpr int kMid = 7;
__device__ __forceinline__ h8 code_operand(const Nibbles &nb, uint32_t w) {
    const uint32_t v = w >> 8;
    return __builtin_bit_cast(h8, (u4){as_u32(nb.low<kMid>(w)), as_u32(nb.high<kMid>(w)), as_u32(nb.low<kMid>(v)), as_u32(nb.high<kMid>(v))});
}
__device__ __forceinline__ float lo_f(uint32_t w) { return (float)as_h2(w)[0]; }
__device__ __forceinline__ float hi_f(uint32_t w) { return (float)as_h2(w)[1]; }

// The query operand of 16 rows: lane (row col, quarter grp) holds channels 32 g + 8 grp ..
template <int D, int NG>
struct Query {
    h8 op[D / 32];
    float sum[NG];  // of the group's channels
    float kx;       // score -> log2 domain
};

template <int D>
__device__ __forceinline__ void load_row(u4 (&w)[D / 32], const unsigned char *row) {
    const int grp = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int g = 0; g < D / 32; ++g) w[g] = *(const u4 *)(row + (32 * g + 8 * grp) * 2);
}

// The row's maximum goes to [2^13, 2^14).
template <int D, int NG>
__device__ __forceinline__ void make_query(Query<D, NG> &Q, const u4 (&w)[D / 32], bool bf16, float scale_log2) {
    constexpr int NS = D / 32;
    int ex;  // top = f 2^ex, f in [1/2, 1)
    if (bf16) {
        float x[NS][8];
        float top = 0.0f;
#pragma unroll
        for (int g = 0; g < NS; ++g)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t v = w[g][i >> 1];
                x[g][i] = __builtin_bit_cast(float, i & 1 ? v & 0xffff0000u : v << 16);
                top = __builtin_fmaxf(top, __builtin_fabsf(x[g][i]));
            }
        top = xmax(top);
        ex = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 14;
#pragma unroll
        for (int g = 0; g < NS; ++g) {
            float y[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) y[n] = __builtin_ldexpf(x[g][n], 14 - ex);
            Q.op[g] = (h8){(_Float16)y[0], (_Float16)y[4], (_Float16)y[1], (_Float16)y[5],
                           (_Float16)y[2], (_Float16)y[6], (_Float16)y[3], (_Float16)y[7]};
        }
    } else {  // in float16 throughout: powers of two
        typedef uint16_t s2 __attribute__((ext_vector_type(2)));
        s2 most = {0, 0};
#pragma unroll
        for (int g = 0; g < NS; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                most = __builtin_elementwise_max(most, __builtin_bit_cast(s2, (uint32_t)w[g][i] & 0x7fff7fffu));
        const float top = xmax((float)__builtin_bit_cast(_Float16, most[0] > most[1] ? most[0] : most[1]));
        // at most 2^30, in two steps (float16's largest is 2^15): then every step of the input is a whole number
        ex = max(top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 14, -16);
        const int e1 = min(14 - ex, 15);
        const _Float16 a = (_Float16)__builtin_ldexpf(1.0f, e1), c = (_Float16)__builtin_ldexpf(1.0f, 14 - ex - e1);
#pragma unroll
        for (int g = 0; g < NS; ++g) {
            u4 y;
#pragma unroll
            for (int n = 0; n < 4; ++n) {  // channels n and n + 4
                const uint32_t at = (n & 1) ? 0x07060302u : 0x05040100u;
                const h2 v = as_h2(__builtin_amdgcn_perm((uint32_t)w[g][2 + (n >> 1)], (uint32_t)w[g][n >> 1], at));
                y[n] = as_u32(v * (h2){a, a} * (h2){c, c});
            }
            Q.op[g] = __builtin_bit_cast(h8, y);
        }
    }
    const h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        f4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < NS / NG; ++st) c = mfma_k32(ones, Q.op[g * (NS / NG) + st], c);
        Q.sum[g] = c[0];
    }
    Q.kx = __builtin_ldexpf(scale_log2, ex - 14);
}

// K meta dword d of a tile for tile_scores: float32 scales, then float32 zeros of the centred codes.
template <int NG>
__device__ __forceinline__ void put_k_meta(float *meta, int d, uint32_t w) {
    const float s = lo_f(w);
    meta[d] = s;
    meta[16 * NG + d] = __builtin_fmaf(s, (float)kMid, hi_f(w));
}
// Scores (of the scaled query) of tokens 4 grp + e of a tile for row col.  `meta`:
// what put_k_meta left of the tile.
template <int D, int NG>
__device__ __forceinline__ f4 tile_scores(const Query<D, NG> &Q, const Nibbles &nb, const uint32_t (&kc)[D / 32], const float *meta) {
    constexpr int NS = D / 32;
    const int grp = (threadIdx.x >> 4) & 3;
    float m[4 * NG], z[4 * NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const f4 w = ((const f4 *)meta)[grp * NG + i], y = ((const f4 *)meta)[4 * NG + grp * NG + i];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[4 * i + e] = w[e], z[4 * i + e] = y[e];
    }
    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        f4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < NS / NG; ++st) c = mfma_k32(code_operand(nb, kc[g * (NS / NG) + st]), Q.op[g * (NS / NG) + st], c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[e] = __builtin_fmaf(m[e * NG + g], c[e], s[e]);
            s[e] = __builtin_fmaf(z[e * NG + g], Q.sum[g], s[e]);
        }
    }
    return s;
}

// The work of a sequence, in units: 32 cached tokens of one head for one chunk of 16 rows.  An
// item (one head and chunk) counts kSetup units more than it has, the time until its first
// tiles are there: without them the runs of short sequences took twice as long as the others
// (a step of 24 sequences of 33 to 65536 tokens: 113 us without, 76 with).
constexpr int kSetup = 2;
struct SeqWork {
    SeqRows r;
    int rows, chunks, units, cost;  // rows = query tokens * g; units of one (head, chunk), and what it counts
};
__device__ __forceinline__ SeqWork seq_work(const PagedAttnParams &p, const SeqRows &r) {
    SeqWork w;
    w.r = r;
    w.rows = min(r.n, p.seqs.max_q) * p.g;
    w.chunks = w.rows <= kFewRows ? (w.rows + kRows - 1) / kRows : 0;  // more rows are paged_tile_kernel's
    w.units = max(1, (r.kv + (kUnitTok - 1)) / kUnitTok);
    w.cost = p.whole ? p.whole : w.units + kSetup;
    return w;
}
__device__ __forceinline__ int seq_total(const PagedAttnParams &p, const SeqWork &w) { return w.chunks * w.cost * p.pool.heads; }

// Where the sequences' units lie: pre[i] is the first unit of sequence i * per, pre[256] the
// total; up to 256 sequences their rows are kept too.
struct Scan {
    int pre[257];
    int wave_sum[kWaves];
    int begin[kThreads], n[kThreads], kv[kThreads], at[kThreads];
};
__device__ __forceinline__ SeqRows scanned_rows(const PagedAttnParams &p, const Scan &sc, int s) {
    return p.seqs.n_seqs <= kThreads ? SeqRows{sc.begin[s], sc.n[s], sc.kv[s], sc.at[s]} : seq_rows(p.seqs, s, p.pool.log_tpp + 4);
}
__device__ __forceinline__ void scan_seqs(const PagedAttnParams &p, Scan &sc, int per) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int mine = 0;
    for (int i = 0; i < per; ++i) {
        const int s = t * per + i;
        if (s < p.seqs.n_seqs) {
            const SeqRows r = seq_rows(p.seqs, s, p.pool.log_tpp + 4);
            mine += seq_total(p, seq_work(p, r));
            if (per == 1) sc.begin[t] = r.begin, sc.n[t] = r.n, sc.kv[t] = r.kv, sc.at[t] = r.at;
        }
    }
    int inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) sc.wave_sum[wave] = inc;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before += sc.wave_sum[w];
    sc.pre[t] = before + inc - mine;
    if (t == kThreads - 1) sc.pre[kThreads] = before + inc;
    __syncthreads();
}

__device__ __forceinline__ int share_of(int total, int groups) {  // units a wave takes
    const int waves = groups * kWaves;
    return max(1, (total + waves - 1) / waves);
}

// Row r of an item's chunk as (query token, head).
__device__ __forceinline__ void write_row(const PagedAttnParams &p, const SeqRows &r, int h, int row, int ch, const float (&o)[8],
                                          float m, float l) {
    const int64_t t = r.begin + row / p.g;
    const int head = h * p.g + row % p.g;
    const float inv = row_inverse(l);
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = to_pair(p.q_bf16, o[2 * i] * inv, o[2 * i + 1] * inv);
    *(u4 *)((unsigned char *)p.out + ((t * p.Hq + head) * p.D + ch) * 2) = w;
    if (p.lse && ch == 0) p.lse[t * p.Hq + head] = row_lse(m, l, kFewBias);
}

}  // namespace

// Single tokens and a few drafted ones.  Bound by issue and, nearly as much, by the cache's bytes:
// 325 vector instructions and 17 MFMAs for 32 tokens of a head (415 and 27 where p is two
// float16), two waves a SIMD.  24 sequences of 33 to 65536 tokens, 32 heads over 8, bfloat16 (299
// MB): 73 us, 4.1 TB/s, and 5 us of merge; 20 rows of nine sequences of 1001 to 9001 tokens,
// float16: 22.5 us and 5.2 us; one row of 517 tokens, whose time
// is the chain of loads from lengths to tiles: 7.4 us and 3.4 us.
//
// The units of all sequences, heads and chunks form one list, cut into equal runs, one a wave:
// every wave has the same work whatever the lengths.  A run that covers an item (all units of
// a sequence, head and chunk) writes its rows; states of items that end or begin inside a
// workgroup's runs are joined through LDS, items that several workgroups share leave partial
// states for paged_merge_kernel.  A wave loads its tiles straight to registers, two units
// ahead; the meta of a tile goes through LDS, where each lane reads its tokens'.
template <int D, int NG, bool TWO>
__global__ __launch_bounds__(kThreads, 2) void paged_decode_kernel(const PagedAttnParams p) {
    constexpr int NS = D / 32, NB = D / 16, TB = paged_tile_bytes(D, NG), EROW = D + 4;
    constexpr int MW = NG == 4 ? 2 : 1;          // meta dwords a lane loads of a tile
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Scan sc;
    __shared__ int e_seq[2 * kWaves], e_item[2 * kWaves], e_flags[2 * kWaves];  // flags: 1 used, 2 starts, 4 ends
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int k_at = (4 * col + grp) * (D / 8);  // K codes of token col, quarter grp
    float *entries = (float *)smem;
    uint32_t *meta = (uint32_t *)(smem + 2 * kWaves * p.rows * EROW * 4) + wave * 2 * 48 * NG;
    if (lane < 2) e_flags[2 * wave + lane] = 0;
    Nibbles nb;
    nb.init();

    const int per = (p.seqs.n_seqs + kThreads - 1) / kThreads;
    scan_seqs(p, sc, per);
    const int total = __builtin_amdgcn_readfirstlane(sc.pre[kThreads]);
    const int share = p.whole ? p.whole / kWaves : share_of(total, p.groups);
    if (blockIdx.x == 0 && !p.whole) {  // for the merge
        p.sums[threadIdx.x] = sc.pre[threadIdx.x];
        if (threadIdx.x == 0) p.sums[kThreads] = total;
    }
    int x = (int)min((int64_t)(blockIdx.x * kWaves + wave) * share, (int64_t)total);
    const int x_end = min(x + share, total);

    // the sequence of unit x
    int s = 0, off = 0;
    SeqWork w{};
    if (x < x_end) {
        int k = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) k += __builtin_popcountll(__builtin_amdgcn_ballot_w64(sc.pre[64 * i + lane] <= x));
        s = (k - 1) * per;
        off = x - __builtin_amdgcn_readfirstlane(sc.pre[k - 1]);
        for (;;) {
            w = seq_work(p, wave_uniform(scanned_rows(p, sc, s)));
            const int n = seq_total(p, w);
            if (off < n) break;
            off -= n;
            ++s;
        }
    }
    while (x < x_end) {
        const int item = off / w.cost, c0 = off - item * w.cost;
        const int c1 = min(w.cost, c0 + (x_end - x));
        const int j0 = max(0, c0 - kSetup), j1 = max(0, c1 - kSetup);
        x += c1 - c0;
        off += c1 - c0;
        if (j1 == 0) break;  // no unit of the item is in the run, and the run ends
        const int h = item / w.chunks, row0 = (item - h * w.chunks) * kRows;
        const int rows = min(kRows, w.rows - row0);

        const int row = row0 + min(col, rows - 1);
        const int qt = row / p.g;
        const int kv = w.r.kv;
        const int see = w.r.sees(p.causal, qt);
        const int see_all = w.r.sees(p.causal, row0 / p.g);
        const int see_any = w.r.sees(p.causal, (row0 + rows - 1) / p.g);
        u4 qw[NS];
        load_row<D>(qw, p.q + (w.r.begin + qt) * p.q_t + (h * p.g + row % p.g) * p.q_h);

        const int32_t *table = p.seqs.table + s * p.seqs.table_stride;
        const int jn = min(j1, (see_any + kUnitTok - 1) / kUnitTok);
        const int log_tpp = p.pool.log_tpp;
        int pb = (2 * j0) >> log_tpp;
        int pid = pb + lane < p.seqs.width ? table[pb + lane] : -1;
        asm volatile("" : "+v"(pid));

        struct Unit {
            uint32_t kc[2][NS], vc[2][NS], m[2][MW];
            int nv[2];  // tokens of the tile that are there
        } U[2];
        auto load = [&](Unit &u, int j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = 2 * j + i;
                const int pi = t >> log_tpp;
                if (pi - pb >= 64) {
                    pb = pi;
                    pid = pb + lane < p.seqs.width ? table[pb + lane] : -1;
                    asm volatile("" : "+v"(pid));  // waited for here: not by every unit, behind its tiles' loads
                }
                uint32_t page = (uint32_t)__builtin_amdgcn_readlane(pid, pi - pb);
                const int left = kv - 16 * t;
                u.nv[i] = page < p.pool.n_pages ? min(left, 16) : 0;
                if (page >= p.pool.n_pages) page = 0;  // read, and masked
                const unsigned char *tile = p.pool.base + (int64_t)page * p.pool.page_bytes +
                                            (int64_t)((h << log_tpp) + (t & ((1 << log_tpp) - 1))) * TB;
                if constexpr (D == 128) {
                    const u4 a = *(const u4 *)(tile + k_at), b = *(const u4 *)(tile + 8 * D + lane * 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) u.kc[i][e] = a[e], u.vc[i][e] = b[e];
                } else {
                    const u2 a = *(const u2 *)(tile + k_at), b = *(const u2 *)(tile + 8 * D + lane * 8);
#pragma unroll
                    for (int e = 0; e < 2; ++e) u.kc[i][e] = a[e], u.vc[i][e] = b[e];
                }
                if constexpr (MW == 2) {
                    const u2 a = *(const u2 *)(tile + 16 * D + lane * 8);
                    u.m[i][0] = a[0], u.m[i][1] = a[1];
                } else {
                    u.m[i][0] = *(const uint32_t *)(tile + 16 * D + (lane & (32 * NG - 1)) * 4);
                }
            }
        };

        float mx = kMinMax, l = 0.0f;
        uint32_t poisoned = 0;  // groups of channels in which the row sees a value that is not finite
        f4 acc[NB], accz = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = (f4){0.f, 0.f, 0.f, 0.f};
        // V scales enter over 2^vexp, which they stay below, and acc holds sums over it: raised like the
        // running maximum, in steps of 2^4, so that caches of one kind of values raise it once
        typedef uint16_t s2 __attribute__((ext_vector_type(2)));
        constexpr uint64_t kScaleLanes = NG == 1 ? 0x00ff000000ff0000u : 0x0000ffff00000000u;  // whose meta is V scales
        int vexp = kLowExp;
        h2 down = {1.0f, 1.0f};  // 2^-vexp in those lanes
        if (kScaleLanes >> lane & 1) down = (h2){(_Float16)0x1p12f, (_Float16)0x1p12f};

        auto work = [&](const Query<D, NG> &Q, Unit &u, int j, auto is_clean) {
            constexpr bool clean = decltype(is_clean)::value;
            if constexpr (!clean) {  // V meta of slots without a token: whatever is there becomes 0
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < MW; ++q) {
                        const int d = (lane & (32 * NG / MW - 1)) * MW + q - 16 * NG;
                        const int tok = ((d & (8 * NG - 1)) / (2 * NG)) * 4 + (d & 1) * 2;
                        const uint32_t keep = (tok < u.nv[i] ? 0xffffu : 0u) | (tok + 1 < u.nv[i] ? 0xffff0000u : 0u);
                        // values that are not finite would reach rows that do not see them as 0 * NaN:
                        // they become 0 too, and the rows that see them NaN in the end
                        const uint32_t bad = d >= 0 ? not_finite(u.m[i][q]) & keep : 0u;
                        if (d >= 0) u.m[i][q] &= keep & ~bad;
                        const int group = (d >> 1) & (NG - 1);
                        for (uint64_t left = __builtin_amdgcn_ballot_w64(bad != 0); left; left &= left - 1) {
                            const int from = __builtin_ctzll(left);
                            const int at = kUnitTok * j + 16 * i + __builtin_amdgcn_readlane(tok, from);
                            const int of = __builtin_amdgcn_readlane(group, from);
                            const uint32_t what = __builtin_amdgcn_readlane(bad, from);
                            if ((at < see && (what & 0xffffu)) || (at + 1 < see && what >> 16)) poisoned |= 1u << of;
                        }
                    }
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // K scales and zeros as float32, then V scales over 2^vexp and V zeros as they are
                uint32_t *m = meta + i * 48 * NG;
#pragma unroll
                for (int q = 0; q < MW; ++q) {
                    const int d = (lane & (32 * NG / MW - 1)) * MW + q;
                    const uint32_t w = u.m[i][q];
                    const float ks = lo_f(w), kz = __builtin_fmaf(ks, (float)kMid, hi_f(w));
                    m[16 * NG + d] = d < 16 * NG ? __builtin_bit_cast(uint32_t, kz) : as_u32(as_h2(w) * down);
                    if (d < 16 * NG) m[d] = __builtin_bit_cast(uint32_t, ks);
                }
            }
            __builtin_amdgcn_wave_barrier();
            f4 sc[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sc[i] = tile_scores<D, NG>(Q, nb, u.kc[i], (const float *)meta + i * 48 * NG) * Q.kx;
                if constexpr (!clean)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int in = 4 * grp + e;
                        if (kUnitTok * j + 16 * i + in >= see || in >= u.nv[i]) sc[i][e] = -INFINITY;
                    }
            }
            float t = sc[0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) t = __builtin_fmaxf(t, sc[e >> 2][e & 3]);
            s2 most = __builtin_elementwise_max(__builtin_bit_cast(s2, u.m[0][0]), __builtin_bit_cast(s2, u.m[1][0]));
            if constexpr (MW == 2)
                most = __builtin_elementwise_max(most, __builtin_elementwise_max(__builtin_bit_cast(s2, u.m[0][MW - 1]), __builtin_bit_cast(s2, u.m[1][MW - 1])));
            const uint16_t below = (uint16_t)((vexp < kHighExp ? (vexp + 15) << 10 : 0x7c00) - 1);  // the largest float16 below 2^vexp
            const uint64_t over = kScaleLanes & __builtin_amdgcn_ballot_w64(
                __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(most, (s2){below, below})) != 0);
            if (__builtin_amdgcn_ballot_w64(t + (kFewBias - mx) > kFewBias) | over) {
                float to_new = 1.0f;  // from the old power to the new one
                if (over) {
                    s2 fin = {0, 0};  // the scales, without those that are not finite
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int q = 0; q < MW; ++q)
                            fin = __builtin_elementwise_max(fin, __builtin_bit_cast(s2, u.m[i][q] & ~not_finite(u.m[i][q]) & 0x7fff7fffu));
                    const int top = max(fin[0], fin[1]), was = vexp;
                    while (vexp < kHighExp && __builtin_amdgcn_ballot_w64(top >= (vexp + 15) << 10) & kScaleLanes) vexp += 4;
                    if (vexp != was) {
                        to_new = __builtin_ldexpf(1.0f, was - vexp);
                        const _Float16 x = (_Float16)__builtin_ldexpf(1.0f, -vexp);
                        if (kScaleLanes >> lane & 1) {
                            down = (h2){x, x};
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int q = 0; q < MW; ++q)
                                    meta[i * 48 * NG + 16 * NG + (lane & (32 * NG / MW - 1)) * MW + q] = as_u32(as_h2(u.m[i][q]) * down);
                        }
                        __builtin_amdgcn_wave_barrier();
                    }
                }
                const float most_t = xmax(t);
                const float mn = most_t > mx ? running_max(most_t, 1.0f, kFewBias) : mx;
                const float alpha = __builtin_amdgcn_exp2f(mx - mn);
                l *= alpha;
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] *= alpha * to_new;
                accz *= alpha;
                mx = mn;
            }
            const float bias = kFewBias - mx;
            float pr[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) pr[e] = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] + bias);
            l += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
            // float16 outputs: p, and p s below, as two float16 that add up to it: one alone would cost
            // them half a step (measured 3.5e-4 of the output's norm; 2.1e-4 is its own rounding).
            // Beside bfloat16's own 1.7e-3 one is as good (2^-12 of each weight, an eighth of its half step).
            h2 ph[4], pl[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                ph[q] = (h2){(_Float16)pr[2 * q], (_Float16)pr[2 * q + 1]};
                if constexpr (TWO) pl[q] = (h2){(_Float16)(pr[2 * q] - (float)ph[q][0]), (_Float16)(pr[2 * q + 1] - (float)ph[q][1])};
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                u4 pw, rw;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const u2 sv = *(const u2 *)(meta + i * 48 * NG + 32 * NG + (grp * NG + g) * 2);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const h2 sc2 = as_h2(sv[q]), t2 = ph[2 * i + q] * sc2;
                        pw[2 * i + q] = as_u32(t2);
                        if constexpr (TWO)
                            rw[2 * i + q] = as_u32(__builtin_elementwise_fma(pl[2 * i + q], sc2, __builtin_elementwise_fma(ph[2 * i + q], sc2, -t2)));
                    }
                }
                // the group's blocks of 16 channels: block 4 h + 2 l + b is nibble 2 l + b of half h
#pragma unroll
                for (int b = g * (NB / NG); b < (g + 1) * (NB / NG); ++b) {
                    const int h4 = b >> 2, n = b & 3;
                    u4 a;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t v = u.vc[q >> 1][(q & 1) * (NB / 4) + h4];
                        const uint32_t x = n >= 2 ? v >> 8 : v;
                        a[q] = as_u32(n & 1 ? nb.high<kMid>(x) : nb.low<kMid>(x));
                    }
                    acc[b] = mfma_k32(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, pw), acc[b]);
                    if constexpr (TWO) acc[b] = mfma_k32(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, rw), acc[b]);
                }
            }
            // row g of the operand: the tokens' zeros of group g, z + 7 s (two float16, or one as p is)
            u4 za = {0u, 0u, 0u, 0u}, zl = {0u, 0u, 0u, 0u};
            if (col < NG) {
                const uint32_t *at = meta + 32 * NG + (grp * NG + col) * 2;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const u2 zw = *(const u2 *)(at + i * 48 * NG + 8 * NG), sw = *(const u2 *)(at + i * 48 * NG);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if constexpr (TWO) {
                            const float mid = __builtin_ldexpf((float)kMid, vexp);
                            const float x = __builtin_fmaf(lo_f(sw[q]), mid, lo_f(zw[q])), y = __builtin_fmaf(hi_f(sw[q]), mid, hi_f(zw[q]));
                            const h2 h = {(_Float16)x, (_Float16)y};
                            za[2 * i + q] = as_u32(h);
                            zl[2 * i + q] = as_u32((h2){(_Float16)(x - (float)h[0]), (_Float16)(y - (float)h[1])});
                        } else {
                            const _Float16 mid = (_Float16)__builtin_ldexpf((float)kMid, vexp);
                            za[2 * i + q] = as_u32(__builtin_elementwise_fma(as_h2(sw[q]), (h2){mid, mid}, as_h2(zw[q])));
                        }
                    }
                }
            }
            const h8 p_hi = __builtin_bit_cast(h8, (u4){as_u32(ph[0]), as_u32(ph[1]), as_u32(ph[2]), as_u32(ph[3])});
            accz = mfma_k32(__builtin_bit_cast(h8, za), p_hi, accz);
            if constexpr (TWO) {
                accz = mfma_k32(__builtin_bit_cast(h8, zl), p_hi, accz);
                accz = mfma_k32(__builtin_bit_cast(h8, za), __builtin_bit_cast(h8, (u4){as_u32(pl[0]), as_u32(pl[1]), as_u32(pl[2]), as_u32(pl[3])}), accz);
            }
        };

        auto consume = [&](const Query<D, NG> &Q, Unit &u, int j) {
            if (kUnitTok * (j + 1) <= see_all && u.nv[0] == 16 && u.nv[1] == 16) work(Q, u, j, std::true_type{});
            else work(Q, u, j, std::false_type{});
        };

        // Both buffers are always loaded (the last unit again at the end), so that a unit waits
        // for its own loads and never for those behind it.
        if (j0 < jn) {
            load(U[0], j0);
            load(U[1], min(j0 + 1, jn - 1));
        }
        Query<D, NG> Q;
        make_query<D, NG>(Q, qw, p.q_bf16, p.scale_log2);
        int j = j0;
        for (; j + 1 < jn; j += 2) {
            consume(Q, U[0], j);
            load(U[0], min(j + 2, jn - 1));
            consume(Q, U[1], j + 1);
            load(U[1], min(j + 3, jn - 1));
        }
        if (j < jn) consume(Q, U[0], j);

        // the segment's state in true units
        const float scale = __builtin_ldexpf(1.0f, vexp);
        l = xsum(l);
        float z[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float v = __shfl(accz[g], col);
            z[g] = poisoned >> g & 1 ? NAN : v;
        }
        const bool starts = j0 == 0, ends = c1 == w.cost;
        const int slot = 2 * wave + (ends ? 0 : 1);
        float *er = entries + (slot * p.rows + col) * EROW;
#pragma unroll
        for (int g = 0; g < NS; ++g) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[2 * i] = __builtin_fmaf(acc[2 * g][i], scale, z[g * NG / NS]);
                o[2 * i + 1] = __builtin_fmaf(acc[2 * g + 1][i], scale, z[g * NG / NS]);
            }
            const int ch = 32 * g + 8 * grp;
            if (col < rows) {
                if (starts && ends) {
                    write_row(p, w.r, h, row, ch, o, mx, l);
                } else {
                    *(f4 *)(er + ch) = (f4){o[0], o[1], o[2], o[3]};
                    *(f4 *)(er + ch + 4) = (f4){o[4], o[5], o[6], o[7]};
                }
            }
        }
        if (!(starts && ends)) {
            if (grp == 0 && col < rows) er[D] = mx, er[D + 1] = l;
            if (lane == 0) {
                e_seq[slot] = s;
                e_item[slot] = item;
                e_flags[slot] = 1 | (starts ? 2 : 0) | (ends ? 4 : 0);
            }
        }

        if (x < x_end && off == seq_total(p, w)) {
            do w = seq_work(p, wave_uniform(scanned_rows(p, sc, ++s)));
            while (w.chunks == 0);
            off = 0;
        }
    }

    // join what the runs left: entries of one item are neighbours, the last of them ends the
    // item or the workgroup's run
    __syncthreads();
    const int flags = lane < 2 * kWaves ? e_flags[lane] : 0;
    uint32_t used = (uint32_t)__builtin_amdgcn_ballot_w64(flags & 1);
    const uint32_t starts = (uint32_t)__builtin_amdgcn_ballot_w64(flags & 2), ends = (uint32_t)__builtin_amdgcn_ballot_w64(flags & 4);
    constexpr int CH = D / 16;
    const int row_t = threadIdx.x >> 4, ch = (threadIdx.x & 15) * CH;
    if (row_t >= p.rows) return;
    while (used) {
        const uint32_t first = used & -used;
        float o[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) o[i] = 0.f;
        float M = kMinMax, L = 0.f;
        int e;
        do {
            e = __builtin_ctz(used);
            used &= used - 1;
            const float *er = entries + (e * p.rows + row_t) * EROW;
            const f2 ml = *(const f2 *)(er + D);
            const float mn = __builtin_fmaxf(M, ml[0]);
            const float a = __builtin_amdgcn_exp2f(M - mn), b = __builtin_amdgcn_exp2f(ml[0] - mn);
#pragma unroll
            for (int i = 0; i < CH; ++i) o[i] = __builtin_fmaf(er[ch + i], b, o[i] * a);
            L = __builtin_fmaf(ml[1], b, L * a);
            M = mn;
        } while (!(ends >> e & 1) && used);
        const bool began = starts & first;
        if (began && (ends >> e & 1)) {
            const SeqWork sw = seq_work(p, scanned_rows(p, sc, e_seq[e]));
            const int it = e_item[e], h = it / sw.chunks, row = (it - h * sw.chunks) * kRows + row_t;
            if (row < sw.rows) {
                float o8[8];
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    o8[i] = o[i];
                    if constexpr (CH == 4) o8[4 + i] = __shfl_down(o[i], 1);  // pairs of threads write together
                }
                if (CH == 8 || !(threadIdx.x & 1)) write_row(p, sw.r, h, row, ch, o8, M, L);
            }
        } else {
            float *pr = p.part + ((int64_t)(2 * blockIdx.x + (began ? 1 : 0)) * p.rows + row_t) * EROW;
#pragma unroll
            for (int i = 0; i < CH; i += 4) *(f4 *)(pr + ch + i) = (f4){o[i], o[i + 1], o[i + 2], o[i + 3]};
            if (ch == 0) *(f2 *)(pr + D) = (f2){M, L};
        }
    }
}

// Items that several workgroups share: one workgroup an item.  Sixteen threads a row; where an
// item has fewer than 16 rows the others take partial states of their own, joined through LDS
// in a fixed order.  Bound by latency: the states of an item are loaded at once, eight a thread
// (3.4 us for one sequence, 5 us for 24).
template <int D>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedAttnParams p) {
    constexpr int EROW = D + 4, CH = D / 16, B = 8;
    __shared__ float so[kThreads][CH + 1], sm[16], sl[16];
    const int per = (p.seqs.n_seqs + kThreads - 1) / kThreads;
    const int s = blockIdx.y, k = s / per;
    int at = p.sums[k];
    const int share = share_of(p.sums[kThreads], p.groups) * kWaves;  // units a workgroup has
    const SeqWork w = seq_work(p, seq_rows(p.seqs, s, p.pool.log_tpp + 4));
    for (int i = k * per; i < s; ++i) at += seq_total(p, seq_work(p, seq_rows(p.seqs, i, p.pool.log_tpp + 4)));
    int rp = 1;
    while (rp < p.rows) rp <<= 1;
    const int t16 = threadIdx.x >> 4, row_t = t16 & (rp - 1), sp = t16 / rp, ps = 16 / rp, ch = (threadIdx.x & 15) * CH;
    for (int item = blockIdx.x; item < w.chunks * p.pool.heads; item += gridDim.x) {
        const int first = at + item * w.cost;
        const int g0 = (first + kSetup) / share, g1 = (first + w.cost - 1) / share;
        if (g0 == g1) continue;
        const int h = item / w.chunks, row = (item - h * w.chunks) * kRows + row_t;
        const bool live = row_t < p.rows && row < w.rows;
        float o[CH];
        float M = kMinMax, L = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) o[i] = 0.f;
        for (int g = g0 + sp; g <= g1 && live; g += B * ps) {
            f4 v[B][CH / 4];
            f2 ml[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int gi = min(g + i * ps, g1);
                const float *pr = p.part + ((int64_t)(2 * gi + (gi == g0 ? 1 : 0)) * p.rows + row_t) * EROW;
#pragma unroll
                for (int c = 0; c < CH / 4; ++c) v[i][c] = ((const f4 *)(pr + ch))[c];
                ml[i] = *(const f2 *)(pr + D);
            }
            float mn = M;
#pragma unroll
            for (int i = 0; i < B; ++i) mn = __builtin_fmaxf(mn, ml[i][0]);
            const float a = __builtin_amdgcn_exp2f(M - mn);
            L *= a;
#pragma unroll
            for (int c = 0; c < CH; ++c) o[c] *= a;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const float b = g + i * ps <= g1 ? __builtin_amdgcn_exp2f(ml[i][0] - mn) : 0.f;
                L = __builtin_fmaf(ml[i][1], b, L);
#pragma unroll
                for (int c = 0; c < CH; ++c) o[c] = __builtin_fmaf(v[i][c >> 2][c & 3], b, o[c]);
            }
            M = mn;
        }
        if (ps > 1) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < CH; ++c) so[threadIdx.x][c] = o[c];
            if (ch == 0) sm[t16] = M, sl[t16] = L;
            __syncthreads();
            if (sp == 0)
                for (int q = 1; q < ps; ++q) {
                    const float m = sm[q * rp + row_t], mn = __builtin_fmaxf(M, m);
                    const float a = __builtin_amdgcn_exp2f(M - mn), b = __builtin_amdgcn_exp2f(m - mn);
                    L = __builtin_fmaf(sl[q * rp + row_t], b, L * a);
#pragma unroll
                    for (int c = 0; c < CH; ++c) o[c] = __builtin_fmaf(so[threadIdx.x + 16 * q * rp][c], b, o[c] * a);
                    M = mn;
                }
        }
        if (sp != 0 || !live) continue;
        float o8[8];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            o8[i] = o[i];
            if constexpr (CH == 4) o8[4 + i] = __shfl_down(o[i], 1);
        }
        if (CH == 8 || !(threadIdx.x & 1)) write_row(p, w.r, h, row, ch, o8, M, L);
    }
}

// The importance.  A wave takes 64 tokens of a sequence and some of its heads (the heads are
// split over the waves of a workgroup, at most four ways), the next head's keys in flight; the
// sums over rows stay in registers, lane by lane of a row, until the end, and are joined in a
// fixed order.  Bound by latency and issue (360 vector instructions for 16 rows and 64 tokens of a
// head), the K half of the cache behind them: one row of two sequences of 12000 tokens, 32 heads over
// 8: 10.4 us; 32 rows of two sequences of 8191 to 16384 tokens: 32 us.  (Queries of the next rows in flight, or three waves a SIMD without the
// second buffer, were no faster: 34 and 41 us.)
template <int D, int NG>
__global__ __launch_bounds__(kThreads, 2) void paged_importance_kernel(const PagedImportanceParams p) {
    constexpr int NS = D / 32, TB = paged_tile_bytes(D, NG), NT = kImpTiles, MT = 16 * NG;
    constexpr uint32_t ALL = (1u << NT) - 1;
    __shared__ __align__(16) float smeta[kWaves][NT * 2 * MT];
    __shared__ float sums[kWaves][NT * 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int k_at = (4 * col + grp) * (D / 8);  // K codes of token col, quarter grp
    const int s = blockIdx.y, hs = p.head_split, h0 = wave & (hs - 1);
    const int blocks = kWaves / hs;              // runs of NT tiles a workgroup has
    const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_tpp + 4));
    const int64_t tok0 = ((int64_t)blockIdx.x * blocks + wave / hs) * (NT * 16);
    const int n = min(r.n, p.seqs.max_q);
    const int64_t kv = n > 0 ? min((int64_t)r.kv, p.n_scores) : 0;  // tokens whose score changes
    const int first = p.q_window > 0 && p.q_window < n ? n - p.q_window : 0;
    const int rows = (n - first) * p.g;
    float sum[NT * 4];
#pragma unroll
    for (int i = 0; i < NT * 4; ++i) sum[i] = 0.f;
    float *meta = smeta[wave];
    Nibbles nb;
    nb.init();
    if (tok0 < kv) {
        const int log_tpp = p.pool.log_tpp, in_page = (1 << log_tpp) - 1;
        const int32_t *table = p.seqs.table + s * p.seqs.table_stride;
        const int t0 = (int)(tok0 >> 4);
        // lane i < NT: the page of tile i; tiles past the end or outside the pool read page 0 and count nothing
        const bool there = lane < NT && 16 * (int64_t)(t0 + lane) < r.kv;
        uint32_t page = there ? (uint32_t)table[(t0 + lane) >> log_tpp] : 0xffffffffu;
        const uint32_t have = (uint32_t)__builtin_amdgcn_ballot_w64(page < p.pool.n_pages);
        if (page >= p.pool.n_pages) page = 0;
        struct Keys {
            uint32_t kc[NT][NS], m[NT];
        } K[2];
        auto load = [&](Keys &k, int h) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const unsigned char *tile = p.pool.base + (int64_t)(uint32_t)__builtin_amdgcn_readlane(page, i) * p.pool.page_bytes +
                                            (int64_t)((h << log_tpp) + ((t0 + i) & in_page)) * TB;
                if constexpr (D == 128) {
                    const u4 a = *(const u4 *)(tile + k_at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) k.kc[i][e] = a[e];
                } else {
                    const u2 a = *(const u2 *)(tile + k_at);
                    k.kc[i][0] = a[0], k.kc[i][1] = a[1];
                }
                k.m[i] = *(const uint32_t *)(tile + 16 * D + (lane & (MT - 1)) * 4);
            }
        };
        auto consume = [&](Keys &k, int h) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < NT; ++i) put_k_meta<NG>(meta + i * 2 * MT, lane & (MT - 1), k.m[i]);
            __builtin_amdgcn_wave_barrier();
            for (int row0 = 0; row0 < rows; row0 += kRows) {
                const bool live = row0 + col < rows;
                const int row = live ? row0 + col : rows - 1;
                const int qt = first + row / p.g;
                const int64_t t = r.begin + qt;
                const int head = h * p.g + row % p.g;
                u4 qw[NS];
                load_row<D>(qw, p.q + t * p.q_t + head * p.q_h);
                const float lse2 = p.lse[t * p.Hq + head] * 1.4426950408889634f;
                Query<D, NG> Q;
                make_query<D, NG>(Q, qw, p.q_bf16, p.scale_log2);
                const float bias = live ? -lse2 : -INFINITY;
                const int see = r.sees(p.causal, qt);
                const bool clean = have == ALL && __builtin_amdgcn_ballot_w64(tok0 + NT * 16 <= see) == ~0ull;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const f4 x = tile_scores<D, NG>(Q, nb, k.kc[i], meta + i * 2 * MT);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], Q.kx, bias));
                        if (!clean) pr = tok0 + 16 * i + 4 * grp + e < see && (have >> i & 1) && live ? pr : 0.f;
                        sum[4 * i + e] += pr;
                    }
                    __builtin_amdgcn_sched_barrier(0);  // one tile's meta in registers at a time
                }
            }
        };
        const int last = h0 + (p.pool.heads - 1 - h0) / hs * hs;
        load(K[0], h0);
        load(K[1], min(h0 + hs, last));
        int h = h0;
        for (; h + hs <= last; h += 2 * hs) {
            consume(K[0], h);
            load(K[0], min(h + 2 * hs, last));
            consume(K[1], h + hs);
            load(K[1], min(h + 3 * hs, last));
        }
        if (h <= last) consume(K[0], h);
    }
    // over the 16 rows: each step halves what a lane holds; lane col ends with its NT / 4 sums of the quad's
#pragma unroll
    for (int d = 8, c = NT * 2; d > 0; d >>= 1, c >>= 1)
#pragma unroll
        for (int i = 0; i < c; ++i) {
            float a = sum[i], b = sum[i + c];
            asm("" : "+v"(a), "+v"(b));  // or a choice of values becomes one of indexes, 16 selects long
            sum[i] = (col & d ? b : a) + __shfl_xor(col & d ? a : b, d);
        }
#pragma unroll
    for (int i = 0; i < NT / 4; ++i) {
        const int v = NT / 4 * col + i;  // tile v / 4, token 4 grp + v % 4 of it
        sums[wave][16 * (v >> 2) + 4 * grp + (v & 3)] = sum[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < blocks * NT * 16; i += kThreads) {
        const int64_t j = (int64_t)blockIdx.x * blocks * (NT * 16) + i;
        if (j >= p.n_scores) break;
        const int b = i / (NT * 16);
        const float *old = p.scores + s * p.score_stride + j;
        float *out = p.out + s * p.out_stride + j;
        if (j < kv) {
            float v = 0.f;
            for (int q = 0; q < hs; ++q) v += sums[b * hs + q][i & (NT * 16 - 1)];
            *out = __builtin_fmaf(*old, p.decay, v / (float)p.Hq);
        } else if (out != old) {
            *out = *old;
        }
    }
}

// The importance of a large decode step: at most 16 rows a head, few heads.  As above, but a wave makes
// its heads' query operands once, in LDS, and takes p.blocks runs of 64 tokens, whose pages it looks up
// at once, the next (run, head)'s keys in flight.  Bound by issue and memory, nearly even: one row of 24
// sequences of 16000 tokens, 32 heads over 8 (246 MB of keys): 69 us, 3.6 TB/s, where the kernel above
// took 103.  Lengths far apart keep less of the card busy (eight of 1000 to 31744: 13.0 against 12).
template <int D, int NG>
__global__ __launch_bounds__(kThreads, 2) void paged_importance_step_kernel(const PagedImportanceParams p) {
    constexpr int NS = D / 32, TB = paged_tile_bytes(D, NG), NT = kImpTiles, MT = 16 * NG;
    constexpr uint32_t ALL = (1u << NT) - 1;
    __shared__ __align__(16) float smeta[kWaves][NT * 2 * MT];
    __shared__ float sums[kWaves][kImpBlocks * NT * 16];
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int k_at = (4 * col + grp) * (D / 8);  // K codes of token col, quarter grp
    const int s = blockIdx.y, hs = p.head_split, h0 = wave & (hs - 1), nh = (p.pool.heads - 1 - h0) / hs + 1;
    const int runs = kWaves / hs, run_tok = p.blocks * NT * 16;
    const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_tpp + 4));
    const int64_t tok0 = ((int64_t)blockIdx.x * runs + wave / hs) * run_tok;
    const int n = min(r.n, p.seqs.max_q);
    const int64_t kv = n > 0 ? min((int64_t)r.kv, p.n_scores) : 0;  // tokens whose score changes
    if (tok0 < kv) {
        const int first = p.q_window > 0 && p.q_window < n ? n - p.q_window : 0;
        const int rows = (n - first) * p.g;
        const bool live = col < rows;
        const int row = live ? col : rows - 1, qt = first + row / p.g;
        const int see = live ? r.sees(p.causal, qt) : 0;
        const int log_tpp = p.pool.log_tpp, in_page = (1 << log_tpp) - 1;
        const int32_t *table = p.seqs.table + s * p.seqs.table_stride;
        const int t0 = (int)(tok0 >> 4);
        // lane i: the page of tile i; tiles past the end or outside the pool read page 0 and count nothing
        const bool there = lane < p.blocks * NT && 16 * (int64_t)(t0 + lane) < r.kv;
        uint32_t page = there ? (uint32_t)table[(t0 + lane) >> log_tpp] : 0xffffffffu;
        const uint32_t have = (uint32_t)__builtin_amdgcn_ballot_w64(page < p.pool.n_pages);
        if (page >= p.pool.n_pages) page = 0;
        struct Keys {
            uint32_t kc[NT][NS], m[NT];
        } K[2];
        auto load = [&](Keys &k, int b, int h) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const unsigned char *tile = p.pool.base + (int64_t)(uint32_t)__builtin_amdgcn_readlane(page, NT * b + i) * p.pool.page_bytes +
                                            (int64_t)((h << log_tpp) + ((t0 + NT * b + i) & in_page)) * TB;
                if constexpr (D == 128) {
                    const u4 a = *(const u4 *)(tile + k_at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) k.kc[i][e] = a[e];
                } else {
                    const u2 a = *(const u2 *)(tile + k_at);
                    k.kc[i][0] = a[0], k.kc[i][1] = a[1];
                }
                k.m[i] = *(const uint32_t *)(tile + 16 * D + (lane & (MT - 1)) * 4);
            }
        };
        const int blocks = (int)min((int64_t)p.blocks, (kv - tok0 + NT * 16 - 1) / (NT * 16)), last = blocks * nh - 1;
        // head k's operand: [NS][64 lanes] of 16 bytes, then [NG + 2][16 rows]: sums, factor, -lse
        unsigned char *qs = smem + wave * p.head_lds * paged_query_bytes(D, NG);
        u4 qw[kImpHeads][NS];
        float lse[kImpHeads];
#pragma unroll
        for (int k = 0; k < kImpHeads; ++k) {  // all at once: the last head's again where there are fewer
            const int64_t t = r.begin + qt;
            const int head = (h0 + min(k, nh - 1) * hs) * p.g + row % p.g;
            load_row<D>(qw[k], p.q + t * p.q_t + head * p.q_h);
            lse[k] = p.lse[t * p.Hq + head];
        }
        load(K[0], 0, h0);
        load(K[1], min(1, last) / nh, h0 + min(1, last) % nh * hs);
#pragma unroll
        for (int k = 0; k < kImpHeads; ++k) {
            if (k >= nh) break;
            Query<D, NG> Q;
            make_query<D, NG>(Q, qw[k], p.q_bf16, p.scale_log2);
            unsigned char *at = qs + k * paged_query_bytes(D, NG);
#pragma unroll
            for (int st = 0; st < NS; ++st) *(h8 *)(at + (st * 64 + lane) * 16) = Q.op[st];
            float *f = (float *)(at + NS * 1024);
            if (grp == 0) {
#pragma unroll
                for (int g = 0; g < NG; ++g) f[g * 16 + col] = Q.sum[g];
                f[NG * 16 + col] = Q.kx;
                f[(NG + 1) * 16 + col] = live ? lse[k] * -1.4426950408889634f : -INFINITY;
            }
        }
        __builtin_amdgcn_wave_barrier();
        float sum[NT * 4];
#pragma unroll
        for (int i = 0; i < NT * 4; ++i) sum[i] = 0.f;
        float *meta = smeta[wave];
        Nibbles nb;
        nb.init();
        int b = 0, k = 0;     // the pair that is next
        auto consume = [&](Keys &keys) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < NT; ++i) put_k_meta<NG>(meta + i * 2 * MT, lane & (MT - 1), keys.m[i]);
            __builtin_amdgcn_wave_barrier();
            const unsigned char *at = qs + k * paged_query_bytes(D, NG);
            const float *f = (const float *)(at + NS * 1024);
            Query<D, NG> Q;
#pragma unroll
            for (int st = 0; st < NS; ++st) Q.op[st] = *(const h8 *)(at + (st * 64 + lane) * 16);
#pragma unroll
            for (int g = 0; g < NG; ++g) Q.sum[g] = f[g * 16 + col];
            Q.kx = f[NG * 16 + col];
            const float bias = f[(NG + 1) * 16 + col];
            const int64_t tok = tok0 + b * (NT * 16);
            const uint32_t mine = have >> (NT * b) & ALL;
            const bool clean = mine == ALL && __builtin_amdgcn_ballot_w64(tok + NT * 16 <= see || !live) == ~0ull;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const f4 x = tile_scores<D, NG>(Q, nb, keys.kc[i], meta + i * 2 * MT);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], Q.kx, bias));
                    if (!clean) pr = tok + 16 * i + 4 * grp + e < see && (mine >> i & 1) ? pr : 0.f;
                    sum[4 * i + e] += pr;
                }
                __builtin_amdgcn_sched_barrier(0);  // one tile's meta in registers at a time
            }
            if (++k < nh) return;
            k = 0;
            // over the 16 rows: each step halves what a lane holds; lane col ends with its NT / 4 sums of the quad's
#pragma unroll
            for (int d = 8, c = NT * 2; d > 0; d >>= 1, c >>= 1)
#pragma unroll
                for (int i = 0; i < c; ++i) {
                    float x = sum[i], y = sum[i + c];
                    asm("" : "+v"(x), "+v"(y));  // or a choice of values becomes one of indexes, 16 selects long
                    sum[i] = (col & d ? y : x) + __shfl_xor(col & d ? x : y, d);
                }
#pragma unroll
            for (int i = 0; i < NT / 4; ++i) {
                const int v = NT / 4 * col + i;  // tile v / 4, token 4 grp + v % 4 of it
                sums[wave][b * (NT * 16) + 16 * (v >> 2) + 4 * grp + (v & 3)] = sum[i];
            }
#pragma unroll
            for (int i = 0; i < NT * 4; ++i) sum[i] = 0.f;
            ++b;
        };
        int lb = min(2, last) / nh, lk = min(2, last) % nh;  // the pair that is loaded next
        auto ahead = [&](Keys &keys) {
            load(keys, lb, h0 + lk * hs);
            if (lb * nh + lk < last && ++lk == nh) lk = 0, ++lb;
        };
        int i = 0;
        for (; i < last; i += 2) {
            consume(K[0]);
            ahead(K[0]);
            consume(K[1]);
            ahead(K[1]);
        }
        if (i == last) consume(K[0]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < runs * run_tok; i += kThreads) {
        const int64_t j = (int64_t)blockIdx.x * runs * run_tok + i;
        if (j >= p.n_scores) break;
        const int run = i / run_tok, in = i - run * run_tok;
        const float *old = p.scores + s * p.score_stride + j;
        float *out = p.out + s * p.out_stride + j;
        if (j < kv) {
            float v = 0.f;
            for (int q = 0; q < hs; ++q) v += sums[run * hs + q][in];
            *out = __builtin_fmaf(*old, p.decay, v / (float)p.Hq);
        } else if (out != old) {
            *out = *old;
        }
    }
}

namespace {
int attn_lds(const PagedAttnParams &p) { return 2 * kWaves * p.rows * (p.D + 4) * 4 + kWaves * 2 * 192 * p.ng; }
constexpr int64_t kSumsBytes = 2048;  // Scan::pre at the start of the workspace
static_assert((kThreads + 1) * 4 <= kSumsBytes, "the sums fit");
}  // namespace

// Most chunks of 16 rows that a sequence of few rows has.
static int few_chunks(const PagedAttnParams &p) {
    return (int)((std::min<int64_t>((int64_t)p.seqs.max_q * p.g, kFewRows) + kRows - 1) / kRows);
}

int64_t paged_attn_plan(PagedAttnParams *p) {
    const int64_t r = (int64_t)p->seqs.max_q * p->g;
    p->rows = (int)std::max<int64_t>(1, std::min<int64_t>(kRows, r));
    const int64_t units = std::max<int64_t>(1, (((int64_t)p->seqs.width << (p->pool.log_tpp + 4)) + kUnitTok - 1) / kUnitTok);
    const int64_t most = (units + kSetup) * p->seqs.n_seqs * p->pool.heads * few_chunks(*p);
    p->groups = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxGroups, (most + kWaves - 1) / kWaves));
    // where every sequence has the most rows there is none of few, and if there is the tiles take it
    if (r > kFewRows && p->seqs.n_tokens == (int64_t)p->seqs.n_seqs * p->seqs.max_q) p->groups = 0;
    // Short contexts and few of them: an item a workgroup, whatever its length, and nothing to merge
    // (the workspace is not used).  Against runs of equal work, us for 128, 256, 384 and 512 tokens,
    // bfloat16: 2 to 64 items: 9.5, 11.1, 12.7, 14.0 and 11.8, 11.8, 11.9, 12.1 (64: 13.7); 128 items: 9.7, 11.3,
    // 12.9, 14.3 and 12.2, 13.5, 13.8, 15.6.  For 512, 1024 and 2048 tokens of 256 items, which fill the
    // card: 14.7, 21.3, 32.4 and 17.7, 23.7, 31.9; 512 items: 19.2, 27.4, 41.8 and 24.7, 32.6, 47.7.  float16 is
    // 5% slower on both sides.  The lengths are on the device: the table's width stands for them.
    const int64_t items = (int64_t)p->seqs.n_seqs * p->pool.heads * few_chunks(*p);
    if (r <= kFewRows && items <= kMaxGroups && units <= (items >= kMaxGroups / 2 ? 32 : 8)) {
        p->whole = (int)((units + kSetup + kWaves - 1) / kWaves * kWaves);
        p->groups = (int)std::max<int64_t>(1, items);
        return kSumsBytes;
    }
    const int64_t own = p->groups ? kSumsBytes + (int64_t)p->groups * 2 * p->rows * (p->D + 4) * 4 : 0;
    p->tile_part = p->part + own / 4;
    return own + paged_tile_plan(p);
}

hipError_t paged_attn_launch(const PagedAttnParams &p0, hipStream_t st) {
    PagedAttnParams p = p0;
    if (p.seqs.n_seqs == 0 || p.seqs.max_q == 0) return hipSuccess;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    if (p.tile_groups) {
        const hipError_t e = paged_tile_launch(p, st);
        if (e != hipSuccess || !p.groups) return e;
    }
    if (!p.whole) {
        p.sums = (int *)p.part;
        p.part += kSumsBytes / 4;
    }
    const size_t lds = attn_lds(p);
    auto go = [&](auto kern) {
        if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        kern<<<dim3(p.groups), dim3(kThreads), lds, st>>>(p);
    };
    auto by_form = [&](auto two) {
        constexpr bool TWO = decltype(two)::value;
        if (p.D == 128) {
            if (p.ng == 4) go(paged_decode_kernel<128, 4, TWO>);
            else if (p.ng == 2) go(paged_decode_kernel<128, 2, TWO>);
            else go(paged_decode_kernel<128, 1, TWO>);
        } else {
            if (p.ng == 2) go(paged_decode_kernel<64, 2, TWO>);
            else go(paged_decode_kernel<64, 1, TWO>);
        }
    };
    if (p.q_bf16) by_form(std::false_type{});
    else by_form(std::true_type{});
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.whole) return e;
    const dim3 grid(p.pool.heads * few_chunks(p), p.seqs.n_seqs);
    if (p.D == 128) paged_merge_kernel<128><<<grid, dim3(kThreads), 0, st>>>(p);
    else paged_merge_kernel<64><<<grid, dim3(kThreads), 0, st>>>(p);
    return hipGetLastError();
}

hipError_t paged_importance_launch(const PagedImportanceParams &p0, hipStream_t st) {
    PagedImportanceParams p = p0;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    const int64_t window = p.q_window > 0 ? std::min(p.q_window, p.seqs.max_q) : p.seqs.max_q;
    if (window * p.g > kFewWindowRows) return paged_importance_tile_launch(p, st);
    p.head_split = p.pool.heads >= 4 ? 4 : p.pool.heads >= 2 ? 2 : 1;
    const int64_t tokens = kImpTiles * 16 * (kWaves / p.head_split);
    p.head_lds = (p.pool.heads + p.head_split - 1) / p.head_split;
    // Runs a wave of a decode step: as many as leave three workgroups a compute unit, what fits there.
    // Fewer than two do not pay for the operands' way through LDS (two sequences of 12000 tokens and 8
    // heads: 9.8 us in the kernel below, 11.1 here).
    const int64_t groups = (p.n_scores + tokens - 1) / tokens * p.seqs.n_seqs;
    p.blocks = (int)std::min<int64_t>(kImpBlocks, (groups + 384) / 768);
    if (window * p.g <= kRows && p.head_lds <= kImpHeads && p.blocks >= 2) {
        const dim3 grid((unsigned)((p.n_scores + tokens * p.blocks - 1) / (tokens * p.blocks)), p.seqs.n_seqs);
        auto go = [&](auto kern) {
            const int lds = kWaves * p.head_lds * paged_query_bytes(p.D, p.ng);
            if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            kern<<<grid, dim3(kThreads), lds, st>>>(p);
        };
        if (p.D == 128) {
            if (p.ng == 4) go(paged_importance_step_kernel<128, 4>);
            else if (p.ng == 2) go(paged_importance_step_kernel<128, 2>);
            else go(paged_importance_step_kernel<128, 1>);
        } else {
            if (p.ng == 2) go(paged_importance_step_kernel<64, 2>);
            else go(paged_importance_step_kernel<64, 1>);
        }
        return hipGetLastError();
    }
    const dim3 grid((unsigned)((p.n_scores + tokens - 1) / tokens), p.seqs.n_seqs), block(kThreads);
    if (p.D == 128) {
        if (p.ng == 4) paged_importance_kernel<128, 4><<<grid, block, 0, st>>>(p);
        else if (p.ng == 2) paged_importance_kernel<128, 2><<<grid, block, 0, st>>>(p);
        else paged_importance_kernel<128, 1><<<grid, block, 0, st>>>(p);
    } else {
        if (p.ng == 2) paged_importance_kernel<64, 2><<<grid, block, 0, st>>>(p);
        else paged_importance_kernel<64, 1><<<grid, block, 0, st>>>(p);
    }
    return hipGetLastError();
}

}  // namespace akv
