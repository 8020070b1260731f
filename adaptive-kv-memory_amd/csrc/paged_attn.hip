// Attention over the paged 4-bit cache, its merge, and the importance of cached tokens.
//
// The mathematics.  A key is c s + z with whole codes c and one float16 (s, z) per token and
// channel group, so q.k = sum over groups of s (q.c) + z (sum of q): the matrix cores take the
// codes themselves, and scale and zero enter once per score in float32.  A code in the low
// bits of a float16 is the subnormal c 2^-24, or 16 c 2^-24 one nibble higher, exact in the
// MFMA; the operand for the query takes the 1/16, its rows are scaled to a maximum in
// [2^13, 2^14), and the factor 2^24 leaves with the softmax scale.  Scores are thus exact to
// float32 rounding, whatever the cache's widths.  Values: o = sum of p (c s + z) is the product
// of the codes with p s (float16, rounded once more than p) plus sum of p z, one more MFMA row
// per channel group.  Softmax state: running maximum and sum per row in float32.
#include <algorithm>

#include "akv_common.h"
#include "paged.h"

namespace akv {
namespace {

constexpr float kMinMax = -0x1p126f;  // a finite start of the running maximum: a row that sees nothing stays at p = 0
constexpr int kThreads = 256, kWaves = 4, kRows = 16;
constexpr int kMaxGroups = 512;       // two workgroups a compute unit

__device__ __forceinline__ float xmax(float x) {
    x = __builtin_fmaxf(x, __shfl_xor(x, 16));
    return __builtin_fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float xsum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ h8 code_operand(uint32_t w) {
    const uint32_t v = w >> 8;
    return __builtin_bit_cast(h8, (u4){w & 0x000F000Fu, w & 0x00F000F0u, v & 0x000F000Fu, v & 0x00F000F0u});
}
__device__ __forceinline__ float lo_f(uint32_t w) { return (float)as_h2(w)[0]; }
__device__ __forceinline__ float hi_f(uint32_t w) { return (float)as_h2(w)[1]; }

// The query operand of 16 rows: lane (row col, quarter grp) holds channels 32 g + 8 grp ..
template <int D, int NG>
struct Query {
    h8 op[D / 32];
    float sum[NG];  // of the group's channels, times 2^-24
    float kx;       // score -> log2 domain
};

template <int D, int NG>
__device__ __forceinline__ void load_query(Query<D, NG> &Q, const unsigned char *row, bool bf16, float scale_log2) {
    constexpr int NS = D / 32;
    const int grp = (threadIdx.x >> 4) & 3;
    float x[NS][8];
    float top = 0.0f;
#pragma unroll
    for (int g = 0; g < NS; ++g) {
        const u4 w = *(const u4 *)(row + (32 * g + 8 * grp) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = w[i];
            x[g][2 * i] = bf16 ? __builtin_bit_cast(float, v << 16) : lo_f(v);
            x[g][2 * i + 1] = bf16 ? __builtin_bit_cast(float, v & 0xffff0000u) : hi_f(v);
            top = __builtin_fmaxf(top, __builtin_fmaxf(__builtin_fabsf(x[g][2 * i]), __builtin_fabsf(x[g][2 * i + 1])));
        }
    }
    top = xmax(top);
    const int ex = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 14;  // top = f 2^ex, f in [1/2, 1)
#pragma unroll
    for (int g = 0; g < NG; ++g) Q.sum[g] = 0.0f;
#pragma unroll
    for (int g = 0; g < NS; ++g) {
        float y[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            y[n] = __builtin_ldexpf(x[g][n], 14 - ex);
            Q.sum[g * NG / NS] += y[n];
        }
        Q.op[g] = (h8){(_Float16)y[0], (_Float16)y[4], (_Float16)(y[1] * 0.0625f), (_Float16)(y[5] * 0.0625f),
                       (_Float16)y[2], (_Float16)y[6], (_Float16)(y[3] * 0.0625f), (_Float16)(y[7] * 0.0625f)};
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) Q.sum[g] = xsum(Q.sum[g]) * 0x1p-24f;
    Q.kx = __builtin_ldexpf(scale_log2, ex + 10);
}

// Scores (times 2^-24 of the scaled query) of tokens 4 grp + e of a tile for row col.  `meta`:
// the tile's K meta in LDS.
template <int D, int NG>
__device__ __forceinline__ f4 tile_scores(const Query<D, NG> &Q, const uint32_t (&kc)[D / 32], const uint32_t *meta) {
    constexpr int NS = D / 32;
    const int grp = (threadIdx.x >> 4) & 3;
    uint32_t m[4 * NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const u4 w = ((const u4 *)meta)[grp * NG + i];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[4 * i + e] = w[e];
    }
    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        f4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < NS / NG; ++st) c = mfma_k32(code_operand(kc[g * (NS / NG) + st]), Q.op[g * (NS / NG) + st], c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = m[e * NG + g];
            s[e] = __builtin_fmaf(lo_f(w), c[e], s[e]);
            s[e] = __builtin_fmaf(hi_f(w), Q.sum[g], s[e]);
        }
    }
    return s;
}

// Units of a sequence: 32 cached tokens of one head for one chunk of 16 rows.
struct SeqWork {
    SeqRows r;
    int rows, chunks, units;  // rows = query tokens * g; units of one (head, chunk)
};
__device__ __forceinline__ SeqWork seq_work(const PagedAttnParams &p, int s) {
    SeqWork w;
    w.r = seq_rows(p.seqs, s, p.pool.log_tpp + 4);
    const int n = min(w.r.n, p.seqs.max_q);
    w.rows = n * p.g;
    w.chunks = (w.rows + kRows - 1) / kRows;
    w.units = max(1, (int)((w.r.kv + kUnitTok - 1) / kUnitTok));
    return w;
}
__device__ __forceinline__ int seq_total(const PagedAttnParams &p, int s) {
    const SeqWork w = seq_work(p, s);
    return w.chunks * w.units * p.pool.heads;
}

// Exclusive sums of the sequences' units: entry i is that of the first sequence of thread i
// (runs of `per` sequences), entry 256 the total.
__device__ __forceinline__ void scan_seqs(const PagedAttnParams &p, int *pre, int per) {
    __shared__ int wave_sum[kWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int mine = 0;
    for (int i = 0; i < per; ++i) {
        const int s = t * per + i;
        if (s < p.seqs.n_seqs) mine += seq_total(p, s);
    }
    int inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wave_sum[wave] = inc;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before += wave_sum[w];
    pre[t] = before + inc - mine;
    if (t == 255) pre[256] = before + inc;
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
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = o[2 * i] * inv, b = o[2 * i + 1] * inv;
        w[i] = p.q_bf16 ? f32_to_bf16_rne(a) | ((uint32_t)f32_to_bf16_rne(b) << 16) : as_u32((h2){(_Float16)a, (_Float16)b});
    }
    *(u4 *)((unsigned char *)p.out + ((t * p.Hq + head) * p.D + ch) * 2) = w;
    // p carries a factor 4
    if (p.lse && ch == 0) p.lse[t * p.Hq + head] = l > 0.0f || l != l ? 0.69314718055994531f * (m + (__builtin_log2f(l) - 2.0f)) : -INFINITY;
}

}  // namespace

// Single tokens and a few drafted ones: bound by the cache's bytes.
//
// The units of all sequences, heads and chunks form one list, cut into equal runs, one a wave:
// every wave has the same work whatever the lengths.  A run that covers an item (all units of
// a sequence, head and chunk) writes its rows; states of items that end or begin inside a
// workgroup's runs are joined through LDS, items that several workgroups share leave partial
// states for paged_merge_kernel.  A wave loads its tiles straight to registers, two units
// ahead; the meta of a tile goes through LDS, where each lane reads its tokens'.
template <int D, int NG>
__global__ __launch_bounds__(kThreads, 2) void paged_decode_kernel(const PagedAttnParams p) {
    constexpr int NS = D / 32, NB = D / 16, TB = paged_tile_bytes(D, NG), EROW = D + 4;
    constexpr int MW = NG == 4 ? 2 : 1;          // meta dwords a lane loads of a tile
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int pre[257];
    __shared__ int e_seq[2 * kWaves], e_item[2 * kWaves], e_flags[2 * kWaves];  // flags: 1 used, 2 starts, 4 ends
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int k_at = (4 * col + grp) * (D / 8);  // K codes of token col, quarter grp
    float *entries = (float *)smem;
    uint32_t *meta = (uint32_t *)(smem + 2 * kWaves * p.rows * EROW * 4) + wave * 2 * 32 * NG;
    if (lane < 2) e_flags[2 * wave + lane] = 0;

    const int per = (p.seqs.n_seqs + 255) / 256;
    scan_seqs(p, pre, per);
    const int total = pre[256];
    const int share = share_of(total, p.groups);
    int x = (int)min((int64_t)(blockIdx.x * kWaves + wave) * share, (int64_t)total);
    const int x_end = min(x + share, total);

    // the sequence of unit x
    int s = 0, off = 0;
    SeqWork w{};
    if (x < x_end) {
        int k = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) k += __builtin_popcountll(__builtin_amdgcn_ballot_w64(pre[64 * i + lane] <= x));
        s = (k - 1) * per;
        off = x - __builtin_amdgcn_readfirstlane(pre[k - 1]);
        for (;;) {
            w = seq_work(p, s);
            const int n = w.chunks * w.units * p.pool.heads;
            if (off < n) break;
            off -= n;
            ++s;
        }
    }
    while (x < x_end) {
        const int item = off / w.units, j0 = off - item * w.units;
        const int j1 = min(w.units, j0 + (x_end - x));
        const int h = item / w.chunks, row0 = (item - h * w.chunks) * kRows;
        const int rows = min(kRows, w.rows - row0);

        const int row = row0 + min(col, rows - 1);
        const int qt = row / p.g;
        const int64_t kv = w.r.kv;
        const int64_t old = p.causal ? kv - w.r.n + 1 : kv;  // cached tokens the call's first row sees
        const int see = (int)(p.causal ? max(old + qt, (int64_t)0) : kv);
        const int see_all = (int)(p.causal ? max(old + row0 / p.g, (int64_t)0) : kv);
        const int see_any = (int)(p.causal ? max(old + (row0 + rows - 1) / p.g, (int64_t)0) : kv);
        Query<D, NG> Q;
        load_query<D, NG>(Q, p.q + (w.r.begin + qt) * p.q_t + (h * p.g + row % p.g) * p.q_h, p.q_bf16, p.scale_log2);

        const int32_t *table = p.seqs.table + s * p.seqs.table_stride;
        const int jn = min(j1, (see_any + kUnitTok - 1) / kUnitTok);
        const int log_tpp = p.pool.log_tpp;
        int pb = (2 * j0) >> log_tpp;
        int pid = pb + lane < p.seqs.width ? table[pb + lane] : -1;

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
                }
                uint32_t page = (uint32_t)__builtin_amdgcn_readlane(pid, pi - pb);
                const int left = (int)(kv - 16 * (int64_t)t);
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
        f4 acc[NB], accz = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = (f4){0.f, 0.f, 0.f, 0.f};

        auto consume = [&](Unit &u, int j) {
            const bool clean = kUnitTok * (j + 1) <= see_all && u.nv[0] == 16 && u.nv[1] == 16;
            if (!clean) {  // V meta of slots without a token: whatever is there becomes 0
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < MW; ++q) {
                        const int d = (lane & (32 * NG / MW - 1)) * MW + q - 16 * NG;
                        const int tok = ((d & (8 * NG - 1)) / (2 * NG)) * 4 + (d & 1) * 2;
                        if (d >= 0) u.m[i][q] &= (tok < u.nv[i] ? 0xffffu : 0u) | (tok + 1 < u.nv[i] ? 0xffff0000u : 0u);
                    }
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t *m = meta + i * 32 * NG;
                if constexpr (MW == 2) *(u2 *)(m + 2 * lane) = (u2){u.m[i][0], u.m[i][1]};
                else m[lane & (32 * NG - 1)] = u.m[i][0];
            }
            __builtin_amdgcn_wave_barrier();
            f4 sc[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sc[i] = tile_scores<D, NG>(Q, u.kc[i], meta + i * 32 * NG) * Q.kx;
                if (!clean)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int in = 4 * grp + e;
                        if (kUnitTok * j + 16 * i + in >= see || in >= u.nv[i]) sc[i][e] = -INFINITY;
                    }
            }
            float t = sc[0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) t = __builtin_fmaxf(t, sc[e >> 2][e & 3]);
            if (__builtin_amdgcn_ballot_w64(t > mx)) {
                const float mn = __builtin_fmaxf(mx, xmax(t));
                const float alpha = __builtin_amdgcn_exp2f(mx - mn);
                l *= alpha;
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] *= alpha;
                accz *= alpha;
                mx = mn;
            }
            // p in (0, 4]: p s stays in float16 for every scale that the append writes
            const float bias = 2.0f - mx;
            float pr[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) pr[e] = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] + bias);
            l += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
            h2 ph[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) ph[q] = (h2){(_Float16)pr[2 * q], (_Float16)pr[2 * q + 1]};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                u4 pw;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const u2 sv = *(const u2 *)(meta + i * 32 * NG + 16 * NG + (grp * NG + g) * 2);
                    pw[2 * i] = as_u32(ph[2 * i] * as_h2(sv[0]));
                    pw[2 * i + 1] = as_u32(ph[2 * i + 1] * as_h2(sv[1]));
                }
                const h8 pg = __builtin_bit_cast(h8, pw);
                // the group's blocks of 16 channels: block 4 h + 2 l + b is nibble 2 l + b of half h
#pragma unroll
                for (int b = g * (NB / NG); b < (g + 1) * (NB / NG); ++b) {
                    const int h4 = b >> 2, n = b & 3;
                    u4 a;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t v = u.vc[q >> 1][(q & 1) * (NB / 4) + h4];
                        a[q] = (n >= 2 ? v >> 8 : v) & (n & 1 ? 0x00F000F0u : 0x000F000Fu);
                    }
                    acc[b] = mfma_k32(__builtin_bit_cast(h8, a), pg, acc[b]);
                }
            }
            u4 za = {0u, 0u, 0u, 0u};
            if (col < NG) {
                const u2 a = *(const u2 *)(meta + 24 * NG + (grp * NG + col) * 2);
                const u2 b = *(const u2 *)(meta + 32 * NG + 24 * NG + (grp * NG + col) * 2);
                za = (u4){a[0], a[1], b[0], b[1]};
            }
            accz = mfma_k32(__builtin_bit_cast(h8, za), __builtin_bit_cast(h8, (u4){as_u32(ph[0]), as_u32(ph[1]), as_u32(ph[2]), as_u32(ph[3])}), accz);
        };

        if (j0 < jn) load(U[0], j0);
        if (j0 + 1 < jn) load(U[1], j0 + 1);
        for (int j = j0; j < jn; j += 2) {
            consume(U[0], j);
            if (j + 2 < jn) load(U[0], j + 2);
            if (j + 1 < jn) {
                consume(U[1], j + 1);
                if (j + 3 < jn) load(U[1], j + 3);
            }
        }

        // the segment's state in true units: 2^24 of the codes (2^20 where they lay a nibble higher), zeros
        l = xsum(l);
        float z[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) z[g] = __shfl(accz[g], col);
        const bool starts = j0 == 0, ends = j1 == w.units;
        const int slot = 2 * wave + (ends ? 0 : 1);
        float *er = entries + (slot * p.rows + col) * EROW;
#pragma unroll
        for (int g = 0; g < NS; ++g) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[2 * i] = __builtin_fmaf(acc[2 * g][i], 0x1p24f, z[g * NG / NS]);
                o[2 * i + 1] = __builtin_fmaf(acc[2 * g + 1][i], 0x1p20f, z[g * NG / NS]);
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

        x += j1 - j0;
        off += j1 - j0;
        if (x < x_end && off == w.chunks * w.units * p.pool.heads) {
            do w = seq_work(p, ++s);
            while (w.chunks == 0);
            off = 0;
        }
    }

    // join what the runs left: entries of one item are neighbours
    __syncthreads();
    const int row_t = threadIdx.x >> 4, ch = (threadIdx.x & 15) * (D / 16);
    float o[8];
    float M = 0.f, L = 0.f;
    bool open = false, began = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.f;
    for (int e = 0; e < 2 * kWaves; ++e) {
        const int f = e_flags[e];
        if (!(f & 1)) continue;
        if (!open) began = f & 2;
        if (row_t < p.rows) {
            const float *er = entries + (e * p.rows + row_t) * EROW;
            const float m = er[D], le = er[D + 1];
            const float mn = open ? __builtin_fmaxf(M, m) : m;
            const float a = open ? __builtin_amdgcn_exp2f(M - mn) : 0.f, b = __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] = open ? __builtin_fmaf(er[ch + i], b, o[i] * a) : er[ch + i];
            L = open ? __builtin_fmaf(le, b, L * a) : le;
            M = mn;
        }
        open = !(f & 4);
        bool last = !open;
        if (open) {  // nothing more of it in this workgroup?
            last = true;
            for (int e2 = e + 1; e2 < 2 * kWaves; ++e2) last &= !(e_flags[e2] & 1);
        }
        if (!last) continue;
        if (began && (f & 4)) {
            const SeqWork sw = seq_work(p, e_seq[e]);
            const int it = e_item[e], h = it / sw.chunks, row = (it - h * sw.chunks) * kRows + row_t;
            if (row_t < kRows && row < sw.rows && row_t < p.rows) {
                if constexpr (D == 128) {
                    write_row(p, sw.r, h, row, ch, o, M, L);
                } else {  // 4 channels a thread: pairs of threads write together
                    float o8[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o8[i] = o[i], o8[4 + i] = __shfl_down(o[i], 1);
                    if (!(threadIdx.x & 1)) write_row(p, sw.r, h, row, ch, o8, M, L);
                }
            }
        } else if (row_t < p.rows) {
            float *pr = p.part + ((int64_t)(2 * blockIdx.x + (began ? 1 : 0)) * p.rows + row_t) * EROW;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) pr[ch + i] = o[i];
            if (ch == 0) pr[D] = M, pr[D + 1] = L;
        }
    }
}

// Items that several workgroups share: one workgroup an item joins their partial states in order.
template <int D>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedAttnParams p) {
    constexpr int EROW = D + 4;
    __shared__ int pre[257];
    const int per = (p.seqs.n_seqs + 255) / 256;
    scan_seqs(p, pre, per);
    const int share = share_of(pre[256], p.groups) * kWaves;  // units a workgroup has
    const int s = blockIdx.y, k = s / per;
    int at = pre[k];
    for (int i = k * per; i < s; ++i) at += seq_total(p, i);
    const SeqWork w = seq_work(p, s);
    for (int item = blockIdx.x; item < w.chunks * p.pool.heads; item += gridDim.x) {
        const int first = at + item * w.units;
        const int g0 = first / share, g1 = (first + w.units - 1) / share;
        if (g0 == g1) continue;
        const int row_t = threadIdx.x >> 4, ch = (threadIdx.x & 15) * (D / 16);
        const int h = item / w.chunks, row = (item - h * w.chunks) * kRows + row_t;
        if (row_t >= p.rows || row >= w.rows) continue;
        float o[8];
        float M = kMinMax, L = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0.f;
        for (int g = g0; g <= g1; ++g) {
            const float *pr = p.part + ((int64_t)(2 * g + (g == g0 ? 1 : 0)) * p.rows + row_t) * EROW;
            const float m = pr[D], l = pr[D + 1];
            const float mn = __builtin_fmaxf(M, m);
            const float a = __builtin_amdgcn_exp2f(M - mn), b = __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] = __builtin_fmaf(pr[ch + i], b, o[i] * a);
            L = __builtin_fmaf(l, b, L * a);
            M = mn;
        }
        if constexpr (D == 128) {
            write_row(p, w.r, h, row, ch, o, M, L);
        } else {
            float o8[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) o8[i] = o[i], o8[4 + i] = __shfl_down(o[i], 1);
            if (!(threadIdx.x & 1)) write_row(p, w.r, h, row, ch, o8, M, L);
        }
    }
}

// The importance: a workgroup takes 64 tokens of a sequence, its waves the heads in turn; the
// sum over rows stays in registers and is joined over heads in a fixed order.  Bound by the K
// half of the cache.
template <int D, int NG>
__global__ __launch_bounds__(kThreads) void paged_importance_kernel(const PagedImportanceParams p) {
    constexpr int NS = D / 32, TB = paged_tile_bytes(D, NG), NT = 4;
    __shared__ __align__(16) uint32_t smeta[kWaves][NT * 16 * NG];
    __shared__ float sums[kWaves][NT * 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int k_at = (4 * col + grp) * (D / 8);  // K codes of token col, quarter grp
    const int s = blockIdx.y;
    const SeqRows r = seq_rows(p.seqs, s, p.pool.log_tpp + 4);
    const int64_t tok0 = (int64_t)blockIdx.x * (NT * 16);
    const int n = min(r.n, p.seqs.max_q);
    const int64_t kv = n > 0 ? min(r.kv, p.n_scores) : 0;  // tokens whose score changes
    const int first = p.q_window > 0 && p.q_window < n ? n - p.q_window : 0;
    const int rows = (n - first) * p.g;
    float sum[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][e] = 0.f;
    uint32_t *meta = smeta[wave];
    if (tok0 < kv) {
        const int log_tpp = p.pool.log_tpp;
        const int32_t *table = p.seqs.table + s * p.seqs.table_stride;
        int64_t at[NT];   // the tiles' places for head 0
        int nv[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int64_t t = (tok0 >> 4) + i;
            const int64_t left = r.kv - 16 * t;
            uint32_t page = left > 0 ? (uint32_t)table[t >> log_tpp] : 0xffffffffu;
            nv[i] = page < p.pool.n_pages ? (int)min(left, (int64_t)16) : 0;
            if (page >= p.pool.n_pages) page = 0;
            at[i] = (int64_t)page * p.pool.page_bytes + (t & ((1 << log_tpp) - 1)) * TB;
        }
        for (int h = wave; h < p.pool.heads; h += kWaves) {
            uint32_t kc[NT][NS];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const unsigned char *tile = p.pool.base + at[i] + ((int64_t)h << log_tpp) * TB;
                if constexpr (D == 128) {
                    const u4 a = *(const u4 *)(tile + k_at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kc[i][e] = a[e];
                } else {
                    const u2 a = *(const u2 *)(tile + k_at);
                    kc[i][0] = a[0], kc[i][1] = a[1];
                }
                meta[i * 16 * NG + (lane & (16 * NG - 1))] = *(const uint32_t *)(tile + 16 * D + (lane & (16 * NG - 1)) * 4);
            }
            __builtin_amdgcn_wave_barrier();
            for (int row0 = 0; row0 < rows; row0 += kRows) {
                const int row = min(row0 + col, rows - 1);
                const int qt = first + row / p.g;
                const int64_t t = r.begin + qt;
                const int head = h * p.g + row % p.g;
                Query<D, NG> Q;
                load_query<D, NG>(Q, p.q + t * p.q_t + head * p.q_h, p.q_bf16, p.scale_log2);
                const float lse2 = row0 + col < rows ? p.lse[t * p.Hq + head] * 1.4426950408889634f : INFINITY;
                const int64_t see = p.causal ? r.kv - r.n + qt + 1 : r.kv;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const f4 sc = tile_scores<D, NG>(Q, kc[i], meta + i * 16 * NG);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int in = 4 * grp + e;
                        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], Q.kx, -lse2));
                        if (tok0 + 16 * i + in < see && in < nv[i]) sum[i][e] += row0 + col < rows ? pr : 0.f;
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = sum[i][e];
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d);
            if (col == 0) sums[wave][16 * i + 4 * grp + e] = v;
        }
    __syncthreads();
    const int64_t j = tok0 + threadIdx.x;
    if (threadIdx.x < NT * 16 && j < p.n_scores) {
        const float *old = p.scores + s * p.score_stride + j;
        float *out = p.out + s * p.out_stride + j;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kWaves; ++q) v += sums[q][threadIdx.x];
        if (j < kv) *out = __builtin_fmaf(*old, p.decay, v / (float)p.Hq);
        else if (out != old) *out = *old;
    }
}

namespace {
int attn_lds(const PagedAttnParams &p) { return 2 * kWaves * p.rows * (p.D + 4) * 4 + kWaves * 2 * 128 * p.ng; }
}  // namespace

int64_t paged_attn_plan(PagedAttnParams *p) {
    const int64_t r = (int64_t)p->seqs.max_q * p->g;
    p->rows = (int)std::max<int64_t>(1, std::min<int64_t>(kRows, r));
    const int64_t units = std::max<int64_t>(1, (((int64_t)p->seqs.width << (p->pool.log_tpp + 4)) + kUnitTok - 1) / kUnitTok);
    const int64_t most = units * p->seqs.n_seqs * p->pool.heads * std::max<int64_t>(1, (r + kRows - 1) / kRows);
    p->groups = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxGroups, (most + kWaves - 1) / kWaves));
    return (int64_t)p->groups * 2 * p->rows * (p->D + 4) * 4;
}

hipError_t paged_attn_launch(const PagedAttnParams &p0, hipStream_t st) {
    PagedAttnParams p = p0;
    if (p.seqs.n_seqs == 0 || p.seqs.max_q == 0) return hipSuccess;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    const size_t lds = attn_lds(p);
    auto go = [&](auto kern) {
        if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        kern<<<dim3(p.groups), dim3(kThreads), lds, st>>>(p);
    };
    if (p.D == 128) {
        if (p.ng == 4) go(paged_decode_kernel<128, 4>);
        else if (p.ng == 2) go(paged_decode_kernel<128, 2>);
        else go(paged_decode_kernel<128, 1>);
    } else {
        if (p.ng == 2) go(paged_decode_kernel<64, 2>);
        else go(paged_decode_kernel<64, 1>);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t items = ((int64_t)p.seqs.max_q * p.g + kRows - 1) / kRows * p.pool.heads;
    const dim3 grid((unsigned)std::min<int64_t>(items, 1024), p.seqs.n_seqs);
    if (p.D == 128) paged_merge_kernel<128><<<grid, dim3(kThreads), 0, st>>>(p);
    else paged_merge_kernel<64><<<grid, dim3(kThreads), 0, st>>>(p);
    return hipGetLastError();
}

hipError_t paged_importance_launch(const PagedImportanceParams &p0, hipStream_t st) {
    PagedImportanceParams p = p0;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    const dim3 grid((unsigned)((p.n_scores + 63) / 64), p.seqs.n_seqs), block(kThreads);
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
