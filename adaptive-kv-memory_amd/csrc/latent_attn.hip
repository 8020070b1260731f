// Attention over the paged latent cache in its absorbed form, its merge, and the importance of
// cached tokens.
//
// The mathematics.  The heads' key matrices are in the queries already, so a cached row (latent c,
// rotated key r) is the key of every head and its latent the value: s = q.c + q_r.r, o = sum of p c.
// The rows of all heads and query tokens of a sequence thus share one stream of cached rows.  A float16 query
// row enters as it is, a bfloat16 one as float16 after scaling by a power of two to a maximum in [2^13, 2^14),
// which leaves with the softmax scale; scores are exact but for float32 sums and, in bfloat16 rows, values below 2^-28
// of the row's largest.  p is one float16 for bfloat16 outputs (an eighth of their own half step), two for float16.
// Softmax state: running maximum and sum per row in float32.
#include <algorithm>
#include <type_traits>

#include "akv_common.h"
#include "latent.h"
#include "latent_device.h"

namespace akv {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kUnit = 64;             // tokens of a unit of work
constexpr int kSetup = 5;             // units that an item's start counts
constexpr int kGroups = 256;          // one workgroup a compute unit

// A row's query: lane (row, quarter grp) holds channels 32 i + 8 grp .. of latent and rope.
template <int DC>
struct Row {
    static constexpr int NI = (DC + kLatentRope) / 32;
    u4 w[NI];
    __device__ __forceinline__ void load(const LatentAttnParams &p, int t, int h, int grp) {
        const unsigned char *q = p.q + t * p.q_t + h * p.q_h + 16 * grp, *qr = p.qr + t * p.qr_t + h * p.qr_h + 16 * grp;
#pragma unroll
        for (int i = 0; i < NI; ++i) w[i] = i < DC / 32 ? *(const u4 *)(q + 64 * i) : *(const u4 *)(qr + 64 * (i - DC / 32));
    }
};

// The work of a sequence, in units of kUnit cached tokens for one tile of rows.
struct Work {
    SeqRows r;
    int rows, tiles, cost;
};
__device__ __forceinline__ Work seq_work(const LatentAttnParams &p, const SeqRows &r) {
    Work w;
    w.r = r;
    w.rows = min(r.n, p.seqs.max_q) * p.H;
    w.tiles = (w.rows + (1 << p.log_tile) - 1) >> p.log_tile;
    w.cost = max(1, (r.kv + kUnit - 1) / kUnit) + kSetup;
    return w;
}

__device__ __forceinline__ int share_of(const LatentAttnParams &p, int total) {
    return max(1, (int)fast_div((uint32_t)(total + p.groups - 1), p.by_groups));
}

// The sequences of a call in LDS: where their units lie (pre[i]: the first unit of sequence i * per,
// pre[256] the total), and up to KEPT sequences their rows (256 or none).
template <int KEPT>
struct Scan {
    int pre[kThreads + 1];
    int wave_sum[kThreads / 64];
    SeqRows rows[KEPT ? KEPT : 1];
};
__device__ __forceinline__ int seqs_per(const LatentAttnParams &p) { return p.seqs.n_seqs <= kThreads ? 1 : (p.seqs.n_seqs + kThreads - 1) / kThreads; }
template <int KEPT>
__device__ __forceinline__ SeqRows rows_of(const LatentAttnParams &p, const Scan<KEPT> &sc, int s) {
    return wave_uniform(p.seqs.n_seqs <= KEPT ? sc.rows[s] : seq_rows(p.seqs, s, p.pool.log_page));
}
// For workgroups of 256 threads or more; the total.
template <int KEPT>
__device__ __forceinline__ int scan_seqs(const LatentAttnParams &p, Scan<KEPT> &sc) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n = p.seqs.n_seqs, per = seqs_per(p);
    int mine = 0, inc = 0;
    if (t < kThreads) {
        for (int i = 0; i < per; ++i) {
            const int s = t * per + i;
            if (s < n) {
                const SeqRows r = seq_rows(p.seqs, s, p.pool.log_page);
                const Work w = seq_work(p, r);
                mine += w.tiles * w.cost;
                if (KEPT && per == 1) sc.rows[t] = r;
            }
        }
        inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 63) sc.wave_sum[wave] = inc;
    }
    __syncthreads();
    if (t < kThreads) {
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) inc += w < wave ? sc.wave_sum[w] : 0;
        sc.pre[t] = inc - mine;
        if (t == kThreads - 1) sc.pre[kThreads] = inc;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(sc.pre[kThreads]);
}

// A run of units as items: whole or partial (sequence, tile of rows).
struct Run {
    int x, x_end, s, off;
    Work w;
};
struct Item {
    int tile, j0, j1;
    bool starts, ends;
};
template <int KEPT>
__device__ __forceinline__ Run run_of(const LatentAttnParams &p, const Scan<KEPT> &sc, int total) {
    const int lane = threadIdx.x & 63, per = seqs_per(p), share = share_of(p, total);
    Run r{};
    r.x = (int)min((int64_t)blockIdx.x * share, (int64_t)total);
    r.x_end = min(r.x + share, total);
    if (r.x >= r.x_end) return r;
    int k = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) k += __builtin_popcountll(__builtin_amdgcn_ballot_w64(sc.pre[64 * i + lane] <= r.x));
    r.s = (k - 1) * per;
    r.off = r.x - __builtin_amdgcn_readfirstlane(sc.pre[k - 1]);
    for (;;) {
        r.w = seq_work(p, rows_of(p, sc, r.s));
        const int n = r.w.tiles * r.w.cost;
        if (r.off < n) break;
        r.off -= n;
        ++r.s;
    }
    return r;
}
// The item that the run's first unit lies in, for the merge, where the run before it holds units of it too
// (an item's first kSetup are none).
__device__ __forceinline__ void note_join(const LatentAttnParams &p, const Run &r, int total) {
    if (threadIdx.x != 0) return;
    const int g = blockIdx.x, share = share_of(p, total);
    LatentJoin j{};
    if (r.x < r.x_end) {
        const int tile = r.off / r.w.cost, start = r.x - (r.off - tile * r.w.cost);
        const int g0 = (start + kSetup) / share, g1 = (start + r.w.cost - 1) / share;
        if (g0 < g) j = LatentJoin{r.w.r.begin, r.w.rows, tile << p.log_tile, (uint16_t)g0, (uint16_t)g1};
    }
    p.joins[g] = j;
}
// The next item's part of the run; false at the end.
template <int KEPT>
__device__ __forceinline__ bool next_item(const LatentAttnParams &p, const Scan<KEPT> &sc, Run &r, Item &it) {
    if (r.x >= r.x_end) return false;
    while (r.off == r.w.tiles * r.w.cost) {
        r.off = 0;
        r.w = seq_work(p, rows_of(p, sc, ++r.s));
    }
    it.tile = r.w.tiles == 1 ? 0 : __builtin_amdgcn_readfirstlane(r.off / r.w.cost);  // (divided by vector instructions)
    const int c0 = r.off - it.tile * r.w.cost, c1 = min(r.w.cost, c0 + (r.x_end - r.x));
    it.j0 = max(0, c0 - kSetup), it.j1 = max(0, c1 - kSetup);
    it.starts = it.j0 == 0, it.ends = c1 == r.w.cost;
    r.x += c1 - c0;
    r.off += c1 - c0;
    return it.j1 > 0;  // else no unit of the item is in the run, and the run ends
}
// Partial states of ROWS rows: sums as 16 x 16 tiles (16 rows, then 16 channels) of a lane's four
// floats, then the rows' maxima and sums.  Entry 0 of a workgroup: the item began before its run; 1: it ends
// behind it.
template <int DC, int ROWS>
__device__ __forceinline__ float *entry_of(const LatentAttnParams &p, int group, bool starts) {
    return p.part + ((int64_t)group * 2 + starts) * (ROWS * (DC + 2));
}

}  // namespace

// Up to 16 rows a sequence (a token's heads).  Bound by the cache's bytes: 24 sequences of up to 65536 tokens
// and 16 heads (269 MB) take 60 us, of which the memory's rate is 49 and the rest an item's chain of
// lengths, pages, loads and its join, which is all of the 13 us of one sequence of 517.  (In the form for more rows:
// 87 us.)
//
// TWO, for float16 outputs: p is two float16, which memory hides (calls of 71.5 against 71 us for the sequences above): one leaves
// outputs up to 2.4e-4 of their norm off, where their own rounding is 2.1e-4.
//
// Each of the four waves takes 16 tokens at a time for all 16 rows, from two buffers of LDS of its own
// that buffer loads fill; nothing is shared until the waves join at an item's end.  What is run once for an item is
// kept short: the code comes from memory too.
template <int DC, bool TWO>
__global__ __launch_bounds__(kThreads, 2) void latent_few_kernel(const LatentAttnParams p) {
    using T = Rows16<DC>;
    constexpr int NI = Row<DC>::NI, NB = DC / 16, ROWB = T::ROWB, SLOTS = 2;
    constexpr int OWN = NB / kWaves;  // blocks of channels that a wave joins and writes
    static_assert(NB * 1024 <= SLOTS * T::BYTES, "a wave's sums fit its buffers");
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Scan<kThreads> sc;
    __shared__ float ms[kWaves][16], ls[kWaves][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const uint32_t ring = __builtin_amdgcn_readfirstlane(lds_addr(smem) + wave * SLOTS * T::BYTES);
    const uint32_t k_at = col * ROWB + ((grp ^ turn(col)) << 4);
    const int vrow = 4 * grp + (col >> 2);
    const uint32_t v_at = vrow * ROWB + ((((col & 3) >> 1) ^ turn(vrow)) << 4) + 8 * (col & 1);

    const int total = scan_seqs(p, sc);
    Run run = run_of(p, sc, total);
    note_join(p, run, total);
    Item it;
    while (next_item(p, sc, run, it)) {
        const Work &w = run.w;
        const int row = min(col, w.rows - 1), qt = (int)fast_div(row, p.by_heads), h = row - qt * p.H;
        const int see = w.r.sees(p.causal, qt), see_all = w.r.sees(p.causal, 0), see_any = w.r.sees(p.causal, (int)fast_div(w.rows - 1, p.by_heads));
        const int key0 = it.j0 * kUnit, key1 = min(it.j1 * kUnit, see_any);
        const int steps = key1 > key0 ? (key1 - key0 + kUnit - 1) / kUnit : 0;
        Pages pages{p.seqs.table + run.s * p.seqs.table_stride, p.seqs.width, 0, 0};
        bool there[SLOTS] = {};
        auto load = [&](int t, int slot) {
            const int k = key0 + t * kUnit + wave * 16;
            const Tile tile = tile_at(p.pool, pages, k, t < steps ? w.r.kv : 0);
            there[slot] = tile.there;
            load_tile<DC>(wave_rsrc(tile.at, tile.rows * ROWB), ring + slot * T::BYTES, lane);
        };
        if (steps) {
            pages.fill(key0 >> p.pool.log_page);
            load(0, 0);
            load(1, 1);
        }
        h8 Q[NI];
        float kx;
        {
            Row<DC> raw;
            raw.load(p, w.r.begin + qt, h, grp);
            kx = query_operand(Q, raw.w, p.q_bf16, p.scale_log2);
        }
        float mx = kMinMax, l = 0.0f;
        f4 acc[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = (f4){0.f, 0.f, 0.f, 0.f};

#pragma unroll 1
        for (int t = 0; t < steps; ++t) {
            const int slot = t & 1;
            wait_vm<T::PIECES>();  // the next step's rows are still on their way
            const uint32_t at = ring + slot * T::BYTES;
            const int first = key0 + t * kUnit + wave * 16;
            const bool here = slot ? there[1] : there[0];
            f4 S2[2] = {};
            const uint32_t ka = at + k_at, kb = ka ^ 64;
#pragma unroll
            for (int c = 0; c < NI; ++c)
                S2[c & 1] = mfma_k32(__builtin_bit_cast(h8, *lds_ptr<u4>((c & 1 ? kb : ka) + (c >> 1) * 128)), Q[c], S2[c & 1]);
            f4 S = S2[0] + S2[1];
            if (!(first + 16 <= see_all && here))
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (first + 4 * grp + e >= see || !here) S[e] = -INFINITY;
            const float top = __builtin_fmaxf(__builtin_fmaxf(S[0], S[1]), __builtin_fmaxf(S[2], S[3]));
            if (__builtin_amdgcn_ballot_w64(__builtin_fmaf(top, kx, kBias - mx) > kBias + kLagBy)) {
                const float most = qmax(top);
                const float mn = __builtin_fmaf(most, kx, kBias - mx) > kBias ? running_max(most, kx, kBias) : mx;
                const float alpha = __builtin_amdgcn_exp2f(mx - mn);
                l *= alpha;
                mx = mn;
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] *= alpha;
            }
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], kx, kBias - mx));
            l += (e[0] + e[1]) + (e[2] + e[3]);
            const h4 P = {(_Float16)e[0], (_Float16)e[1], (_Float16)e[2], (_Float16)e[3]};
            h4 rest;
            if constexpr (TWO)
#pragma unroll
                for (int i = 0; i < 4; ++i) rest[i] = (_Float16)(e[i] - (float)P[i]);
            const uint32_t va = at + v_at;
            constexpr int AHEAD = 4;  // reads that are under way
            u2 V[AHEAD];
            auto value = [&](int b) { return read_transposed((va ^ (32 * (b & 3))) + (b >> 2) * 128); };
#pragma unroll
            for (int b = 0; b < AHEAD; ++b) V[b] = value(b);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if constexpr (TWO) acc[b] = mfma_k16(__builtin_bit_cast(h4, V[b % AHEAD]), rest, acc[b]);
                acc[b] = mfma_k16(__builtin_bit_cast(h4, V[b % AHEAD]), P, acc[b]);
                if (b + AHEAD < NB) V[b % AHEAD] = value(b + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
            wait_lgkm0();
            asm volatile("" ::: "memory");
            // (one copy of the loads' code for both buffers)
            const int k = key0 + (t + SLOTS) * kUnit + wave * 16;
            const Tile tile = tile_at(p.pool, pages, k, t + SLOTS < steps ? w.r.kv : 0);
            if (slot) there[1] = tile.there;
            else there[0] = tile.there;
            load_tile<DC>(wave_rsrc(tile.at, tile.rows * ROWB), __builtin_amdgcn_readfirstlane(at), lane);
        }
        wait_vm<0>();

        // The waves' states meet in LDS, each wave then sums its share of the channels.
        l = qsum(l);
        if (grp == 0) ms[wave][col] = mx, ls[wave][col] = l;
        __syncthreads();
        float mj = ms[0][col];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) mj = __builtin_fmaxf(mj, ms[i][col]);
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) l += ls[i][col] * __builtin_amdgcn_exp2f(ms[i][col] - mj);
        const float alpha = __builtin_amdgcn_exp2f(mx - mj);
        unsigned char *states = smem + wave * SLOTS * T::BYTES + lane * 16;
#pragma unroll
        for (int b = 0; b < NB; ++b) *(f4 *)(states + b * 1024) = acc[b] * alpha;
        __syncthreads();
        const bool whole = it.starts && it.ends;
        const float inv = row_inverse(l);
        const int64_t o = (int64_t)(w.r.begin + qt) * p.H + h;
        unsigned char *out = (unsigned char *)p.out + o * (2 * DC) + 8 * grp;
        float *e = entry_of<DC, 16>(p, blockIdx.x, it.starts);
#pragma unroll 2
        for (int b = wave * OWN; b < (wave + 1) * OWN; ++b) {
            f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kWaves; ++i) v += *(const f4 *)(smem + i * SLOTS * T::BYTES + b * 1024 + lane * 16);
            if (whole) {
                v *= inv;
                if (col < w.rows) *(u2 *)(out + 32 * b) = (u2){out_pair(p.q_bf16, v[0], v[1]), out_pair(p.q_bf16, v[2], v[3])};
            } else {
                *(f4 *)(e + b * 256 + lane * 4) = v;
            }
        }
        if (wave == 0 && grp == 0) {
            if (!whole) e[16 * DC + col] = mj, e[16 * DC + 16 + col] = l;
            else if (p.lse && col < w.rows) p.lse[o] = row_lse(mj, l, kBias);
        }
        __syncthreads();
    }
}

// More rows: all heads of a token on one card, drafted tokens, chunks.
//
// Two groups of four waves take 64 rows each and walk the cache in steps of 32 tokens, whose rows lie in
// LDS once for all waves.  For the scores a wave has 16 rows, whose queries stay in registers, and all 32 tokens;
// p goes through LDS, and for the second product a wave has its group's 64 rows and a quarter of the
// channels.  While one group's waves make scores, the other's are at the second product, so that each SIMD
// has a wave for the softmax and one for the matrix cores.  A barrier ends each such half step: when it opens,
// what one group leaves in LDS for itself is there, and so are the rows that are needed next.  SPLIT: both groups
// take the same 64 rows, and every other step each; they join at an item's end.  Else 128 rows.
// TWO, for float16 outputs: what p's float16 leave over follows as bytes, five bits of exponent and two of mantissa (the
// upper halves of float16; 4 KB, where LDS has no 8 left), and the values are read again for it.  p is then off by
// 2^-14 of itself, and outputs by their own rounding, 2.05e-4 of the norm (2.4e-4 with one float16), for 79 us
// instead of 67 (9 sequences of up to 16385 tokens, 1 to 5 query tokens of 64 heads).
// 40 sequences of up to 9001 tokens, 128 heads (41 GFLOP), bfloat16: 72 us, and 22 for the merge.  Neither MFMAs (busy 28% of
// the cycles) nor LDS (24%, no conflicts) bound it but what a half step of 32 tokens does one after
// the other: read, multiply, softmax, write p, meet.  Splitting 128 rows of so few sequences over all compute units costs
// 67 MB of partial states written and read.
template <int DC>
struct RowsForm {
    static constexpr int KS = 32, CB = DC / 64, SLOTS = 4;
    static constexpr int SLOT = 2 * Rows16<DC>::BYTES, PIECES = Rows16<DC>::PIECES, LOADS = (PIECES + 3) / 4;
    static constexpr int LDS = SLOTS * SLOT + 8 * 1024, LDS_TWO = LDS + 4 * 1024;  // the rows, p of both groups, its rest
    static_assert(4 * CB * 4 * 1024 <= SLOTS * SLOT, "a group's sums fit the buffers");
};
template <int DC, bool SPLIT, bool TWO>
__global__ __launch_bounds__(512, 2) void latent_rows_kernel(const LatentAttnParams p) {
    using F = RowsForm<DC>;
    using T = Rows16<DC>;
    constexpr int NI = Row<DC>::NI, ROWB = T::ROWB, ROWS = SPLIT ? 64 : 128, CB = F::CB, SLOTS = F::SLOTS, RB = 4;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Scan<TWO ? 0 : kThreads> sc;
    __shared__ float alphas[2][64];
    __shared__ __align__(16) int flags[2][4];
    __shared__ int miss[SLOTS][2];               // whether a tile of 16 tokens has no page
    __shared__ uint16_t offsets[T::PIECES][64];  // what a lane loads of a piece: in LDS, registers are scarce
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave >> 2, wg = wave & 3;
    const uint32_t ring = lds_addr(smem), p_ring = ring + SLOTS * F::SLOT + group * 4096, rest_ring = ring + F::LDS + group * 2048;
    for (int i = wave; i < T::PIECES; i += 8) offsets[i][threadIdx.x & 63] = (uint16_t)T::offset(i, threadIdx.x & 63);

    const int total = scan_seqs(p, sc);
    Run run = run_of(p, sc, total);
    note_join(p, run, total);
    Item it;
    while (next_item(p, sc, run, it)) {
        const Work &w = run.w;
        const int row0 = it.tile * ROWS, rows = min(ROWS, w.rows - row0), mine = (SPLIT ? 0 : 64 * group) + 16 * wg;  // the wave's first for the scores
        const int see_all = w.r.sees(p.causal, (int)fast_div(row0, p.by_heads));
        const int see_any = w.r.sees(p.causal, (int)fast_div(row0 + rows - 1, p.by_heads));
        const int key0 = it.j0 * kUnit, key1 = min(it.j1 * kUnit, see_any);
        const int steps = key1 > key0 ? (key1 - key0 + F::KS - 1) / F::KS : 0;
        const int halves = SPLIT ? steps + 1 : 2 * steps + 1;
        Pages pages{p.seqs.table + run.s * p.seqs.table_stride, p.seqs.width, 0, 0};
        auto load = [&](int t, int slot) {  // a group takes 16 of the 32 rows
            const Tile tile = tile_at(p.pool, pages, key0 + t * F::KS + 16 * group, t < steps ? w.r.kv : 0);
            const int ln = lane_again();
            if (ln == 0) miss[slot][group] = !tile.there;
            const u4 rsrc = wave_rsrc(tile.at, tile.rows * ROWB);
            const uint32_t offs = lds_addr((const unsigned char *)offsets) + 2 * ln, to = ring + slot * F::SLOT + group * T::BYTES;
            uint32_t off[F::LOADS];
            // pieces wg, wg + 4, ..; the last one again where a wave has one less, so that all count alike
#pragma unroll
            for (int i = 0; i < F::LOADS; ++i) off[i] = *lds_ptr<uint16_t>(offs + (wg + 4 * i < T::PIECES ? wg + 4 * i : wg + 4 * i - 4) * 128);
#pragma unroll
            for (int i = 0; i < F::LOADS; ++i)
                dma_kib(rsrc, __builtin_amdgcn_readfirstlane(to + (wg + 4 * i < T::PIECES ? wg + 4 * i : wg + 4 * i - 4) * 1024), off[i]);
        };
        if (steps) {
            pages.fill(key0 >> p.pool.log_page);
            load(0, 0);
            load(1, 1);
        }
        h8 Q[NI];
        float kx;
        {
            const int row = row0 + min(mine + (int)(threadIdx.x & 15), rows - 1), qt = (int)fast_div(row, p.by_heads), h = row - qt * p.H;
            Row<DC> raw;
            raw.load(p, w.r.begin + qt, h, (threadIdx.x >> 4) & 3);
            kx = query_operand(Q, raw.w, p.q_bf16, p.scale_log2);
        }
        float mx = kMinMax, l = 0.0f;
        f4 acc[RB][CB];
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int b = 0; b < CB; ++b) acc[r][b] = (f4){0.f, 0.f, 0.f, 0.f};
        wait_vm<F::LOADS>();
        wait_lgkm0();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

#pragma unroll 1
        for (int i = 0; i < halves; ++i) {
            // in a group's half step without scores, the shorter one; the second group's is a step later, and so is what
            // it overwrites done with
            const bool fetch = SPLIT || ((i ^ group) & 1);
            if (fetch) load(SPLIT ? i + 2 : (i >> 1) + 2, (SPLIT ? i + 2 : (i >> 1) + 2) & (SLOTS - 1));
            const int lane = lane_again(), col = lane & 15, grp = lane >> 4;
            const bool scores = ((i ^ group) & 1) == 0;
            const int t = SPLIT ? (scores ? i : i - 1) : ((scores ? i : i - 1) - group) >> 1;
            if (t >= 0 && t < steps) {
                const uint32_t at = ring + (t & (SLOTS - 1)) * F::SLOT, p_at = p_ring + lane * 16;
                if (scores) {
                    const uint32_t ka = at + col * ROWB + ((grp ^ turn(col)) << 4), kb = ka ^ 64;
                    constexpr int READS = 2 * NI, AHEAD = 4;  // reads that are under way
                    f4 S[2] = {};
                    h8 K[AHEAD];
                    auto key = [&](int n) {
                        const int c = n >> 1;
                        return __builtin_bit_cast(h8, *lds_ptr<u4>((c & 1 ? kb : ka) + (n & 1) * T::BYTES + (c >> 1) * 128));
                    };
#pragma unroll
                    for (int n = 0; n < AHEAD; ++n) K[n] = key(n);
                    const int gone = miss[t & (SLOTS - 1)][0] | miss[t & (SLOTS - 1)][1] << 1;
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int n = 0; n < READS; ++n) {
                        S[n & 1] = mfma_k32(K[n % AHEAD], Q[n >> 1], S[n & 1]);
                        if (n + AHEAD < READS) K[n % AHEAD] = key(n + AHEAD);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    const int first = key0 + t * F::KS, lost = __builtin_amdgcn_readfirstlane(gone);
                    if (first + F::KS > see_all || lost) {
                        const int see = w.r.sees(p.causal, (int)fast_div(row0 + min(mine + col, rows - 1), p.by_heads));
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (first + 16 * k + 4 * grp + e >= see || (lost >> k & 1)) S[k][e] = -INFINITY;
                    }
                    float top = S[0][0];
#pragma unroll
                    for (int e = 1; e < 8; ++e) top = __builtin_fmaxf(top, S[e >> 2][e & 3]);
                    float alpha = 1.0f;
                    const bool over = __builtin_amdgcn_ballot_w64(__builtin_fmaf(top, kx, kBias - mx) > kBias + kLagBy) != 0;
                    if (over) {
                        top = qmax(top);
                        const float mn = __builtin_fmaf(top, kx, kBias - mx) > kBias ? running_max(top, kx, kBias) : mx;
                        alpha = __builtin_amdgcn_exp2f(mx - mn);
                        l *= alpha;
                        mx = mn;
                        if (grp == 0) alphas[group][16 * wg + col] = alpha;
                    } else if (grp == 0) {
                        alphas[group][16 * wg + col] = 1.0f;
                    }
                    if (lane == 0) flags[group][wg] = over;
                    u4 P;
                    u2 rest;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float e[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) e[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[k][q], kx, kBias - mx));
                        l += (e[0] + e[1]) + (e[2] + e[3]);
                        int bytes = 0;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const h2 high = {(_Float16)e[2 * q], (_Float16)e[2 * q + 1]};
                            P[2 * k + q] = as_u32(high);
                            if constexpr (TWO) {
                                const float x = e[2 * q] - (float)high[0], y = e[2 * q + 1] - (float)high[1];
                                bytes = q ? __builtin_amdgcn_cvt_pk_bf8_f32(x, y, bytes, true) : __builtin_amdgcn_cvt_pk_bf8_f32(x, y, bytes, false);
                            }
                        }
                        rest[k] = (uint32_t)bytes;
                    }
                    if constexpr (TWO) *lds_mut<u2>(rest_ring + lane * 8 + wg * 512) = rest;
                    *lds_mut<u4>(p_at + wg * 1024) = P;
                } else {
                    const int vrow = 4 * grp + (col >> 2);
                    const uint32_t va = at + vrow * ROWB + ((((col & 3) >> 1) ^ turn(vrow)) << 4) + 8 * (col & 1);
                    constexpr int AHEAD = 2;
                    h8 V[AHEAD], P[RB];
                    auto value = [&](int b) {
                        const int c = wg * CB + b;
                        const uint32_t x = (va ^ (32 * (c & 3))) + (c >> 2) * 128;
                        const u2 lo = read_transposed(x), hi = read_transposed(x + T::BYTES);
                        return __builtin_bit_cast(h8, (u4){lo[0], lo[1], hi[0], hi[1]});
                    };
                    const u4 f = *(const u4 *)flags[group];
#pragma unroll
                    for (int r = 0; r < RB; ++r) P[r] = __builtin_bit_cast(h8, *lds_ptr<u4>(p_at + r * 1024));
#pragma unroll
                    for (int b = 0; b < AHEAD; ++b) V[b] = value(b);
                    if (__builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3])) {
#pragma unroll
                        for (int r = 0; r < RB; ++r) {
                            const float a = alphas[group][16 * r + col];
#pragma unroll
                            for (int b = 0; b < CB; ++b) acc[r][b] *= a;
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    constexpr int READS = (TWO ? 2 : 1) * CB;  // the rest of p meets the same values
#pragma unroll
                    for (int n = 0; n < READS; ++n) {
                        const int b = n % CB;
                        if (n == CB)
#pragma unroll
                            for (int r = 0; r < RB; ++r) {  // the upper bytes of float16
                                const u2 w = *lds_ptr<u2>(rest_ring + lane * 8 + r * 512);
                                P[r] = __builtin_bit_cast(h8, (u4){__builtin_amdgcn_perm(w[0], w[0], 0x010c000cu), __builtin_amdgcn_perm(w[0], w[0], 0x030c020cu),
                                                                   __builtin_amdgcn_perm(w[1], w[1], 0x010c000cu), __builtin_amdgcn_perm(w[1], w[1], 0x030c020cu)});
                            }
#pragma unroll
                        for (int r = 0; r < RB; ++r) acc[r][b] = mfma_k32(V[n % AHEAD], P[r], acc[r][b]);
                        if (n + AHEAD < READS) V[n % AHEAD] = value((n + AHEAD) % CB);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            if (fetch) wait_vm<F::LOADS>();
            wait_lgkm0();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        wait_vm<0>();
        const int lane = lane_again(), col = lane & 15, grp = lane >> 4;
        l = qsum(l);
        // the rows' sums and maxima for all waves: in the p of the groups
        float *const sums = (float *)(smem + SLOTS * F::SLOT + group * 4096);
        if (grp == 0) sums[16 * wg + col] = l, sums[64 + 16 * wg + col] = mx;
        __syncthreads();
        if constexpr (SPLIT) {
            if (group == 1)
#pragma unroll
                for (int r = 0; r < RB; ++r)
#pragma unroll
                    for (int b = 0; b < CB; ++b) *(f4 *)(smem + ((wg * RB + r) * CB + b) * 1024 + lane * 16) = acc[r][b];
            __syncthreads();
        }
        if (!SPLIT || group == 0) {
            const bool all = it.starts && it.ends;
            const int base = SPLIT ? 0 : 64 * group;
            float *e = entry_of<DC, ROWS>(p, blockIdx.x, it.starts);
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                float lr = sums[16 * r + col], mr = sums[64 + 16 * r + col];
                if constexpr (SPLIT) {
                    const float lo = sums[1024 + 16 * r + col], mo = sums[1024 + 64 + 16 * r + col];
                    const float mn = __builtin_fmaxf(mr, mo), x = __builtin_amdgcn_exp2f(mr - mn), y = __builtin_amdgcn_exp2f(mo - mn);
                    lr = lr * x + lo * y;
                    mr = mn;
#pragma unroll
                    for (int b = 0; b < CB; ++b) {
                        const f4 o = *(const f4 *)(smem + ((wg * RB + r) * CB + b) * 1024 + lane * 16);
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[r][b][q] = __builtin_fmaf(o[q], y, acc[r][b][q] * x);
                    }
                }
                if (all) {
                    const int at = row0 + base + 16 * r + col;
                    if (at < w.rows) {
                        const float inv = row_inverse(lr);
                        const int t = (int)fast_div(at, p.by_heads);
                        const int64_t o = (int64_t)(w.r.begin + t) * p.H + (at - t * p.H);
                        unsigned char *out = (unsigned char *)p.out + o * (2 * DC) + wg * CB * 32 + 8 * grp;
#pragma unroll
                        for (int b = 0; b < CB; ++b) {
                            const f4 v = acc[r][b] * inv;
                            *(u2 *)(out + 32 * b) = (u2){out_pair(p.q_bf16, v[0], v[1]), out_pair(p.q_bf16, v[2], v[3])};
                        }
                        if (p.lse && wg == 0 && grp == 0) p.lse[o] = row_lse(mr, lr, kBias);
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < CB; ++b) *(f4 *)(e + ((base / 16 + r) * (DC / 16) + wg * CB + b) * 256 + lane * 4) = acc[r][b];
                    if (wg == 0 && grp == 0) e[ROWS * DC + base + 16 * r + col] = mr, e[ROWS * DC + ROWS + base + 16 * r + col] = lr;
                }
            }
        }
        __syncthreads();
    }
}

// Joins the partial states of items that several workgroups share.  Every run but the first that begins inside an item
// has workgroups here, and the runs of an item divide its parts, two 16-channel blocks of 16 rows each: there are at most
// 255 such runs, whatever sequences and rows a call has.  Each of a workgroup's waves takes every fourth state.
// Bound by the states' bytes where they are many (22 us for 128 rows of 40 sequences: 67 MB), else by its loads'
// chain (4.0 us for one of 517 tokens).
template <int DC, int ROWS>
__global__ __launch_bounds__(kThreads) void latent_merge_kernel(const LatentAttnParams p) {
    constexpr int NB = DC / 16, PER = 2, SPLIT = NB / PER, PARTS = ROWS / 16 * SPLIT;
    __shared__ __align__(16) f4 sums[kWaves][PER][64];
    __shared__ float ms[kWaves][16], ls[kWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const LatentJoin j = p.joins[blockIdx.y + 1];
    const int g0 = j.g0, g1 = j.g1, nth = (int)blockIdx.y - g0;
    for (int part = nth * (int)gridDim.x + (int)blockIdx.x; part < PARTS; part += (g1 - g0) * (int)gridDim.x) {
        const int r = part / SPLIT, b0 = part % SPLIT * PER;
        if (j.row0 + 16 * r >= j.rows) return;  // (also where there is no item: rows 0)
        float m = kMinMax;
        for (int g = g0 + wave + kWaves * grp; g <= g1; g += 4 * kWaves)
            m = __builtin_fmaxf(m, entry_of<DC, ROWS>(p, g, g == g0)[ROWS * DC + 16 * r + col]);
        m = qmax(m);
        float l = 0.0f;
        f4 acc[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int g = g0 + wave; g <= g1; g += kWaves) {
            const float *e = entry_of<DC, ROWS>(p, g, g == g0);
            const float a = __builtin_amdgcn_exp2f(e[ROWS * DC + 16 * r + col] - m);
            l += e[ROWS * DC + ROWS + 16 * r + col] * a;
#pragma unroll
            for (int i = 0; i < PER; ++i) acc[i] += *(const f4 *)(e + (r * NB + b0 + i) * 256 + lane * 4) * a;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) sums[wave][i][lane] = acc[i];
        if (grp == 0) ms[wave][col] = m, ls[wave][col] = l;
        __syncthreads();
        const int row = j.row0 + 16 * r + col;
        if (wave < PER && row < j.rows) {
            float mx = ms[0][col];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) mx = __builtin_fmaxf(mx, ms[i][col]);
            f4 o = {0.f, 0.f, 0.f, 0.f};
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                const float a = __builtin_amdgcn_exp2f(ms[i][col] - mx);
                l += ls[i][col] * a;
                o += sums[i][wave][lane] * a;
            }
            const int qt = (int)fast_div(row, p.by_heads), h = row - qt * p.H;
            const int64_t at = (int64_t)(j.begin + qt) * p.H + h;
            o *= row_inverse(l);
            *(u2 *)((unsigned char *)p.out + at * (2 * DC) + 32 * (b0 + wave) + 8 * grp) =
                (u2){out_pair(p.q_bf16, o[0], o[1]), out_pair(p.q_bf16, o[2], o[3])};
            if (p.lse && grp == 0 && b0 + wave == 0) p.lse[at] = row_lse(mx, l, kBias);
        }
        __syncthreads();
    }
}

// The importance: sum over rows and heads of 2^(s - lse), for 32 tokens a wave, whose rows stay in
// registers while query rows go through LDS as the other operand.
//
// Up to 16 rows a sequence: bound by the cache's bytes (8 sequences of up to 31744 tokens, 16 heads, 93 MB: 23 us).
template <int DC>
__global__ __launch_bounds__(kThreads, 1) void latent_importance_few_kernel(const LatentImportanceParams p) {
    constexpr int NI = Row<DC>::NI, W = DC + kLatentRope, CH = W / 8, ROWB = 2 * W, MINE = (CH + 15) / 16;
    __shared__ __align__(16) u4 op[NI * 64];
    __shared__ float kxs[16], ls[16];
    __shared__ int sees[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const int s = blockIdx.y;
    const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_page));
    const int n = min(r.n, p.seqs.max_q), win = p.q_window > 0 ? min(p.q_window, n) : n;
    const int64_t block0 = (int64_t)blockIdx.x * (kWaves * 32);
    const int64_t lim = min((int64_t)r.kv, p.n_scores);
    const bool live = n > 0 && block0 < lim;
    const int64_t tok0 = block0 + wave * 32;
    // the token whose score this lane writes
    const int64_t mine = tok0 + 4 * (col & 4) + 4 * grp + (col & 3);
    const bool writes = col < 8 && mine < p.n_scores;
    float *out = p.out + s * p.out_stride;
    const float *old = p.scores + s * p.score_stride;
    float sum[2][4] = {};
    bool have[2] = {false, false};
    float before = 0.0f;
    if (live) {
        const int rows = win * p.H;
        // 16 lanes stage a row
        const int sr = threadIdx.x >> 4, sl = threadIdx.x & 15;
        u4 w[MINE];
        float lse_in = 0.0f;
        int see_in = 0;
        {
            const int i = min(sr, rows - 1), qt = (int)fast_div(i, p.by_heads), h = i - qt * p.H;
            const int64_t t = r.begin + n - win + qt;
            const unsigned char *q = p.q + t * p.q_t + h * p.q_h, *qr = p.qr + t * p.qr_t + h * p.qr_h;
#pragma unroll
            for (int j = 0; j < MINE; ++j) {
                const int c = sl + 16 * j;
                w[j] = (u4){0, 0, 0, 0};
                if (c < CH) w[j] = c < DC / 8 ? ((const u4 *)q)[c] : ((const u4 *)qr)[c - DC / 8];
            }
            lse_in = p.lse[t * p.H + h];
            see_in = sr < rows ? r.sees(p.causal, n - win + qt) : 0;
        }
        h8 K[2][NI];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t t = tok0 + 16 * i;
            uint32_t page = ~0u;
            if (t < lim) page = (uint32_t)p.seqs.table[s * p.seqs.table_stride + (t >> p.pool.log_page)];
            have[i] = page < p.pool.n_pages;
            const unsigned char *at = p.pool.base + (int64_t)(have[i] ? page : 0) * p.pool.page_bytes +
                                      (have[i] ? (t & ((1 << p.pool.log_page) - 1)) : 0) * ROWB + col * ROWB + 16 * grp;
#pragma unroll
            for (int c = 0; c < NI; ++c) K[i][c] = p.pool.n_pages ? *(const h8 *)(at + 64 * c) : (h8){};
        }
        if (writes) before = old[mine];
        int ex = 14;
        if (p.q_bf16) {
            const us2 pair = largest(w);
            uint32_t top = max(pair[0], pair[1]);
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
            ex = row_exponent(top);
            const float x = __builtin_ldexpf(1.0f, 14 - ex);
#pragma unroll
            for (int j = 0; j < MINE; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[j][e] = scaled_pair(w[j][e], x);
        }
        // chunk c of row sr lies at place sr ^ 4 (c % 4) of the sixteen of the chunk: writes and reads fall on all banks
#pragma unroll
        for (int j = 0; j < MINE; ++j) {
            const int c = sl + 16 * j;
            if (c < CH) op[c * 16 + (sr ^ 4 * (c & 3))] = w[j];
        }
        if (sl == 0) {
            kxs[sr] = row_factor(p.scale_log2, ex);
            ls[sr] = lse_in * 1.4426950408889634f;
            sees[sr] = see_in;
        }
        __syncthreads();
        f4 S[2] = {};
#pragma unroll
        for (int c = 0; c < NI; ++c) {
            const h8 q = __builtin_bit_cast(h8, op[c * 64 + grp * 16 + (col ^ 4 * grp)]);
#pragma unroll
            for (int i = 0; i < 2; ++i) S[i] = mfma_k32(K[i][c], q, S[i]);
        }
        const float kx = kxs[col], lse = ls[col];
        const int see = sees[col];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i][e], kx, -lse));
                sum[i][e] = tok0 + 16 * i + 4 * grp + e < see ? v : 0.0f;
            }
    } else if (writes) before = old[mine];
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) sum[i][e] += __shfl_xor(sum[i][e], d);
            v = col == 4 * i + e ? sum[i][e] : v;
        }
    if (writes) {
        if (n > 0 && mine < lim) out[mine] = __builtin_fmaf(before, p.decay, (col < 4 ? have[0] : have[1]) ? v / (float)p.H : 0.0f);
        else if (out + mine != old + mine) out[mine] = before;
    }
}

// For more rows.  First every query row is made an operand once: blocks of 16 rows as the lanes read them, then
// the rows' factors, log-sums and how many tokens they see.  They come in pairs, what lacks sees none.
template <int DC>
struct QueryBlock {
    static constexpr int NI = Row<DC>::NI, BYTES = (NI + 1) * 1024;
};
__device__ __forceinline__ int64_t first_block(const LatentImportanceParams &p, const SeqRows &r, int s) {
    return (p.q_window > 0 ? (int64_t)s * min(p.q_window, p.seqs.max_q) : (int64_t)r.begin) * p.H / 16 + 3 * s;
}
template <int DC>
__global__ __launch_bounds__(kThreads) void latent_importance_queries_kernel(const LatentImportanceParams p) {
    using B = QueryBlock<DC>;
    constexpr int CH = (DC + kLatentRope) / 8, MINE = (CH + 15) / 16;
    const int s = blockIdx.y, b = blockIdx.x, sr = threadIdx.x >> 4, sl = threadIdx.x & 15;
    const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_page));
    const int n = min(r.n, p.seqs.max_q), win = p.q_window > 0 ? min(p.q_window, n) : n, rows = win * p.H;
    if (16 * (b & ~1) >= rows) return;
    const int row = 16 * b + sr, i = min(row, rows - 1), qt = (int)fast_div(i, p.by_heads), h = i - qt * p.H;
    const int64_t t = r.begin + n - win + qt;
    const unsigned char *q = p.q + t * p.q_t + h * p.q_h, *qr = p.qr + t * p.qr_t + h * p.qr_h;
    u4 w[MINE];
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        const int c = sl + 16 * j;
        w[j] = (u4){0, 0, 0, 0};
        if (c < CH) w[j] = c < DC / 8 ? ((const u4 *)q)[c] : ((const u4 *)qr)[c - DC / 8];
    }
    int ex = 14;
    if (p.q_bf16) {
        const us2 pair = largest(w);
        uint32_t top = max(pair[0], pair[1]);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        ex = row_exponent(top);
        const float x = __builtin_ldexpf(1.0f, 14 - ex);
#pragma unroll
        for (int j = 0; j < MINE; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[j][e] = scaled_pair(w[j][e], x);
    }
    unsigned char *to = p.blocks + (first_block(p, r, s) + b) * B::BYTES;
#pragma unroll
    for (int j = 0; j < MINE; ++j)
        if (const int c = sl + 16 * j; c < CH) ((u4 *)to)[c * 16 + sr] = w[j];
    if (sl == 0) {
        float *of = (float *)(to + B::NI * 1024);
        of[sr] = row_factor(p.scale_log2, ex);
        of[16 + sr] = p.lse[t * p.H + h] * 1.4426950408889634f;
        ((int *)of)[32 + sr] = row < rows ? r.sees(p.causal, n - win + qt) : 0;
    }
}

// Then a workgroup takes 128 tokens, two waves of a SIMD the same 32 and every other block; buffer loads
// bring pairs of blocks three steps ahead.  2 sequences of up to 16384 tokens, 32 query tokens of 64 heads: 7 and 77 us,
// of which the products alone, with nothing to load, are 50 (every workgroup making its own operands: 120).
template <int DC>
__global__ __launch_bounds__(2 * kThreads, 2) void latent_importance_rows_kernel(const LatentImportanceParams p) {
    using B = QueryBlock<DC>;
    constexpr int NI = B::NI, ROWB = 2 * (DC + kLatentRope), SLOTS = 4, SLOT = 2 * B::BYTES;
    constexpr int PIECES = SLOT / 1024, LOADS = (PIECES + 7) / 8;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float joined[2][kWaves][32];
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all & 3, group = all >> 2;
    const int col = lane & 15, grp = lane >> 4;
    const int s = blockIdx.y;
    const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_page));
    const int n = min(r.n, p.seqs.max_q), win = p.q_window > 0 ? min(p.q_window, n) : n;
    const int64_t block0 = (int64_t)blockIdx.x * (kWaves * 32);
    const int64_t lim = min((int64_t)r.kv, p.n_scores);
    const bool live = n > 0 && block0 < lim;
    const int64_t tok0 = block0 + wave * 32;
    // the token whose score this lane writes
    const int64_t mine = tok0 + 4 * (col & 4) + 4 * grp + (col & 3);
    const bool writes = group == 0 && col < 8 && mine < p.n_scores;
    float *out = p.out + s * p.out_stride;
    const float *old = p.scores + s * p.score_stride;
    float sum[2][4] = {};
    bool have[2] = {false, false};
    float before = 0.0f;
    if (writes) before = old[mine];
    if (live) {
        h8 K[2][NI];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t t = tok0 + 16 * i;
            uint32_t page = ~0u;
            if (t < lim) page = (uint32_t)p.seqs.table[s * p.seqs.table_stride + (t >> p.pool.log_page)];
            have[i] = page < p.pool.n_pages;
            const unsigned char *at = p.pool.base + (int64_t)(have[i] ? page : 0) * p.pool.page_bytes +
                                      (have[i] ? (t & ((1 << p.pool.log_page) - 1)) : 0) * ROWB + col * ROWB + 16 * grp;
#pragma unroll
            for (int c = 0; c < NI; ++c) K[i][c] = p.pool.n_pages ? *(const h8 *)(at + 64 * c) : (h8){};
        }
        const int steps = (win * p.H + 31) / 32;
        const unsigned char *from = p.blocks + first_block(p, r, s) * B::BYTES;
        const uint32_t ring = lds_addr(smem);
        auto load = [&](int b) {
            const u4 rsrc = wave_rsrc(from + (int64_t)b * SLOT, b < steps ? SLOT : 0);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                // (the last one again where a wave has one less, so that all count alike)
                const int k = all + 8 * i < PIECES ? all + 8 * i : all + 8 * i - 8;
                dma_kib(rsrc, __builtin_amdgcn_readfirstlane(ring + (b & (SLOTS - 1)) * SLOT + k * 1024), lane * 16 + k * 1024);
            }
        };
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < NI; ++c) asm volatile("" : "+v"(K[i][c]));  // waited for here, not in the loop
#pragma unroll
        for (int b = 0; b < SLOTS - 1; ++b) load(b);
#pragma unroll 1
        for (int b = 0; b < steps; ++b) {
            wait_vm<(SLOTS - 2) * LOADS>();
            wait_lgkm0();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            load(b + SLOTS - 1);
            constexpr int AHEAD = 6;  // reads that are under way
            const uint32_t at = ring + (b & (SLOTS - 1)) * SLOT + group * B::BYTES, of = at + NI * 1024 + col * 4;
            auto query = [&](int c) { return __builtin_bit_cast(h8, *lds_ptr<u4>(at + lane * 16 + c * 1024)); };
            f4 S[2] = {};
            h8 Q[AHEAD];
#pragma unroll
            for (int c = 0; c < AHEAD; ++c) Q[c] = query(c);
            const float kx = *lds_ptr<float>(of), lse = *lds_ptr<float>(of + 64);
            const int see = *lds_ptr<int>(of + 128);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < NI; ++c) {
#pragma unroll
                for (int i = 0; i < 2; ++i) S[i] = mfma_k32(K[i][c], Q[c % AHEAD], S[i]);
                if (c + AHEAD < NI) Q[c % AHEAD] = query(c + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
            const int left = (int)(see - tok0) - 4 * grp;  // of this lane's tokens, counted from its first
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i][e], kx, -lse));
                    sum[i][e] += 16 * i + e < left ? v : 0.0f;
                }
        }
        wait_vm<0>();
    }
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) sum[i][e] += __shfl_xor(sum[i][e], d);
            v = col == 4 * i + e ? sum[i][e] : v;
        }
    if (col < 8) joined[group][wave][8 * grp + col] = v;
    __syncthreads();
    if (!writes) return;
    v = joined[0][wave][8 * grp + col] + joined[1][wave][8 * grp + col];
    if (n > 0 && mine < lim) out[mine] = __builtin_fmaf(before, p.decay, (col < 4 ? have[0] : have[1]) ? v / (float)p.H : 0.0f);
    else if (out + mine != old + mine) out[mine] = before;
}

namespace {
constexpr int64_t kJoinBytes = kGroups * (int64_t)sizeof(LatentJoin);
}  // namespace

int64_t latent_attn_plan(LatentAttnParams *p) {
    const int64_t rows = (int64_t)p->seqs.max_q * p->H;
    // tiles of 16 rows, 64 or 128: 40 sequences of up to 9001 tokens take 47 us as one of 16 and 63 as one of 64
    // with 16 heads, 64 us as one of 64 and 70 as one of 128 with 32 heads, 66 and 73 with 64
    p->log_tile = rows <= 16 ? 4 : rows <= 64 ? 6 : 7;
    const int64_t units = (((int64_t)p->seqs.width << p->pool.log_page) + kUnit - 1) / kUnit + 1 + kSetup;
    const int64_t tiles = (rows + (1 << p->log_tile) - 1) >> p->log_tile;
    p->groups = (int)std::max<int64_t>(1, std::min<int64_t>(kGroups, units * tiles * p->seqs.n_seqs));
    p->by_heads = make_fast_div((uint32_t)p->H);
    p->by_groups = make_fast_div((uint32_t)p->groups);
    return kJoinBytes + ((int64_t)p->groups * 2 * (p->Dc + 2) * 4 << p->log_tile);
}

hipError_t latent_attn_launch(const LatentAttnParams &p0, hipStream_t st) {
    LatentAttnParams p = p0;
    if (p.seqs.n_seqs == 0 || p.seqs.max_q == 0) return hipSuccess;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    p.part = (float *)((unsigned char *)p.joins + kJoinBytes);
    auto go = [&](auto kern, auto merge, int threads, int lds) {
        (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        kern<<<dim3(p.groups), dim3(threads), lds, st>>>(p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.groups == 1) return e;
        const int parts = (p.Dc / 32) << (p.log_tile - 4);
        merge<<<dim3(std::min(32, parts / 2), p.groups - 1), dim3(kThreads), 0, st>>>(p);
        return hipGetLastError();
    };
    auto of = [&](auto dc) {
        constexpr int DC = decltype(dc)::value;
        using F = RowsForm<DC>;
        const int few = 2 * kWaves * Rows16<DC>::BYTES;
        if (p.log_tile == 4 && p.q_bf16) return go(latent_few_kernel<DC, false>, latent_merge_kernel<DC, 16>, kThreads, few);
        if (p.log_tile == 4) return go(latent_few_kernel<DC, true>, latent_merge_kernel<DC, 16>, kThreads, few);
        if (p.q_bf16) {
            if (p.log_tile == 6) return go(latent_rows_kernel<DC, true, false>, latent_merge_kernel<DC, 64>, 512, F::LDS);
            return go(latent_rows_kernel<DC, false, false>, latent_merge_kernel<DC, 128>, 512, F::LDS);
        }
        if (p.log_tile == 6) return go(latent_rows_kernel<DC, true, true>, latent_merge_kernel<DC, 64>, 512, F::LDS_TWO);
        return go(latent_rows_kernel<DC, false, true>, latent_merge_kernel<DC, 128>, 512, F::LDS_TWO);
    };
    return p.Dc == 512 ? of(std::integral_constant<int, 512>{}) : of(std::integral_constant<int, 256>{});
}

static int64_t importance_rows(const LatentImportanceParams &p) {  // of a sequence, at most
    return (int64_t)(p.q_window > 0 ? std::min(p.q_window, p.seqs.max_q) : p.seqs.max_q) * p.H;
}
int64_t latent_importance_plan(LatentImportanceParams *p) {
    p->by_heads = make_fast_div((uint32_t)p->H);
    if (importance_rows(*p) <= 16) return 0;
    const int64_t rows = p->q_window > 0 ? p->seqs.n_seqs * importance_rows(*p) : p->seqs.n_tokens * p->H;
    return (rows / 16 + 3 * (p->seqs.n_seqs + 1)) * (p->Dc == 512 ? QueryBlock<512>::BYTES : QueryBlock<256>::BYTES);
}

hipError_t latent_importance_launch(const LatentImportanceParams &p0, hipStream_t st) {
    LatentImportanceParams p = p0;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    const dim3 grid((unsigned)((p.n_scores + kWaves * 32 - 1) / (kWaves * 32)), p.seqs.n_seqs);
    const int64_t rows = importance_rows(p);
    auto of = [&](auto dc) {
        constexpr int DC = decltype(dc)::value;
        // (16 rows of 8 sequences of up to 31744 tokens: 23 us here, 5 + 46 below, which has half the tokens under way)
        if (rows <= 16) {
            latent_importance_few_kernel<DC><<<grid, dim3(kThreads), 0, st>>>(p);
            return hipGetLastError();
        }
        latent_importance_queries_kernel<DC><<<dim3((unsigned)((rows + 31) / 32 * 2), p.seqs.n_seqs), dim3(kThreads), 0, st>>>(p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        auto kernel = latent_importance_rows_kernel<DC>;
        const int lds = 8 * QueryBlock<DC>::BYTES;
        (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        kernel<<<grid, dim3(2 * kThreads), lds, st>>>(p);
        return hipGetLastError();
    };
    return p.Dc == 512 ? of(std::integral_constant<int, 512>{}) : of(std::integral_constant<int, 256>{});
}

}  // namespace akv
