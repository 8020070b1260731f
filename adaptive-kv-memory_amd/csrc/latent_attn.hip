// Attention over the paged latent cache in its absorbed form, its merge, and the importance of
// cached tokens.
//
// The mathematics.  The heads' key matrices are in the queries already, so a cached row (latent c,
// rotated key r) is the key of every head and its latent the value: s = q.c + q_r.r, o = sum of p c.
// The rows of all heads and query tokens of a sequence thus share one stream of cached rows.  A query
// row is scaled by a power of two to a maximum in [2^13, 2^14), which leaves with the softmax scale,
// and enters as float16 whatever its type; scores are exact but for float32 sums.  p is one float16.
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
constexpr int kSetup = 2;             // units that an item's start counts
constexpr int kGroups = 256;          // one workgroup a compute unit

// A row's query operand: lane (row, quarter grp) holds channels 32 i + 8 grp .. of latent and rope.
template <int DC>
struct Row {
    static constexpr int NI = (DC + kLatentRope) / 32;
    u4 w[NI];
    __device__ __forceinline__ void load(const unsigned char *q, const unsigned char *qr, int grp) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            w[i] = i < DC / 32 ? *(const u4 *)(q + 64 * i + 16 * grp) : *(const u4 *)(qr + 64 * (i - DC / 32) + 16 * grp);
    }
    __device__ __forceinline__ float make(h8 (&op)[NI], bool bf16, float scale_log2) const {
        return scaled_row(op, [&](int i, int e) { return query_value(w[i], e, bf16); }, scale_log2);
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
    w.tiles = (w.rows + p.row_tile - 1) / p.row_tile;
    w.cost = max(1, (r.kv + kUnit - 1) / kUnit) + kSetup;
    return w;
}

struct Scan {
    int pre[kThreads + 1];
    int wave_sum[kWaves];
};
// pre[i]: the first unit of sequence i * per, pre[256] the total.  For workgroups of 256 threads or more.
__device__ __forceinline__ void scan_seqs(const LatentAttnParams &p, Scan &sc, int per) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int mine = 0, inc = 0;
    if (t < kThreads) {
        for (int i = 0; i < per; ++i) {
            const int s = t * per + i;
            if (s < p.seqs.n_seqs) {
                const Work w = seq_work(p, seq_rows(p.seqs, s, p.pool.log_page));
                mine += w.tiles * w.cost;
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
        int before = 0;
        for (int w = 0; w < wave; ++w) before += sc.wave_sum[w];
        sc.pre[t] = before + inc - mine;
        if (t == kThreads - 1) sc.pre[kThreads] = before + inc;
    }
    __syncthreads();
}
__device__ __forceinline__ int share_of(int total, int groups) { return max(1, (total + groups - 1) / groups); }

// A run of units as items: whole or partial (sequence, tile of rows).
struct Run {
    int x, x_end, s, off;
    Work w;
};
struct Item {
    int tile, j0, j1;
    bool starts, ends;
};
__device__ __forceinline__ Run run_of(const LatentAttnParams &p, Scan &sc) {
    const int lane = threadIdx.x & 63, per = (p.seqs.n_seqs + kThreads - 1) / kThreads;
    const int total = __builtin_amdgcn_readfirstlane(sc.pre[kThreads]);
    const int share = share_of(total, p.groups);
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
        r.w = seq_work(p, wave_uniform(seq_rows(p.seqs, r.s, p.pool.log_page)));
        const int n = r.w.tiles * r.w.cost;
        if (r.off < n) break;
        r.off -= n;
        ++r.s;
    }
    return r;
}
// The next item's part of the run; false at the end.
__device__ __forceinline__ bool next_item(const LatentAttnParams &p, Run &r, Item &it) {
    if (r.x >= r.x_end) return false;
    while (r.off == r.w.tiles * r.w.cost) {
        r.off = 0;
        r.w = seq_work(p, wave_uniform(seq_rows(p.seqs, ++r.s, p.pool.log_page)));
    }
    it.tile = r.off / r.w.cost;
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
__device__ __forceinline__ void keep_sums(const LatentAttnParams &p, const Scan &sc) {  // for the merge
    if (blockIdx.x == 0 && threadIdx.x <= kThreads) {
        p.sums[threadIdx.x] = sc.pre[threadIdx.x];
        if (threadIdx.x == 0) p.sums[kThreads] = sc.pre[kThreads];
    }
}

}  // namespace

// Up to 16 rows a sequence (a token's heads).  Bound by the cache's bytes.
//
// Each of the four waves takes 16 tokens at a time for all 16 rows, from two buffers of LDS of its own
// that buffer loads fill; nothing is shared until the waves join at an item's end.
template <int DC>
__global__ __launch_bounds__(kThreads, 1) void latent_few_kernel(const LatentAttnParams p) {
    using T = Rows16<DC>;
    constexpr int NI = Row<DC>::NI, NB = DC / 16, ROWB = T::ROWB, SLOTS = 2;
    constexpr int STATE = NB * 1024 + 512;  // bytes of a wave's state on its way to another
    static_assert(2 * STATE <= kWaves * SLOTS * T::BYTES, "the joins fit");
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Scan sc;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const uint32_t ring = __builtin_amdgcn_readfirstlane(lds_addr(smem) + wave * SLOTS * T::BYTES);

    uint32_t voff[T::PIECES];
#pragma unroll
    for (int i = 0; i < T::PIECES; ++i) voff[i] = T::offset(i, lane);
    const uint32_t k_at = col * ROWB + ((grp ^ turn(col)) << 4);
    const int vrow = 4 * grp + (col >> 2);
    const uint32_t v_at = vrow * ROWB + ((((col & 3) >> 1) ^ turn(vrow)) << 4) + 8 * (col & 1);

    scan_seqs(p, sc, (p.seqs.n_seqs + kThreads - 1) / kThreads);
    keep_sums(p, sc);
    Run run = run_of(p, sc);
    Item it;
    while (next_item(p, run, it)) {
        const Work &w = run.w;
        const int row = min(col, w.rows - 1), qt = row / p.H, h = row - qt * p.H;
        const int see = w.r.sees(p.causal, qt), see_all = w.r.sees(p.causal, 0), see_any = w.r.sees(p.causal, (w.rows - 1) / p.H);
        const int key0 = it.j0 * kUnit, key1 = min(it.j1 * kUnit, see_any);
        const int steps = key1 > key0 ? (key1 - key0 + 16 * kWaves - 1) / (16 * kWaves) : 0;
        Row<DC> raw;
        raw.load(p.q + (w.r.begin + qt) * p.q_t + h * p.q_h, p.qr + (w.r.begin + qt) * p.qr_t + h * p.qr_h, grp);
        Pages pages{p.seqs.table + run.s * p.seqs.table_stride, p.seqs.width, 0, 0};
        bool there[SLOTS] = {};
        auto load = [&](int t, int slot) {
            const int k = key0 + (t * kWaves + wave) * 16;
            const Tile tile = tile_at(p.pool, pages, k, t < steps ? w.r.kv : 0);
            there[slot] = tile.there;
            const u4 rsrc = wave_rsrc(tile.at, tile.rows * ROWB);
#pragma unroll
            for (int i = 0; i < T::PIECES; ++i) dma_kib(rsrc, ring + slot * T::BYTES + i * 1024, voff[i]);
        };
        if (steps) {
            pages.fill(key0 >> p.pool.log_page);
            load(0, 0);
            load(1, 1);
        }
        h8 Q[NI];
        const float kx = raw.make(Q, p.q_bf16, p.scale_log2);
        float mx = kMinMax, l = 0.0f;
        f4 acc[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = (f4){0.f, 0.f, 0.f, 0.f};

        auto step = [&](int t, int slot) {
            wait_vm<T::PIECES>();  // the next step's rows are still on their way
            const uint32_t at = ring + slot * T::BYTES;
            const int first = key0 + (t * kWaves + wave) * 16;
            f4 S2[2] = {};
            const uint32_t ka = at + k_at, kb = ka ^ 64;
#pragma unroll
            for (int c = 0; c < NI; ++c)
                S2[c & 1] = mfma_k32(__builtin_bit_cast(h8, *lds_ptr<u4>((c & 1 ? kb : ka) + (c >> 1) * 128)), Q[c], S2[c & 1]);
            f4 S = S2[0] + S2[1];
            if (!(first + 16 <= see_all && there[slot]))
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (first + 4 * grp + e >= see || !there[slot]) S[e] = -INFINITY;
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
            const h4 P = {(_Float16)e[0], (_Float16)e[1], (_Float16)e[2], (_Float16)e[3]};  // 2^-12 of a weight
            const uint32_t va = at + v_at;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                acc[b] = mfma_k16(__builtin_bit_cast(h4, read_transposed((va ^ (32 * (b & 3))) + (b >> 2) * 128)), P, acc[b]);
            wait_lgkm0();
            asm volatile("" ::: "memory");
            load(t + SLOTS, slot);
        };
        for (int t = 0; t < steps; t += 2) {
            step(t, 0);
            if (t + 1 < steps) step(t + 1, 1);
        }
        wait_vm<0>();

        l = qsum(l);
#pragma unroll
        for (int n = kWaves / 2; n >= 1; n >>= 1) {
            __syncthreads();
            unsigned char *place = smem + (wave & (n - 1)) * STATE;
            float *ml = (float *)(place + NB * 1024);
            if (wave >= n && wave < 2 * n) {
#pragma unroll
                for (int b = 0; b < NB; ++b) *(f4 *)(place + b * 1024 + lane * 16) = acc[b];
                ml[lane] = mx, ml[64 + lane] = l;
            }
            __syncthreads();
            if (wave < n) {
                const float mo = ml[lane], lo = ml[64 + lane], mn = __builtin_fmaxf(mx, mo);
                const float a = __builtin_amdgcn_exp2f(mx - mn), c = __builtin_amdgcn_exp2f(mo - mn);
                l = l * a + lo * c;
                mx = mn;
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] = acc[b] * a + *(const f4 *)(place + b * 1024 + lane * 16) * c;
            }
        }
        if (wave == 0) {
            if (it.starts && it.ends) {
                const float inv = row_inverse(l);
                if (col < w.rows) {
                    const int64_t o = (int64_t)(w.r.begin + qt) * p.H + h;
                    unsigned char *out = (unsigned char *)p.out + o * (2 * DC) + 8 * grp;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const f4 v = acc[b] * inv;
                        *(u2 *)(out + 32 * b) = (u2){to_pair(p.q_bf16, v[0], v[1]), to_pair(p.q_bf16, v[2], v[3])};
                    }
                    if (p.lse && grp == 0) p.lse[o] = row_lse(mx, l, kBias);
                }
            } else {
                float *e = entry_of<DC, 16>(p, blockIdx.x, it.starts);
#pragma unroll
                for (int b = 0; b < NB; ++b) *(f4 *)(e + b * 256 + lane * 4) = acc[b];
                if (grp == 0) e[16 * DC + col] = mx, e[16 * DC + 16 + col] = l;
            }
        }
        __syncthreads();
    }
}

// More rows: all heads of a token on one card, drafted tokens, chunks.
//
// A workgroup of NW waves takes 16 RB rows and walks the cache in steps of 32 tokens, whose rows lie in
// LDS once for all waves.  For the scores a wave has 16 rows (and half of the tokens, where there are fewer row
// blocks than waves), whose queries stay in registers; p goes through LDS, and for the second product a
// wave has all rows and its share of the channels, so that the sums of 128 rows x 512 channels fit the
// registers of eight waves and a value is read from LDS by one wave only.  One barrier a step: when it opens, p and
// the factors of this step are there, the next step's rows are too, and the step before is read by all.
template <int DC, int RB>
struct RowsForm {
    static constexpr int NW = RB == 2 ? 4 : 8, KW = NW / RB, KS = 32, KT = 2 / KW;
    static constexpr int ROWS = 16 * RB, CB = DC / 16 / NW, SLOTS = RB == 8 ? 3 : 4;
    static constexpr int SLOT = 2 * Rows16<DC>::BYTES, PIECES = 2 * Rows16<DC>::PIECES, LOADS = (PIECES + NW - 1) / NW;
    static constexpr int LDS = SLOTS * SLOT + 2 * RB * 1024;
};
template <int DC, int RB>
__global__ __launch_bounds__((RB == 2 ? 256 : 512), (RB == 2 ? 1 : 2)) void latent_rows_kernel(const LatentAttnParams p) {
    using F = RowsForm<DC, RB>;
    using T = Rows16<DC>;
    constexpr int NI = Row<DC>::NI, ROWB = T::ROWB, ROWS = F::ROWS, NW = F::NW, KW = F::KW, KT = F::KT, CB = F::CB, SLOTS = F::SLOTS;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Scan sc;
    __shared__ float alphas[2][ROWS], tops[2][2][ROWS];  // (tops: the waves that share rows; at the end the sums)
    __shared__ int flags[2][8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int rbw = wave % RB, kw = wave / RB;
    const uint32_t ring = lds_addr(smem), p_at = ring + SLOTS * F::SLOT;

    uint32_t voff[F::LOADS];  // pieces wave, wave + NW, ..: of the first tile of 16 rows, then the second
#pragma unroll
    for (int i = 0; i < F::LOADS; ++i) {
        int n = wave + NW * i;
        if (n >= F::PIECES) n -= NW;  // the last one again, so that all waves count alike
        voff[i] = T::offset(n % T::PIECES, lane);
    }
    const uint32_t k_at = kw * T::BYTES + col * ROWB + ((grp ^ turn(col)) << 4);
    const int vrow = 4 * grp + (col >> 2);
    const uint32_t v_at = vrow * ROWB + ((((col & 3) >> 1) ^ turn(vrow)) << 4) + 8 * (col & 1);

    scan_seqs(p, sc, (p.seqs.n_seqs + kThreads - 1) / kThreads);
    keep_sums(p, sc);
    Run run = run_of(p, sc);
    Item it;
    while (next_item(p, run, it)) {
        const Work &w = run.w;
        const int row0 = it.tile * ROWS, rows = min(ROWS, w.rows - row0);
        const int row = row0 + min(16 * rbw + col, rows - 1), qt = row / p.H, h = row - qt * p.H;
        const int see = w.r.sees(p.causal, qt), see_all = w.r.sees(p.causal, row0 / p.H);
        const int see_any = w.r.sees(p.causal, (row0 + rows - 1) / p.H);
        const int key0 = it.j0 * kUnit, key1 = min(it.j1 * kUnit, see_any);
        const int steps = key1 > key0 ? (key1 - key0 + F::KS - 1) / F::KS : 0;
        h8 Q[NI];
        float kx;
        {
            Row<DC> raw;
            raw.load(p.q + (w.r.begin + qt) * p.q_t + h * p.q_h, p.qr + (w.r.begin + qt) * p.qr_t + h * p.qr_h, grp);
            kx = raw.make(Q, p.q_bf16, p.scale_log2);
        }
        Pages pages{p.seqs.table + run.s * p.seqs.table_stride, p.seqs.width, 0, 0};
        uint32_t there = 0;  // bits 2 slot ..
        auto load = [&](int t, int slot) {
            const int k = key0 + t * F::KS, kv = t < steps ? w.r.kv : 0;
            const Tile a = tile_at(p.pool, pages, k, kv), b = tile_at(p.pool, pages, k + 16, kv);
            there = (there & ~(3u << 2 * slot)) | ((uint32_t)a.there | (uint32_t)b.there << 1) << 2 * slot;
            const u4 ra = wave_rsrc(a.at, a.rows * ROWB), rb = wave_rsrc(b.at, b.rows * ROWB);
#pragma unroll
            for (int i = 0; i < F::LOADS; ++i) {
                int n = wave + NW * i;
                if (n >= F::PIECES) n -= NW;
                dma_kib(n < T::PIECES ? ra : rb, __builtin_amdgcn_readfirstlane(ring + slot * F::SLOT + n * 1024), voff[i]);
            }
        };
        if (steps) {
            pages.fill(key0 >> p.pool.log_page);
#pragma unroll
            for (int t = 0; t < SLOTS - 1; ++t) load(t, t);
        }
        float mx = kMinMax, l = 0.0f;
        f4 acc[RB][CB];
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int b = 0; b < CB; ++b) acc[r][b] = (f4){0.f, 0.f, 0.f, 0.f};
        wait_vm<(SLOTS - 2) * F::LOADS>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

        int slot = 0, ahead = SLOTS - 1;
        for (int t = 0; t < steps; ++t) {
            const int buf = t & 1;
            const uint32_t at = ring + slot * F::SLOT;
            f4 S[2] = {};  // of two tiles, or of one in two parts
            const uint32_t ka = at + k_at, kb = ka ^ 64;
#pragma unroll
            for (int c = 0; c < NI; ++c)
#pragma unroll
                for (int i = 0; i < KT; ++i) {
                    const h8 k = __builtin_bit_cast(h8, *lds_ptr<u4>((c & 1 ? kb : ka) + i * T::BYTES + (c >> 1) * 128));
                    f4 &x = S[KT == 2 ? i : c & 1];
                    x = mfma_k32(k, Q[c], x);
                }
            if constexpr (KT == 1) S[0] = S[0] + S[1];
            const int first = key0 + t * F::KS + 16 * kw;
            const uint32_t have = there >> (2 * slot + kw) & ((1u << KT) - 1);
            if (!(first + 16 * KT <= see_all && have == (1u << KT) - 1))
#pragma unroll
                for (int i = 0; i < KT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (first + 16 * i + 4 * grp + e >= see || !(have >> i & 1)) S[i][e] = -INFINITY;
            float top = S[0][0];
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = __builtin_fmaxf(top, S[i][e]);
            if constexpr (KW == 2) {  // the rows' other tokens
                top = qmax(top);
                if (grp == 0) tops[buf][kw][16 * rbw + col] = top;
                wait_lgkm0();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                top = __builtin_fmaxf(top, tops[buf][kw ^ 1][16 * rbw + col]);
            }
            float alpha = 1.0f;
            const bool over = __builtin_amdgcn_ballot_w64(__builtin_fmaf(top, kx, kBias - mx) > kBias + kLagBy) != 0;
            if (over) {
                if constexpr (KW == 1) top = qmax(top);
                const float mn = __builtin_fmaf(top, kx, kBias - mx) > kBias ? running_max(top, kx, kBias) : mx;
                alpha = __builtin_amdgcn_exp2f(mx - mn);
                l *= alpha;
                mx = mn;
            }
            if (grp == 0) alphas[buf][16 * rbw + col] = alpha;
            if (lane == 0) flags[buf][wave] = over;
            u4 P;
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                float e[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) e[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i][q], kx, kBias - mx));
                l += (e[0] + e[1]) + (e[2] + e[3]);
                P[2 * i] = as_u32((h2){(_Float16)e[0], (_Float16)e[1]});
                P[2 * i + 1] = as_u32((h2){(_Float16)e[2], (_Float16)e[3]});
            }
            unsigned char *pw = smem + SLOTS * F::SLOT + (buf * RB + rbw) * 1024 + lane * 16;
            if constexpr (KT == 2) *(u4 *)pw = P;
            else *(u2 *)(pw + 8 * kw) = (u2){P[0], P[1]};
            wait_vm<(SLOTS - 3) * F::LOADS>();
            wait_lgkm0();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            load(t + SLOTS - 1, ahead);
            int any = 0;
#pragma unroll
            for (int i = 0; i < NW; ++i) any |= flags[buf][i];
            if (__builtin_amdgcn_readfirstlane(any)) {
#pragma unroll
                for (int r = 0; r < RB; ++r) {
                    const float a = alphas[buf][16 * r + col];
#pragma unroll
                    for (int b = 0; b < CB; ++b) acc[r][b] *= a;
                }
            }
            const uint32_t va = at + v_at;
            h8 V[CB];
#pragma unroll
            for (int b = 0; b < CB; ++b) {
                const int c = wave * CB + b;
                const uint32_t x = (va ^ (32 * (c & 3))) + (c >> 2) * 128;
                const u2 lo = read_transposed(x), hi = read_transposed(x + T::BYTES);
                V[b] = __builtin_bit_cast(h8, (u4){lo[0], lo[1], hi[0], hi[1]});
            }
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                const h8 pr = __builtin_bit_cast(h8, *lds_ptr<u4>(p_at + (buf * RB + r) * 1024 + lane * 16));
#pragma unroll
                for (int b = 0; b < CB; ++b) acc[r][b] = mfma_k32(V[b], pr, acc[r][b]);
            }
            slot = slot + 1 == SLOTS ? 0 : slot + 1;
            ahead = ahead + 1 == SLOTS ? 0 : ahead + 1;
        }
        wait_vm<0>();
        __syncthreads();
        l = qsum(l);
        if (grp == 0) tops[0][kw][16 * rbw + col] = l, tops[1][kw][16 * rbw + col] = mx;
        __syncthreads();
        const bool all = it.starts && it.ends;
        float *e = entry_of<DC, ROWS>(p, blockIdx.x, it.starts);
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            float lr = tops[0][0][16 * r + col];
            if constexpr (KW == 2) lr += tops[0][1][16 * r + col];
            const float mr = tops[1][0][16 * r + col];
            if (all) {
                const int at = row0 + 16 * r + col;
                if (at < w.rows) {
                    const float inv = row_inverse(lr);
                    const int t = at / p.H;
                    const int64_t o = (int64_t)(w.r.begin + t) * p.H + (at - t * p.H);
                    unsigned char *out = (unsigned char *)p.out + o * (2 * DC) + wave * CB * 32 + 8 * grp;
#pragma unroll
                    for (int b = 0; b < CB; ++b) {
                        const f4 v = acc[r][b] * inv;
                        *(u2 *)(out + 32 * b) = (u2){to_pair(p.q_bf16, v[0], v[1]), to_pair(p.q_bf16, v[2], v[3])};
                    }
                    if (p.lse && wave == 0 && grp == 0) p.lse[o] = row_lse(mr, lr, kBias);
                }
            } else {
#pragma unroll
                for (int b = 0; b < CB; ++b) *(f4 *)(e + (r * (DC / 16) + wave * CB + b) * 256 + lane * 4) = acc[r][b];
                if (wave == 0 && grp == 0) e[ROWS * DC + 16 * r + col] = mr, e[ROWS * DC + ROWS + 16 * r + col] = lr;
            }
        }
        __syncthreads();
    }
}

// Joins the partial states of items that several workgroups share: a wave takes four of the 16-channel
// blocks of 16 rows.
template <int DC, int ROWS>
__global__ __launch_bounds__(kThreads) void latent_merge_kernel(const LatentAttnParams p) {
    constexpr int NB = DC / 16, PER = 4, SPLIT = NB / (PER * kWaves);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const int s = blockIdx.y, part = blockIdx.x % SPLIT, block = blockIdx.x / SPLIT;
    const int tile = block / (ROWS / 16), r = block % (ROWS / 16);
    const int per = (p.seqs.n_seqs + kThreads - 1) / kThreads;
    const Work w = seq_work(p, wave_uniform(seq_rows(p.seqs, s, p.pool.log_page)));
    const int row0 = tile * ROWS + 16 * r;
    if (tile >= w.tiles || row0 >= w.rows) return;
    int start = p.sums[s / per] + tile * w.cost;
    for (int i = s / per * per; i < s; ++i) {
        const Work b = seq_work(p, wave_uniform(seq_rows(p.seqs, i, p.pool.log_page)));
        start += b.tiles * b.cost;
    }
    const int share = share_of(p.sums[kThreads], p.groups);
    // the runs that hold units of the item (its first kSetup are none)
    const int g0 = (start + kSetup) / share, g1 = (start + w.cost - 1) / share;
    if (g0 == g1) return;
    float m = kMinMax;
    for (int g = g0; g <= g1; ++g) m = __builtin_fmaxf(m, entry_of<DC, ROWS>(p, g, g == g0)[ROWS * DC + 16 * r + col]);
    float l = 0.0f;
    f4 acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = (f4){0.f, 0.f, 0.f, 0.f};
    const int b0 = (part * kWaves + wave) * PER;
#pragma unroll 2
    for (int g = g0; g <= g1; ++g) {
        const float *e = entry_of<DC, ROWS>(p, g, g == g0);
        const float a = __builtin_amdgcn_exp2f(e[ROWS * DC + 16 * r + col] - m);
        l += e[ROWS * DC + ROWS + 16 * r + col] * a;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] += *(const f4 *)(e + (r * NB + b0 + i) * 256 + lane * 4) * a;
    }
    const int row = row0 + col;
    if (row >= w.rows) return;
    const int qt = row / p.H, h = row - qt * p.H;
    const int64_t o = (int64_t)(w.r.begin + qt) * p.H + h;
    const float inv = row_inverse(l);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const f4 v = acc[i] * inv;
        *(u2 *)((unsigned char *)p.out + o * (2 * DC) + 32 * (b0 + i) + 8 * grp) =
            (u2){to_pair(p.q_bf16, v[0], v[1]), to_pair(p.q_bf16, v[2], v[3])};
    }
    if (p.lse && grp == 0 && b0 == 0) p.lse[o] = row_lse(m, l, kBias);
}

// The importance: sum over rows and heads of 2^(s - lse), for 32 tokens a wave, whose rows stay in
// registers while 16 query rows at a time go through LDS as the other operand.
template <int DC>
__global__ __launch_bounds__(kThreads, 1) void latent_importance_kernel(const LatentImportanceParams p) {
    constexpr int NI = Row<DC>::NI, W = DC + kLatentRope, CH = W / 8, ROWB = 2 * W;
    __shared__ __align__(16) u4 op[2][NI * 64];
    __shared__ float kxs[2][16], ls[2][16];
    __shared__ int sees[2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const int s = blockIdx.y;
    const SeqRows r = wave_uniform(seq_rows(p.seqs, s, p.pool.log_page));
    const int n = min(r.n, p.seqs.max_q), win = p.q_window > 0 ? min(p.q_window, n) : n;
    const int64_t block0 = (int64_t)blockIdx.x * (kWaves * 32);
    const int64_t lim = min((int64_t)r.kv, p.n_scores);
    const bool live = n > 0 && block0 < lim;
    const int64_t tok0 = block0 + wave * 32;
    h8 K[2][NI];
    bool have[2] = {false, false};
    if (live) {
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
    }
    float sum[2][4] = {};
    if (live) {
        const int rows = win * p.H, blocks = (rows + 15) / 16;
        // 16 lanes stage a row
        const int sr = threadIdx.x >> 4, sl = threadIdx.x & 15;
        constexpr int MINE = (CH + 15) / 16;
        u4 w[MINE];
        float lse_in = 0.0f;
        int see_in = 0;
        auto fetch = [&](int b) {
            const int row = 16 * b + sr, i = min(row, rows - 1);
            const int qt = n - win + i / p.H, h = i % p.H;
            const int64_t t = r.begin + qt;
            const unsigned char *q = p.q + t * p.q_t + h * p.q_h, *qr = p.qr + t * p.qr_t + h * p.qr_h;
#pragma unroll
            for (int j = 0; j < MINE; ++j) {
                const int c = sl + 16 * j;
                w[j] = (u4){0, 0, 0, 0};
                if (c < CH) w[j] = c < DC / 8 ? ((const u4 *)q)[c] : ((const u4 *)qr)[c - DC / 8];
            }
            lse_in = p.lse[t * p.H + h];
            see_in = row < rows ? r.sees(p.causal, qt) : 0;
        };
        auto stage = [&](int buf) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < MINE; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf(query_value(w[j], e, p.q_bf16)));
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, d));
            const int ex = row_exponent(top);
#pragma unroll
            for (int j = 0; j < MINE; ++j) {
                const int c = sl + 16 * j;
                h8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (_Float16)__builtin_ldexpf(query_value(w[j], e, p.q_bf16), 14 - ex);
                if (c < CH) op[buf][(c >> 2) * 64 + (c & 3) * 16 + sr] = __builtin_bit_cast(u4, v);
            }
            if (sl == 0) {
                kxs[buf][sr] = row_factor(p.scale_log2, ex);
                ls[buf][sr] = lse_in * 1.4426950408889634f;
                sees[buf][sr] = see_in;
            }
        };
        fetch(0);
        for (int b = 0; b < blocks; ++b) {
            stage(b & 1);
            __syncthreads();
            if (b + 1 < blocks) fetch(b + 1);
            f4 S[2] = {};
#pragma unroll
            for (int c = 0; c < NI; ++c) {
                const h8 q = __builtin_bit_cast(h8, op[b & 1][c * 64 + lane]);
#pragma unroll
                for (int i = 0; i < 2; ++i) S[i] = mfma_k32(K[i][c], q, S[i]);
            }
            const float kx = kxs[b & 1][col], lse = ls[b & 1][col];
            const int see = sees[b & 1][col];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i][e], kx, -lse));
                    sum[i][e] += tok0 + 16 * i + 4 * grp + e < see ? v : 0.0f;
                }
        }
    }
    float *out = p.out + s * p.out_stride;
    const float *old = p.scores + s * p.score_stride;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = sum[i][e];
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d);
            const int64_t j = tok0 + 16 * i + 4 * grp + e;
            if (col == 0 && j < p.n_scores) {
                if (n > 0 && j < lim) out[j] = __builtin_fmaf(old[j], p.decay, have[i] ? v / (float)p.H : 0.0f);
                else if (out + j != old + j) out[j] = old[j];
            }
        }
}

namespace {
constexpr int64_t kSumsBytes = 2048;
static_assert((kThreads + 1) * 4 <= kSumsBytes, "the sums fit");
}  // namespace

int64_t latent_attn_plan(LatentAttnParams *p) {
    const int64_t rows = (int64_t)p->seqs.max_q * p->H;
    p->row_tile = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    const int64_t units = (((int64_t)p->seqs.width << p->pool.log_page) + kUnit - 1) / kUnit + 1 + kSetup;
    const int64_t tiles = (rows + p->row_tile - 1) / p->row_tile;
    p->groups = (int)std::max<int64_t>(1, std::min<int64_t>(kGroups, units * tiles * p->seqs.n_seqs));
    return kSumsBytes + (int64_t)p->groups * 2 * p->row_tile * (p->Dc + 2) * 4;
}

hipError_t latent_attn_launch(const LatentAttnParams &p0, hipStream_t st) {
    LatentAttnParams p = p0;
    if (p.seqs.n_seqs == 0 || p.seqs.max_q == 0) return hipSuccess;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    p.part = (float *)((unsigned char *)p.sums + kSumsBytes);
    auto go = [&](auto kern, auto merge, int threads, int lds) {
        (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        kern<<<dim3(p.groups), dim3(threads), lds, st>>>(p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.groups == 1) return e;
        const int64_t tiles = ((int64_t)p.seqs.max_q * p.H + p.row_tile - 1) / p.row_tile;
        const dim3 grid((unsigned)(tiles * (p.row_tile / 16) * (p.Dc / 256)), p.seqs.n_seqs);
        merge<<<grid, dim3(kThreads), 0, st>>>(p);
        return hipGetLastError();
    };
    auto of = [&](auto dc) {
        constexpr int DC = decltype(dc)::value;
        auto rows = [&](auto rb) {
            constexpr int RB = decltype(rb)::value;
            using F = RowsForm<DC, RB>;
            return go(latent_rows_kernel<DC, RB>, latent_merge_kernel<DC, F::ROWS>, 64 * F::NW, F::LDS);
        };
        if (p.row_tile == 16) return go(latent_few_kernel<DC>, latent_merge_kernel<DC, 16>, kThreads, 2 * kWaves * Rows16<DC>::BYTES);
        if (p.row_tile == 32) return rows(std::integral_constant<int, 2>{});
        if (p.row_tile == 64) return rows(std::integral_constant<int, 4>{});
        return rows(std::integral_constant<int, 8>{});
    };
    return p.Dc == 512 ? of(std::integral_constant<int, 512>{}) : of(std::integral_constant<int, 256>{});
}

hipError_t latent_importance_launch(const LatentImportanceParams &p0, hipStream_t st) {
    LatentImportanceParams p = p0;
    if (p.pool.n_pages == 0) p.seqs.width = 0;
    const dim3 grid((unsigned)((p.n_scores + kWaves * 32 - 1) / (kWaves * 32)), p.seqs.n_seqs);
    if (p.Dc == 512) latent_importance_kernel<512><<<grid, dim3(kThreads), 0, st>>>(p);
    else latent_importance_kernel<256><<<grid, dim3(kThreads), 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace akv
