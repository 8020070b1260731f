// Eviction: which tokens of each sequence stay, by the attention that they gathered.
//
// One workgroup a sequence.  A score's bits, turned so that they order like the floats, are counted by
// their upper 11 bits, then those of the bin that the budget's border falls into by the next 11, then by
// the last 10: the border's exact value and how many of the tokens at it stay (of equal ones the lowest
// positions leave).  A second look deals the places: ballots give a token's place in its wave, a scan over
// the waves' counts the rest, so the list ascends.  Their orders stay in registers between (up to 32 a thread; longer
// sequences are read once a look).
#include <algorithm>
#include <type_traits>

#include "akv_common.h"
#include "latent.h"

namespace akv {
namespace {

constexpr int kEvictThreads = 1024, kEvictWaves = 16;

// Bits that order like the scores, above 0: NaN above all numbers (both signs alike), zeros alike.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0xfffffffeu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

struct EvictShared {
    uint32_t bins[2048];
    uint32_t counts[32 * kEvictWaves];  // of a chunk's (row of the block, wave)
    uint32_t wave_sum[kEvictWaves];
    uint32_t found, above;
};

// Exclusive sums over the workgroup of a value a thread, and the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t *wave_sum, uint32_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 63) wave_sum[wave] = inc;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kEvictWaves; ++w) {
        const uint32_t v = wave_sum[w];
        before += w < wave ? v : 0;
        total += v;
    }
    return before + inc - x;
}

}  // namespace

template <int R>
__global__ __launch_bounds__(kEvictThreads) void evict_kernel(const EvictParams p) {
    __shared__ EvictShared sh;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, s = blockIdx.x;
    const float *scores = p.scores + s * p.score_stride;
    int64_t n64 = p.lens[s];
    n64 = n64 < 0 ? 0 : n64 > p.n_scores ? p.n_scores : n64;
    int64_t k64 = p.budgets ? p.budgets[s] : p.budget;
    k64 = k64 < 0 ? 0 : k64;
    k64 = k64 > p.max_keep ? p.max_keep : k64;
    const uint32_t n = (uint32_t)n64, k = (uint32_t)(k64 < n64 ? k64 : n64);
    const uint32_t head = (uint32_t)min((int64_t)p.first, n64), tail = n - (uint32_t)min((int64_t)p.last, n64);
    const uint32_t chunks = max(1u, (n + R * kEvictThreads - 1) / (R * kEvictThreads));
    uint32_t order[R];  // 0: no token; protected ones lie above every score
    auto fetch = [&](uint32_t c) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t i = (c * R + r) * kEvictThreads + t;
            order[r] = i < n ? __builtin_bit_cast(uint32_t, scores[i]) : 0;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t i = (c * R + r) * kEvictThreads + t;
            order[r] = i >= n ? 0 : i < head || i >= tail ? 0xffffffffu : order_of(__builtin_bit_cast(float, order[r]));
        }
    };
    fetch(0);

    uint32_t border = 0, ties = 0, at_border = 0;  // the border's order, how many of those at it stay, how many there are
    if (k < n && k > 0) {
        uint32_t need = k;  // of those below what is decided
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            __syncthreads();
            sh.bins[t] = sh.bins[t + kEvictThreads] = 0;
            __syncthreads();
            for (uint32_t c = 0; c < chunks; ++c) {
                if (chunks > 1) fetch(c);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint32_t o = order[r];
                    const bool in = pass == 0 ? o != 0 : o >> (shift + bits) == border >> (shift + bits);
                    const uint64_t who = __builtin_amdgcn_ballot_w64(in);
                    if (!who) continue;
                    const uint32_t bin = o >> shift & ((1u << bits) - 1);
                    // tokens of one score are many where most have none: one count for the wave
                    const uint32_t lead = __builtin_amdgcn_readlane(bin, __builtin_ctzll(who));
                    const uint64_t same = __builtin_amdgcn_ballot_w64(in && bin == lead);
                    if (lane == (int)__builtin_ctzll(who)) atomicAdd(&sh.bins[lead], (uint32_t)__builtin_popcountll(same));
                    if (in && bin != lead) atomicAdd(&sh.bins[bin], 1u);
                }
            }
            __syncthreads();
            // from the top: the bin in which the need is met (thread t: the two bins from 2047 - 2 t down)
            const uint32_t a = sh.bins[2047 - 2 * t], b = sh.bins[2046 - 2 * t];
            uint32_t total;
            const uint32_t before = block_scan(a + b, sh.wave_sum, total);
            if (before < need && need <= before + a) sh.found = 2047 - 2 * t, sh.above = before;
            else if (before + a < need && need <= before + a + b) sh.found = 2046 - 2 * t, sh.above = before + a;
            __syncthreads();
            border |= sh.found << shift;
            need -= sh.above;
            at_border = sh.bins[sh.found];
        }
        ties = need;
    }
    // the places: above the border all, at it the last `ties` of them
    const uint32_t leave = at_border - ties;
    uint32_t ties_before = 0, kept_before = 0;
    int32_t *keep = p.keep + s * p.keep_stride;
    float *kept = p.kept ? p.kept + s * p.kept_stride : nullptr;
    for (uint32_t c = 0; c < chunks && k > 0; ++c) {
        if (chunks > 1) fetch(c);
        auto deal = [&](auto counts_of, uint32_t &before) {  // counts of every (r, wave) become places
            uint32_t mine[R];
            __syncthreads();
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint64_t who = __builtin_amdgcn_ballot_w64(counts_of(r));
                mine[r] = __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
                if (lane == 0) sh.counts[r * kEvictWaves + wave] = (uint32_t)__builtin_popcountll(who);
            }
            __syncthreads();
            const uint32_t v = t < R * kEvictWaves ? sh.counts[t] : 0;
            uint32_t total;
            const uint32_t base = block_scan(v, sh.wave_sum, total);
            if (t < R * kEvictWaves) sh.counts[t] = base;
            __syncthreads();
            struct {
                uint32_t at[R];
            } places;
#pragma unroll
            for (int r = 0; r < R; ++r) places.at[r] = before + sh.counts[r * kEvictWaves + wave] + mine[r];
            before += total;
            return places;
        };
        uint64_t stays = 0;
        if (k == n) {
#pragma unroll
            for (int r = 0; r < R; ++r) stays |= (uint64_t)(order[r] != 0) << r;
        } else {
            const auto tie = deal([&](int r) { return order[r] == border; }, ties_before);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t o = order[r];
                stays |= (uint64_t)(o > border || (o == border && tie.at[r] >= leave)) << r;
            }
        }
        const auto place = deal([&](int r) { return (stays >> r & 1) != 0; }, kept_before);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (stays >> r & 1) {
                const uint32_t i = (c * R + r) * kEvictThreads + t;
                keep[place.at[r]] = (int32_t)i;
                if (kept) kept[place.at[r]] = scores[i];
            }
    }
    for (int64_t i = k + t; i < p.max_keep; i += kEvictThreads) keep[i] = 0;
    if (kept)
        for (int64_t i = k + t; i < p.n_scores; i += kEvictThreads) kept[i] = 0.0f;
    if (t == 0) p.n_keep[s] = (int32_t)k;
}

hipError_t evict_launch(const EvictParams &p, hipStream_t s) {
    if (p.n_seqs == 0) return hipSuccess;
    const dim3 grid((unsigned)p.n_seqs), block(kEvictThreads);
    // orders a thread holds: 8 sequences of 1900 tokens take 9.3 us with 2 and 19 with 32, of 2111 11 us with 8 and
    // 18 with 32
    if (p.n_scores <= 2 * kEvictThreads) evict_kernel<2><<<grid, block, 0, s>>>(p);
    else if (p.n_scores <= 8 * kEvictThreads) evict_kernel<8><<<grid, block, 0, s>>>(p);
    else evict_kernel<32><<<grid, block, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace akv
