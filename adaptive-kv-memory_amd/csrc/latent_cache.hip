// The paged latent cache's data movement: append (rounded into slots), read, and the compaction of
// sequences to the tokens that stay.  All of it is bound by memory.
//
// Eight lanes take a token: lane i of them the 16-byte pieces i, i + 8, .. of its row, of which the last
// is the rotated key's.  A row that holds a value that is not finite is kept as latents 0 and a rotated key of
// NaN: its score is NaN in every row that sees it, and 0 times its value 0 in those that do not.
#include <algorithm>

#include "akv_common.h"
#include "latent.h"
#include "paged_device.h"

namespace akv {
namespace {

constexpr float kTop = 61440.0f;  // appended values are clamped to this
constexpr uint32_t kNaN2 = 0x7e007e00u;

__device__ __forceinline__ bool any_of_eight(bool x) {  // of a token's lanes
    return (__builtin_amdgcn_ballot_w64(x) >> (threadIdx.x & 56) & 0xff) != 0;
}

// The row of token t, null if it has no slot.
__device__ __forceinline__ unsigned char *slot_of(const LatentRowsParams &p, int t, bool live) {
    const int s = seq_of(p.seqs, t, live);
    if (s < 0) return nullptr;
    const SeqRows r = seq_rows(p.seqs, s, p.pool.log_page);
    const int64_t pos = (int64_t)r.at + (t - r.begin);
    if (t < r.begin || t >= r.begin + r.n || pos < 0 || pos >> p.pool.log_page >= p.seqs.width) return nullptr;
    const uint32_t page = (uint32_t)p.seqs.table[s * p.seqs.table_stride + (pos >> p.pool.log_page)];
    if (page >= p.pool.n_pages) return nullptr;
    return p.pool.base + page * p.pool.page_bytes + (pos & ((1 << p.pool.log_page) - 1)) * p.pool.row_bytes;
}

template <int DT>
struct Eight {  // eight values as they come
    u4 a, b;
    __device__ __forceinline__ void load(const unsigned char *p) {
        a = *(const u4 *)p;
        if constexpr (DT == AKV_DT_F32) b = ((const u4 *)p)[1];
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (DT == AKV_DT_F32) return __builtin_bit_cast(float, (uint32_t)(i < 4 ? a[i & 3] : b[i & 3]));
        const uint32_t w = a[i >> 1];
        if constexpr (DT == AKV_DT_F16) return (float)as_h2(w)[i & 1];
        return __builtin_bit_cast(float, i & 1 ? w & 0xffff0000u : w << 16);
    }
};

}  // namespace

// 33800 float32 tokens of 576 channels (117 MB in and out): 24 us, 4.9 TB/s; the smallest calls 3 us, a launch and
// the chain from the row's sequence to its page.
template <int DC, int DT>
__global__ __launch_bounds__(256) void latent_append_kernel(const LatentRowsParams p) {
    constexpr int N = (DC + kLatentRope) / 64, E = DT == AKV_DT_F32 ? 32 : 16;
    const int i = threadIdx.x & 7;
    const int64_t first = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    const int last = (int)p.seqs.n_tokens - 1;
    const bool live = first <= last;
    const int t = live ? (int)first : last;
    unsigned char *row = slot_of(p, t, live);
    Eight<DT> x[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
        x[j].load(j < N - 1 ? p.latent + t * p.latent_t + (8 * j + i) * E : p.rope + t * p.rope_t + i * E);
    u4 w[N];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float a = x[j].at(2 * q), b = x[j].at(2 * q + 1);
            bad |= !(__builtin_fabsf(a) < INFINITY) | !(__builtin_fabsf(b) < INFINITY);
            w[j][q] = as_u32((h2){(_Float16)__builtin_amdgcn_fmed3f(a, -kTop, kTop), (_Float16)__builtin_amdgcn_fmed3f(b, -kTop, kTop)});
        }
    bad = any_of_eight(bad);
    if (!row) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (bad)
#pragma unroll
            for (int q = 0; q < 4; ++q) w[j][q] = j < N - 1 ? 0u : kNaN2;
        *(u4 *)(row + (8 * j + i) * 16) = w[j];
    }
}

// The same tokens to float16 (78 MB): 13 us, in part from the cache behind L2.
template <int DC, int DT>
__global__ __launch_bounds__(256) void latent_read_kernel(const LatentRowsParams p) {
    constexpr int N = (DC + kLatentRope) / 64, E = DT == AKV_DT_F32 ? 32 : 16;
    const int i = threadIdx.x & 7;
    const int64_t first = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    const int last = (int)p.seqs.n_tokens - 1;
    const bool live = first <= last;
    const int t = live ? (int)first : last;
    const unsigned char *row = slot_of(p, t, live);
    u4 w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = row ? *(const u4 *)(row + (8 * j + i) * 16) : (u4){0, 0, 0, 0};
    const bool bad = any_of_eight((w[N - 1][0] & 0x7fffu) > 0x7c00u);
    if (!live) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = bad ? __builtin_nanf("") : (float)as_h2(w[j][q >> 1])[q & 1];
        unsigned char *to = j < N - 1 ? p.latent + t * p.latent_t + (8 * j + i) * E : p.rope + t * p.rope_t + i * E;
        if constexpr (DT == AKV_DT_F32) {
            ((f4 *)to)[0] = (f4){x[0], x[1], x[2], x[3]};
            ((f4 *)to)[1] = (f4){x[4], x[5], x[6], x[7]};
        } else {
            u4 o;
#pragma unroll
            for (int q = 0; q < 4; ++q) o[q] = to_pair(DT == AKV_DT_BF16, x[2 * q], x[2 * q + 1]);
            *(u4 *)to = o;
        }
    }
}

// z: layer, y: sequence, x: 32 tokens of it.  6 sequences to 8192 tokens each in 8 layers (0.8 GB): 160 us, 5.1 TB/s.
template <int N>
__global__ __launch_bounds__(256) void latent_compact_kernel(const LatentCompactParams p) {
    const int s = blockIdx.y, i = threadIdx.x & 7;
    const int64_t j = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    const int log_page = p.pool.log_page, in_page = (1 << log_page) - 1;
    int64_t n = p.n_keep[s];
    const int64_t cap = (int64_t)p.dst_width << log_page;
    n = n > p.max_keep ? p.max_keep : n;
    n = n > cap ? cap : n;
    if (j >= n) return;
    const int64_t pos = p.keep[s * p.keep_stride + j];
    if (pos < 0 || pos >= ((int64_t)p.src_width << log_page)) return;
    const uint32_t from = (uint32_t)p.src_table[s * p.src_stride + (pos >> log_page)];
    const uint32_t to = (uint32_t)p.dst_table[s * p.dst_stride + (j >> log_page)];
    if (from >= p.pool.n_pages || to >= p.pool.n_pages) return;
    unsigned char *base = p.pool.base + blockIdx.z * p.layer_bytes + i * 16;
    const unsigned char *src = base + from * p.pool.page_bytes + (pos & in_page) * (128 * N);
    unsigned char *dst = base + to * p.pool.page_bytes + (j & in_page) * (128 * N);
    if (src == dst) return;
    u4 w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = *(const u4 *)(src + 128 * k);
#pragma unroll
    for (int k = 0; k < N; ++k) *(u4 *)(dst + 128 * k) = w[k];
}

namespace {
template <typename Go>
hipError_t by_type(const LatentRowsParams &p, Go go) {
    auto of = [&](auto dc) {
        constexpr int DC = decltype(dc)::value;
        if (p.dt == AKV_DT_F16) go(std::integral_constant<int, DC>{}, std::integral_constant<int, AKV_DT_F16>{});
        else if (p.dt == AKV_DT_BF16) go(std::integral_constant<int, DC>{}, std::integral_constant<int, AKV_DT_BF16>{});
        else go(std::integral_constant<int, DC>{}, std::integral_constant<int, AKV_DT_F32>{});
    };
    if (p.Dc == 512) of(std::integral_constant<int, 512>{});
    else of(std::integral_constant<int, 256>{});
    return hipGetLastError();
}
}  // namespace

hipError_t latent_append_launch(const LatentRowsParams &p, hipStream_t s) {
    if (p.seqs.n_tokens == 0 || p.seqs.n_seqs == 0) return hipSuccess;
    const dim3 grid((unsigned)((p.seqs.n_tokens + 31) / 32));
    return by_type(p, [&](auto dc, auto dt) {
        latent_append_kernel<decltype(dc)::value, decltype(dt)::value><<<grid, dim3(256), 0, s>>>(p);
    });
}
hipError_t latent_read_launch(const LatentRowsParams &p, hipStream_t s) {
    if (p.seqs.n_tokens == 0) return hipSuccess;
    const dim3 grid((unsigned)((p.seqs.n_tokens + 31) / 32));
    return by_type(p, [&](auto dc, auto dt) {
        latent_read_kernel<decltype(dc)::value, decltype(dt)::value><<<grid, dim3(256), 0, s>>>(p);
    });
}

hipError_t latent_compact_launch(const LatentCompactParams &p, hipStream_t s) {
    if (p.max_keep == 0 || p.n_seqs == 0 || p.layers == 0) return hipSuccess;
    const dim3 grid((unsigned)((p.max_keep + 31) / 32), (unsigned)p.n_seqs, (unsigned)p.layers);
    if (p.pool.row_bytes == 1152) latent_compact_kernel<9><<<grid, dim3(256), 0, s>>>(p);
    else latent_compact_kernel<5><<<grid, dim3(256), 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace akv
