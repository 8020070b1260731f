// Parameter blocks and device views of the paged 4-bit cache (akv_paged_* of akv_hip.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "akv_hip.h"

namespace akv {

constexpr int kTileTok = 16;   // tokens of a tile
constexpr int kUnitTok = 32;   // tokens a wave of the attention takes at a time: two tiles
constexpr int kRows = 16;      // query rows (tokens x heads of a group) that a wave takes
// Sequences of more rows a cached head go to the tile kernel: a chunk of 16 rows costs a compute
// unit 0.7 us for 64 tokens, a tile of up to 256 rows 2 us.  Chunks against a tile, us, 48, 64 and 80
// rows: 16 sequences of 8192 tokens and 8 heads, bfloat16: 120, 143, 168 against 152, 148, 151;
// float16: 129, 165, 199 against 164, 164, 172; one of 32768: 43, 50, 57 against 76, 76, 79 and
// 48, 56, 65 against 78, 79, 83.
constexpr int kFewRows = 64;
// The same for the importance, by the rows that a call's sequences may have.  16 rows a wave
// against 128 a workgroup, us: two sequences of 12000 tokens and 8 heads, 128, 256 and 2048 rows: 40,
// 72, 502 against 38, 60, 362 (in bfloat16 33 against 37 at 128); one of 2000: 28, 50, 412 against
// 25, 40, 229.
constexpr int kFewWindowRows = 128;

__host__ __device__ constexpr int paged_tile_bytes(int D, int ng) { return 16 * D + 128 * ng; }

// One layer of a pool as a kernel sees it.
struct PagedView {
    unsigned char *base;       // the layer's first page
    int64_t page_bytes;        // every head of a page
    uint32_t n_pages;
    int heads, log_tpp;        // log2 of the tiles a page has of one head
};

struct PagedSeqs {
    const int32_t *table, *kv_lens, *q_starts;
    int64_t table_stride, n_tokens;
    int n_seqs, width, max_q;
};

struct PagedRowsParams {
    PagedView pool;
    PagedSeqs seqs;
    int D, ng, dt;
    int log_lanes;             // log2 of a group's lanes, eight channels each
    unsigned char *k, *v;
    int64_t k_t, k_h, v_t, v_h;
};

struct PagedAttnParams {
    PagedView pool;
    PagedSeqs seqs;
    int D, ng, Hq, g;          // g = Hq / heads
    int q_bf16, causal;
    float scale_log2;          // sm_scale * log2(e)
    const unsigned char *q;
    int64_t q_t, q_h;
    void *out;
    float *lse;
    float *part;               // the workspace; in the kernels, partial states of items that several workgroups share
    float *tile_part;          // the same of the tile kernel
    int *sums;                 // first units of the sequences
    int groups, tile_groups;   // workgroups of the two kernels
    int few_rows;              // the tile kernel takes sequences of more rows
    int rows;                  // most rows of an item
    int whole;                 // > 0: every item counts this many units and is a workgroup's
};

struct PagedImportanceParams {
    PagedView pool;
    PagedSeqs seqs;
    int D, ng, Hq, g;
    int q_bf16, causal, q_window;
    float scale_log2, decay;
    const unsigned char *q;
    int64_t q_t, q_h;
    const float *lse, *scores;
    float *out;
    int64_t n_scores, score_stride, out_stride;
    int head_split;            // waves that share a run of tokens, each with its heads
    int head_lds, blocks;      // most heads of a wave; runs of a wave (a decode step's)
};

struct PagedCopyParams {
    unsigned char *data;
    int64_t page_bytes, n_pages, n;
    int layers;
    const int32_t *src, *dst;
};

struct PagedCompactParams {
    PagedView pool;            // layer 0
    int64_t layer_bytes;
    int layers, D, ng, n_seqs;
    const int32_t *src_table, *dst_table;
    int64_t src_stride, dst_stride;
    int src_width, dst_width;
    const int32_t *keep, *n_keep;
    int64_t keep_stride, max_keep;
};

hipError_t paged_append_launch(const PagedRowsParams &p, hipStream_t s);
hipError_t paged_read_launch(const PagedRowsParams &p, hipStream_t s);
hipError_t paged_copy_launch(const PagedCopyParams &p, hipStream_t s);
hipError_t paged_compact_launch(const PagedCompactParams &p, hipStream_t s);
// Sets the launch's sizes and the parts of the workspace; its bytes.
int64_t paged_attn_plan(PagedAttnParams *p);
hipError_t paged_attn_launch(const PagedAttnParams &p, hipStream_t s);
int64_t paged_tile_plan(PagedAttnParams *p);
hipError_t paged_tile_launch(const PagedAttnParams &p, hipStream_t s);
hipError_t paged_importance_launch(const PagedImportanceParams &p, hipStream_t s);
hipError_t paged_importance_tile_launch(const PagedImportanceParams &p, hipStream_t s);

#ifdef __HIPCC__
// Rows [begin, begin + n) of sequence s in the call's tensors, its cached tokens that have a slot, and
// the first row's place (of a sequence that outgrew its table they are not kv's last ones).
struct SeqRows {
    int begin, n, kv, at;
    // Tokens that row i sees.
    __device__ __forceinline__ int sees(int causal, int i) const { return causal ? min(max(at + i + 1, 0), kv) : kv; }
};
// The same of a sequence that is one for the whole wave, in scalar registers.
__device__ __forceinline__ SeqRows wave_uniform(const SeqRows &r) {
    return {__builtin_amdgcn_readfirstlane(r.begin), __builtin_amdgcn_readfirstlane(r.n), __builtin_amdgcn_readfirstlane(r.kv),
            __builtin_amdgcn_readfirstlane(r.at)};
}
__device__ __forceinline__ SeqRows seq_rows(const PagedSeqs &q, int s, int log_page) {
    const int64_t lim = q.n_tokens;
    int64_t a = q.q_starts[s], b = q.q_starts[s + 1];
    a = a < 0 ? 0 : a > lim ? lim : a;
    b = b < a ? a : b > lim ? lim : b;
    const int64_t cap = (int64_t)q.width << log_page;
    const int64_t len = q.kv_lens[s] < 0 ? 0 : q.kv_lens[s];
    return {(int)a, (int)(b - a), (int)(len > cap ? cap : len), (int)(len - (b - a))};
}
#endif

}  // namespace akv
