// Parameter blocks of the paged latent cache (akv_latent_* of akv_hip.h) and of the eviction.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "akv_hip.h"
#include "fastdiv.h"
#include "paged.h"

namespace akv {

constexpr int kLatentRope = 64;    // channels of the shared rotated key
constexpr int kLatentHead = 128;   // channels of a head's own keys, and of its values, in the expanded form

// One layer of a pool as a kernel sees it: rows of Dc + Dr float16, page_size of them a page.
struct LatentView {
    unsigned char *base;
    int64_t page_bytes;
    uint32_t n_pages;
    int log_page, row_bytes;
};

struct LatentRowsParams {
    LatentView pool;
    PagedSeqs seqs;
    int Dc, dt;
    unsigned char *latent, *rope;
    int64_t latent_t, rope_t;
};

// What the merge joins where a run begins inside an item: rows [row0, rows) of a sequence's, in the runs g0 to g1.
struct LatentJoin {
    int begin, rows, row0;
    uint16_t g0, g1;
};

struct LatentAttnParams {
    LatentView pool;
    PagedSeqs seqs;
    int Dc, H, q_bf16, causal;
    float scale_log2;          // sm_scale * log2(e)
    const unsigned char *q, *qr;
    int64_t q_t, q_h, qr_t, qr_h;
    void *out;
    float *lse;
    LatentJoin *joins;         // the workspace: one of every run, then partial states
    float *part;
    int groups, log_tile;      // workgroups, log2 of the rows of one
    FastDiv by_heads, by_groups;
};

// The expanded form: keys and values of `heads` heads at a time are made from the latents, then attended to.
struct LatentPrefillParams {
    LatentView pool;
    PagedSeqs seqs;
    int Dc, H, q_bf16, causal;
    float scale_log2;
    const unsigned char *q;
    int64_t q_t, q_h;
    void *out;                 // (n_tokens, H, kLatentHead)
    const unsigned char *w;    // [H][Dc / 32][16][64 lanes] of 16 bytes
    const float *w_scale;      // [H][2 kLatentHead]
    int64_t *sums;             // the workspace: first costs of the sequences, partial states, keys, values
    float *part;
    unsigned char *keys, *values;  // [heads][cap] rows of kLatentHead float16
    int64_t rest;              // bytes from them to what their float16 leave over; 0 for bfloat16 queries: none
    int64_t cap, seq_cap;      // rows of a head, and of a sequence in it
    int head0, heads;          // those of this pass
    int groups, rows;          // workgroups, and the attention's query tokens of one
};

struct LatentImportanceParams {
    LatentView pool;
    PagedSeqs seqs;
    int Dc, H, q_bf16, causal, q_window;
    float scale_log2, decay;
    const unsigned char *q, *qr;
    int64_t q_t, q_h, qr_t, qr_h;
    const float *lse, *scores;
    float *out;
    int64_t n_scores, score_stride, out_stride;
    FastDiv by_heads;
    unsigned char *blocks;     // the workspace, for more than 16 rows a sequence: query rows as operands
};

struct LatentCompactParams {
    LatentView pool;           // layer 0
    int64_t layer_bytes;
    int layers, n_seqs;
    const int32_t *src_table, *dst_table;
    int64_t src_stride, dst_stride;
    int src_width, dst_width;
    const int32_t *keep, *n_keep;
    int64_t keep_stride, max_keep;
};

struct EvictParams {
    const float *scores;
    int64_t n_scores, score_stride;
    const int32_t *lens, *budgets;  // budgets may be null: `budget` for all
    int64_t budget;
    int n_seqs, first, last;
    int32_t *keep, *n_keep;
    float *kept;                    // may be null
    int64_t keep_stride, max_keep, kept_stride;
};

hipError_t latent_append_launch(const LatentRowsParams &p, hipStream_t s);
hipError_t latent_read_launch(const LatentRowsParams &p, hipStream_t s);
hipError_t latent_compact_launch(const LatentCompactParams &p, hipStream_t s);
// Sets the launch's sizes; bytes of the workspace.
int64_t latent_attn_plan(LatentAttnParams *p);
hipError_t latent_attn_launch(const LatentAttnParams &p, hipStream_t s);
int64_t latent_prefill_plan(LatentPrefillParams *p);
hipError_t latent_prefill_launch(const LatentPrefillParams &p, hipStream_t s);
int64_t latent_importance_plan(LatentImportanceParams *p);
hipError_t latent_importance_launch(const LatentImportanceParams &p, hipStream_t s);
hipError_t evict_launch(const EvictParams &p, hipStream_t s);

}  // namespace akv
