// serve.h — kernel parameter blocks and launches of the serving operators: the
// paged 8-bit cache (paged.hip), row sampling (sample_rows.hip) and products on
// 8-bit floats (fp8.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/qtts.h"

namespace qtts {

struct PagedAppendParams {
    qtts_paged_kv kv;
    qtts_paged_seqs s;
    qtts_paged_rows r;
    int kv_items;   // pages one sequence's rows can touch
    int q_items;    // blocks over one sequence's queries
    int cap;        // tokens a sequence may reach
};

struct PagedAttnParams {
    qtts_paged_kv kv;
    qtts_paged_seqs s;
    const float *q;
    float *out;
    int heads, ld_q, ld_out;
    float scale;
    int window;
    int cap;  // tokens a sequence may reach
    // the launch's own
    int tiles;           // column tiles of one sequence and kv head
    int whole, nsplit;   // AttnPlan
    float *part;         // kPagedPartFloats: chunks' results
    unsigned *counters;  // kPagedCounters, zero between launches
};

struct PagedReadParams {
    qtts_paged_kv kv;
    qtts_paged_seqs s;
    const int32_t *lens;
    float *k_out, *v_out;
    int ld_k, ld_v;
    int cap;  // tokens a sequence may reach
};

struct SampleRowsParams {
    const float *logits;
    long long ld;
    int rows, vocab;
    qtts_row_sampler p;
    const float *u;
    int32_t *tokens;
    float *probs;
    void *scratch;         // for long rows: as many at once as it holds
    size_t scratch_bytes;
};

struct Fp8Params {
    qtts_fp8_weight w;
    const float *x, *add;
    float *y;
    int ld_x, ld_add, ld_y, rows;
    uint8_t *xc;          // kFp8ScratchBytes: rows as the products take them
    float *part;          // kFp8PartFloats: split sums
    unsigned *counters;   // kFp8Counters, zero between launches
    // the launch's own
    int kb;               // blocks of the contraction
    int tiles_n, splits, each;  // Fp8Plan; blocks of a split
};

// The host's checks (paged_plan.h, fp8_plan.h) have refused what a launch cannot hold.
void launch_paged_append(hipStream_t st, const PagedAppendParams &p);
void launch_paged_attention(hipStream_t st, const PagedAttnParams &p);
void launch_paged_read(hipStream_t st, const PagedReadParams &p);
void launch_sample_rows(hipStream_t st, const SampleRowsParams &p);
void launch_fp8_gemm(hipStream_t st, const Fp8Params &p);
void launch_fp8_quantize(hipStream_t st, const float *src, int ld_src, const qtts_fp8_weight &w);

}  // namespace qtts
