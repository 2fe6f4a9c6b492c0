// serve.h — kernel parameter blocks and launches of the serving operators: the
// paged 8-bit cache (paged.hip) and row sampling (sample_rows.hip).
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

// The host's checks (paged_plan.h) have refused what a launch cannot hold.
void launch_paged_append(hipStream_t st, const PagedAppendParams &p);
void launch_paged_attention(hipStream_t st, const PagedAttnParams &p);
void launch_paged_read(hipStream_t st, const PagedReadParams &p);
void launch_sample_rows(hipStream_t st, const SampleRowsParams &p);

}  // namespace qtts
