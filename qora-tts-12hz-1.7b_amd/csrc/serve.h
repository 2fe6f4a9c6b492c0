// serve.h — kernel parameter blocks and launches of the serving operators: the
// paged 8-bit cache (paged.hip) and its pages (pages.hip), row sampling
// (sample_rows.hip) and products on 8-bit floats (fp8.hip).
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
    int window, sinks;
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

struct RemapParams {
    qtts_paged_pool pool;
    const int32_t *source, *tokens;
    int window, sinks;
    int32_t *copied;
    int32_t *scratch;   // kPoolEntries
    unsigned *counter;  // 0 between launches
};

struct ReserveParams {
    qtts_paged_pool pool;
    const int32_t *starts, *ends;
    int32_t *lacking;
    int32_t *scratch;  // num_pages
};

struct CompactParams {
    qtts_paged_pool pool;
    int32_t *from, *to, *live;
    int32_t *scratch;  // num_pages + 1
};

struct CopyPagesParams {
    qtts_paged_kv a, b;
    const int32_t *from, *to;
};

struct CopyOpenParams {
    qtts_paged_kv kv;
    const int32_t *from, *to, *tokens;
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
    int2 *changes;        // kFp8ChangesBytes: fp8_power and the factor into its unit, for each block of the weight
    float *part;          // kFp8PartFloats: split sums
    // the launch's own
    int kb;               // blocks of the contraction
    int tiles_n, whole, splits, each;  // Fp8Plan
};

// The host's checks (paged_plan.h, pages_plan.h, fp8_plan.h) have refused what a
// launch cannot hold.
void launch_paged_append(hipStream_t st, const PagedAppendParams &p);
void launch_paged_attention(hipStream_t st, const PagedAttnParams &p);
void launch_paged_read(hipStream_t st, const PagedReadParams &p);
void launch_paged_remap(hipStream_t st, const RemapParams &p);
void launch_paged_reserve(hipStream_t st, const ReserveParams &p);
void launch_paged_compact(hipStream_t st, const CompactParams &p);
void launch_paged_copy_pages(hipStream_t st, const CopyPagesParams &p, int n);
void launch_paged_copy_open(hipStream_t st, const CopyOpenParams &p, int n);
void launch_sample_rows(hipStream_t st, const SampleRowsParams &p);
void launch_fp8_gemm(hipStream_t st, const Fp8Params &p);
void launch_fp8_quantize(hipStream_t st, const float *src, int ld_src, const qtts_fp8_weight &w);

}  // namespace qtts
