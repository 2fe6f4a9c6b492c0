// paged_plan.h — what decides which memory the paged cache's kernels touch:
// the checks of a call's arguments, and how a kernel reads one sequence of it.
// Plain C++ without device code, so that the CPU tests run the same lines.
#pragma once

#include <cmath>
#include <cstdint>

#include "../../include/qtts.h"

#ifdef __HIPCC__
#define QTTS_HD __host__ __device__ __forceinline__
#else
#define QTTS_HD inline
#endif

namespace qtts {

// A refused call: its status and why (null: nothing wrong).
struct Refusal {
    qtts_status status;
    const char *why;
};

constexpr Refusal kAccepted{QTTS_OK, nullptr};
constexpr long long kPagedMaxBlocks = (1LL << 24) - 1;  // of one launch: its threads are counted in 32 bits
constexpr int kSampleRowsMaxVocab = 1 << 19;

inline bool aligned_to(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

inline bool paged_empty(const qtts_paged_seqs &s) { return s.batch == 0 || s.rows == 0 || s.max_rows == 0; }

// Tokens that a sequence may reach.
QTTS_HD long long tokens_cap(const qtts_paged_kv &kv, const qtts_paged_seqs &s) {
    const long long held = (long long)s.max_pages * kv.page_size;
    return s.max_tokens > 0 && s.max_tokens < held ? s.max_tokens : held;
}

inline Refusal check_paged(const qtts_paged_kv &kv, const qtts_paged_seqs &s) {
    if (kv.head_dim != 64 && kv.head_dim != 128) return {QTTS_ESHAPE, "paged cache: head_dim must be 64 or 128"};
    if (kv.page_size != 16 && kv.page_size != 32 && kv.page_size != 64 && kv.page_size != 128)
        return {QTTS_ESHAPE, "paged cache: page_size must be 16, 32, 64 or 128"};
    if (kv.num_pages < 1 || kv.kv_heads < 1 || kv.kv_heads > 1024 || kv.num_slots < 1)
        return {QTTS_ESHAPE, "paged cache: num_pages, kv_heads (to 1024) and num_slots must be positive"};
    if ((long long)kv.num_pages * kv.kv_heads > (1LL << 31) - 1)
        return {QTTS_ERANGE, "paged cache: more than 2^31 - 1 blocks (pages times kv heads)"};
    if (!kv.k_codes || !kv.v_codes || !kv.k_scales || !kv.v_scales || !kv.k_open || !kv.v_open)
        return {QTTS_EINVAL, "paged cache: null buffer"};
    if (!aligned_to(kv.k_codes, 16) || !aligned_to(kv.v_codes, 16) || !aligned_to(kv.k_open, 16) ||
        !aligned_to(kv.v_open, 16) || !aligned_to(kv.k_scales, 4) || !aligned_to(kv.v_scales, 4))
        return {QTTS_EINVAL, "paged cache: buffers must be 16-byte aligned"};
    if (s.batch < 0 || s.batch > 65536 || s.rows < 0 || s.max_rows < 0 || s.max_pages < 0 || s.max_tokens < 0)
        return {QTTS_ESHAPE,
                "paged sequences: batch must be 0..65536, rows, max_rows, max_pages and max_tokens not negative"};
    if ((long long)s.max_pages * kv.page_size > (1LL << 30))
        return {QTTS_ERANGE, "paged sequences: more than 2^30 tokens in a page table row"};
    if (paged_empty(s)) return kAccepted;
    if (s.max_rows > s.rows) return {QTTS_ESHAPE, "paged sequences: max_rows above rows"};
    if (s.rows > (1 << 30)) return {QTTS_ERANGE, "paged sequences: more than 2^30 rows"};
    if (!s.page_table && s.max_pages > 0) return {QTTS_EINVAL, "paged sequences: null page table"};
    if (!s.slots || !s.starts || !s.row_offsets) return {QTTS_EINVAL, "paged sequences: null array"};
    if (!aligned_to(s.page_table, 4) || !aligned_to(s.slots, 4) || !aligned_to(s.starts, 4) ||
        !aligned_to(s.row_offsets, 4))
        return {QTTS_EINVAL, "paged sequences: misaligned array"};
    return kAccepted;
}

// Rows of `width` floats that the kernels read or write four at a time.
inline Refusal check_rows(const float *p, int32_t ld, long long width) {
    if (!p) return {QTTS_EINVAL, "null rows"};
    if (!aligned_to(p, 16) || ld % 4 != 0) return {QTTS_EINVAL, "rows must be 16-byte aligned, strides a multiple of 4"};
    if (ld < width) return {QTTS_ESHAPE, "a row stride below the row"};
    return kAccepted;
}

inline Refusal check_heads(const qtts_paged_kv &kv, int32_t heads) {
    if (heads < 1 || heads > 1024 || heads % kv.kv_heads != 0)
        return {QTTS_ESHAPE, "heads must be a multiple of kv_heads, at most 1024"};
    return kAccepted;
}

#define QTTS_REFUSE(expr)              \
    do {                               \
        const Refusal r_ = (expr);     \
        if (r_.why) return r_;         \
    } while (0)

// Blocks of an append's sequence: K's and V's for every page that its rows touch
// at most, and a share of the query heads each.
struct AppendPlan {
    int kv_items;       // pages
    int threads;        // of a block
    long long q_items;  // blocks of query heads
    long long blocks;   // of the launch
};

inline AppendPlan append_plan(const qtts_paged_kv &kv, const qtts_paged_seqs &s, const qtts_paged_rows &r) {
    const int P = kv.page_size, lanes = kv.head_dim / 8;
    AppendPlan a;
    a.kv_items = (int)(((long long)s.max_rows + P - 2) / P + 1);
    a.threads = P * lanes < 256 ? P * lanes : 256;
    const long long fours = r.q ? (long long)s.max_rows * ((r.heads + 3) / 4) : 0;
    a.q_items = (fours + a.threads / lanes - 1) / (a.threads / lanes);
    a.blocks = s.batch * (2LL * a.kv_items * kv.kv_heads + a.q_items);
    return a;
}

inline Refusal check_append(const qtts_paged_kv &kv, const qtts_paged_seqs &s, const qtts_paged_rows &r) {
    QTTS_REFUSE(check_paged(kv, s));
    const long long hd = kv.head_dim, width = kv.kv_heads * hd;
    if (r.q) {
        QTTS_REFUSE(check_heads(kv, r.heads));
        if ((r.q_norm == nullptr) != (r.k_norm == nullptr))
            return {QTTS_EINVAL, "paged append: give both norms or neither"};
    }
    if ((r.rope_cos == nullptr) != (r.rope_sin == nullptr))
        return {QTTS_EINVAL, "paged append: give both rotation tables or neither"};
    if (r.rope_cos && (r.rope_rows < 1 || !aligned_to(r.rope_cos, 16) || !aligned_to(r.rope_sin, 16)))
        return {QTTS_EINVAL, "paged append: rotation tables must have rows and be 16-byte aligned"};
    if (!aligned_to(r.q_norm, 8) || !aligned_to(r.k_norm, 8))
        return {QTTS_EINVAL, "paged append: norms must be 8-byte aligned"};
    if (r.k_norm && !(r.eps >= 0.0f && std::isfinite(r.eps)))
        return {QTTS_EINVAL, "paged append: eps must be finite and not negative"};
    if (paged_empty(s)) return kAccepted;
    QTTS_REFUSE(check_rows(r.k, r.ld_k, width));
    QTTS_REFUSE(check_rows(r.v, r.ld_v, width));
    if (r.q) {
        QTTS_REFUSE(check_rows(r.q, r.ld_q, r.heads * hd));
        QTTS_REFUSE(check_rows(r.q_out, r.ld_q_out, r.heads * hd));
        if (r.q == r.q_out && r.ld_q != r.ld_q_out)
            return {QTTS_EINVAL, "paged append: in place, q_out takes q's stride"};
    }
    if (append_plan(kv, s, r).blocks > kPagedMaxBlocks)
        return {QTTS_ERANGE, "paged append: more blocks than a launch holds"};
    return kAccepted;
}

// How attention divides its pairs (a sequence and kv head, and column tile) over
// blocks.  Two blocks a compute unit are one round of them.  A pair takes one
// block in full rounds; the pairs of the last, incomplete round share it by
// dividing their tokens, joined through scratch of kPagedPartFloats and a counter
// each.  Smaller chunks everywhere cost more than they even out: 64 ragged
// sequences of up to 8000 tokens (512 pairs) took 160 us with one block a pair,
// 180 us with four and 204 us with eight; 4 of 32760 (32 pairs) 49 us with 16
// blocks a pair, 57 us with 32.
constexpr int kPagedRound = 512;
constexpr int kPagedMaxSplits = 256;
constexpr long long kPagedCounters = kPagedRound;
constexpr long long kPagedPartFloats = 4LL << 20;  // 3/2 of a round's blocks of 32 columns, at least

// Floats that a chunk's column takes there: its output, its reference, its sum and
// the power of two that is the sum's (one more keeps the rows on 16 bytes).
QTTS_HD constexpr int part_floats(int head_dim) { return head_dim + 4; }

struct AttnPlan {
    int whole;   // pairs of one block
    int nsplit;  // blocks of each of the others
};

// Columns (query rows of a kv head's group) that a block takes: 4 on int8
// products, 16 or 32 on binary16 ones.  Where a page's bytes are the cost, few
// columns cost as much as one: 16 sequences of 2064 tokens, 8 kv heads, took 20 us
// at up to 4 columns on int8 products (21 on the others), at 8 columns 27 us on
// int8 and 25 on binary16, at 16 columns 24 us (40 in tiles of 32).  Tiles of 32
// halve the reading of pages and the products' operands, but leave half as many
// blocks, which pays once those fill three quarters of a round: with 256 of them
// (rows of 1024 columns behind 2000 tokens) 52 us against 45 in tiles of 16, with
// 384 62 against 74, with 532 80 against 105.
enum AttnMode { kAttnI8, kAttn16, kAttn32 };

inline AttnMode attn_mode(long long columns, long long heads) {
    if (columns <= 4) return kAttnI8;
    return columns > 16 && (columns + 31) / 32 * heads >= kPagedRound * 3 / 4 ? kAttn32 : kAttn16;
}

// Tokens that a block takes at least where it shares a pair: one step of its
// waves, and with 32 columns four, as their joining costs more.
QTTS_HD constexpr int attn_least(int columns) { return columns == 32 ? 512 : 256; }

inline AttnPlan attn_plan(long long pairs, long long cap, int columns) {
    const int least = attn_least(columns);
    const long long steps = (cap + least - 1) / least, rest = pairs % kPagedRound;
    long long n = rest ? (kPagedRound + rest / 2) / rest : 1;
    n = n > steps ? steps : n;
    n = n > kPagedMaxSplits ? kPagedMaxSplits : n;
    if (n <= 1) return {(int)pairs, 1};
    return {(int)(pairs - rest), (int)n};
}

struct AttnShape {
    AttnMode mode;
    int tiles;         // of columns, a sequence and kv head's
    int whole, nsplit; // as in AttnPlan
    long long blocks;  // of the launch
};

// Tokens that a tile of 32 rows sees at most under a window and with sinks, whose
// stretches begin at multiples of 64.
inline long long seen_span(int window, int sinks) { return (long long)window + sinks + 64 + 64 + 32; }

// `span`: tokens that a tile sees at most, where the plan is to go by it (0: by what
// a sequence may reach).
inline AttnShape attn_shape(const qtts_paged_kv &kv, const qtts_paged_seqs &s, int heads, long long span = 0) {
    const long long columns = (long long)s.max_rows * (heads / kv.kv_heads), kvs = (long long)s.batch * kv.kv_heads;
    const AttnMode mode = attn_mode(columns, kvs);
    const int each = mode == kAttnI8 ? 4 : mode == kAttn16 ? 16 : 32;
    const long long tiles = (columns + each - 1) / each, pairs = kvs * tiles;
    if (pairs > kPagedMaxBlocks) return {mode, 0, 0, 0, pairs};
    const long long cap = tokens_cap(kv, s);
    const AttnPlan p = attn_plan(pairs, span > 0 && span < cap ? span : cap, each);
    return {mode, (int)tiles, p.whole, p.nsplit, p.whole + (pairs - p.whole) * p.nsplit};
}

// One for each page that a sequence's positions touch at most, and kv head.
inline int read_items(const qtts_paged_kv &kv, const qtts_paged_seqs &s) {
    return (int)(((long long)s.max_rows + kv.page_size - 2) / kv.page_size + 1);
}
inline long long read_blocks(const qtts_paged_kv &kv, const qtts_paged_seqs &s) {
    return (long long)s.batch * read_items(kv, s) * kv.kv_heads;
}

inline Refusal check_attention(const qtts_paged_kv &kv, const qtts_paged_seqs &s, int32_t heads, const float *q,
                               int32_t ld_q, float scale, int32_t window, const float *out, int32_t ld_out) {
    QTTS_REFUSE(check_paged(kv, s));
    QTTS_REFUSE(check_heads(kv, heads));
    if (window < 0) return {QTTS_EINVAL, "paged attention: window must not be negative"};
    if (!std::isfinite(scale)) return {QTTS_EINVAL, "paged attention: scale must be finite"};
    if (paged_empty(s)) return kAccepted;
    QTTS_REFUSE(check_rows(q, ld_q, (long long)heads * kv.head_dim));
    QTTS_REFUSE(check_rows(out, ld_out, (long long)heads * kv.head_dim));
    if (q == out && ld_q != ld_out) return {QTTS_EINVAL, "paged attention: in place, out takes q's stride"};
    if (attn_shape(kv, s, heads).blocks > kPagedMaxBlocks)
        return {QTTS_ERANGE, "paged attention: more blocks than a launch holds"};
    return kAccepted;
}

inline Refusal check_attention_sinks(const qtts_paged_kv &kv, const qtts_paged_seqs &s, int32_t heads, const float *q,
                                     int32_t ld_q, float scale, int32_t window, int32_t sinks, const float *out,
                                     int32_t ld_out) {
    if (sinks < 0) return {QTTS_EINVAL, "paged attention: sinks must not be negative"};
    QTTS_REFUSE(check_attention(kv, s, heads, q, ld_q, scale, window, out, ld_out));
    if (paged_empty(s) || sinks == 0 || window == 0) return kAccepted;
    if (attn_shape(kv, s, heads, seen_span(window, sinks)).blocks > kPagedMaxBlocks)
        return {QTTS_ERANGE, "paged attention: more blocks than a launch holds"};
    return kAccepted;
}

inline Refusal check_read(const qtts_paged_kv &kv, const qtts_paged_seqs &s, const int32_t *lens, const float *k_out,
                          int32_t ld_k, const float *v_out, int32_t ld_v) {
    QTTS_REFUSE(check_paged(kv, s));
    if (!aligned_to(lens, 4)) return {QTTS_EINVAL, "paged read: misaligned lens"};
    if (paged_empty(s)) return kAccepted;
    const long long width = (long long)kv.kv_heads * kv.head_dim;
    if (k_out) QTTS_REFUSE(check_rows(k_out, ld_k, width));
    if (v_out) QTTS_REFUSE(check_rows(v_out, ld_v, width));
    if (read_blocks(kv, s) > kPagedMaxBlocks) return {QTTS_ERANGE, "paged read: more blocks than a launch holds"};
    return kAccepted;
}

inline Refusal check_sample_rows(const float *logits, int64_t ld, int32_t rows, int32_t vocab,
                                 const qtts_row_sampler &p, const float *uniform, const int32_t *tokens,
                                 const float *probs) {
    if (vocab < 1 || vocab > kSampleRowsMaxVocab) return {QTTS_ESHAPE, "sample_rows: vocab must be 1..524288"};
    if (rows < 0) return {QTTS_ESHAPE, "sample_rows: rows must not be negative"};
    if (ld < vocab) return {QTTS_ESHAPE, "sample_rows: stride below the row"};
    if (rows == 0) return kAccepted;
    if (!logits || !uniform || !tokens) return {QTTS_EINVAL, "sample_rows: null argument"};
    if (!aligned_to(logits, 4) || !aligned_to(uniform, 4) || !aligned_to(tokens, 4) || !aligned_to(probs, 4) ||
        !aligned_to(p.temperature, 4) || !aligned_to(p.top_k, 4) || !aligned_to(p.top_p, 4) || !aligned_to(p.min_p, 4))
        return {QTTS_EINVAL, "sample_rows: misaligned argument"};
    return kAccepted;
}

// The tokens between the first `sinks` and a window that begins at `low`, in whole
// 64s: numbers from `edge` on are `hole` below their tokens.  No hole where the two
// meet.
struct SeenHole {
    int hole, edge;
};
QTTS_HD SeenHole seen_hole(int low, int high, int sinks) {
    const int edge = ((sinks < high ? sinks : high) + 63) & ~63, from = low & ~63;
    return {from > edge ? from - edge : 0, edge};
}

// Tokens of one block where `nsplit` share `span` tokens.
QTTS_HD int chunk_of(int span, int nsplit, int least) {
    const int each = span / nsplit + (span % nsplit != 0);
    return (each + least - 1) / least * least;
}

// One sequence of a call as the kernels see it: whatever the device arrays
// hold, rows row0 .. row0 + rows lie in the call's buffers, and where `ok`,
// positions 0 .. start + rows in the page table row and the slot in the slots.
struct PagedSeq {
    int start, rows, row0, slot;
    const int32_t *pages;
    bool ok;  // false: left out
};

QTTS_HD PagedSeq load_seq(const qtts_paged_seqs &s, int b, int num_slots, long long cap) {
    PagedSeq q;
    const int r0 = s.row_offsets[b], r1 = s.row_offsets[b + 1];
    q.row0 = r0 < 0 ? 0 : r0 > s.rows ? s.rows : r0;
    const int n = (r1 > s.rows ? s.rows : r1 < 0 ? 0 : r1) - q.row0;
    q.rows = n < 0 ? 0 : n > s.max_rows ? s.max_rows : n;
    q.start = s.starts[b];
    q.slot = s.slots[b];
    q.pages = s.page_table + (size_t)b * s.max_pages;
    q.ok = q.start >= 0 && (long long)q.start + q.rows <= cap && q.slot >= 0 && q.slot < num_slots;
    return q;
}

}  // namespace qtts
