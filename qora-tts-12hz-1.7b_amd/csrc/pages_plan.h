// pages_plan.h — what decides which memory the operations on a cache's pages
// touch: the checks of a call's arguments, and which pages a row keeps.  Plain
// C++ without device code, so that the CPU tests run the same lines.
#pragma once

#include <cstdint>
#include <initializer_list>

#include "../../include/qtts.h"
#include "paged_plan.h"

namespace qtts {

constexpr int kPoolBatch = 8192;                    // rows whose slots one block hands on through LDS
constexpr long long kPoolEntries = 4LL << 20;       // of a page table: its copy lies in scratch
constexpr int kPoolPages = (4 << 20) - 64;          // names of pages, and their number, in scratch
// Entries that one block remaps in its registers, in 3.5 us; more go through scratch
// (8128 in 4.8 to 5.9 us, one block 9 to 13), from there to the table by one block or, above
// kRemapStored, in a second launch.
constexpr int kRemapThreads = 1024, kRemapEach = 2;
constexpr int kRemapStored = 16384;
// Entries that the block which finds the moves renames itself, 8192 in 2 us: with 8128
// it takes 12.5 us, with a second launch 10.4 and 4.7; with 144 6.6, or 6.2 and 1.5.
constexpr int kRenameOne = 16384;
constexpr int kPoolChunk = 16384;                   // pages that a block looks at in one go (counted in 16 bits)

inline Refusal check_pool(const qtts_paged_pool &p) {
    if (p.page_size != 16 && p.page_size != 32 && p.page_size != 64 && p.page_size != 128)
        return {QTTS_ESHAPE, "page pool: page_size must be 16, 32, 64 or 128"};
    if (p.num_pages < 1 || p.batch < 0 || p.max_pages < 0)
        return {QTTS_ESHAPE, "page pool: num_pages must be positive, batch and max_pages not negative"};
    if (p.batch > kPoolBatch) return {QTTS_ESHAPE, "page pool: batch to 8192"};
    if (p.num_pages > kPoolPages) return {QTTS_ERANGE, "page pool: more than 2^22 - 64 pages"};
    if ((long long)p.batch * p.max_pages > kPoolEntries)
        return {QTTS_ERANGE, "page pool: more than 2^22 entries in the page table"};
    if ((long long)p.max_pages * p.page_size > (1LL << 30))
        return {QTTS_ERANGE, "page pool: more than 2^30 tokens in a page table row"};
    if (!p.refs) return {QTTS_EINVAL, "page pool: null refs"};
    if (!aligned_to(p.refs, 16)) return {QTTS_EINVAL, "page pool: refs must be 16-byte aligned"};
    if (p.batch == 0) return kAccepted;
    if ((!p.page_table && p.max_pages > 0) || !p.slots) return {QTTS_EINVAL, "page pool: null array"};
    if (!aligned_to(p.page_table, 4) || !aligned_to(p.slots, 4)) return {QTTS_EINVAL, "page pool: misaligned array"};
    return kAccepted;
}

// Whether an array that a call writes is one of others.
inline bool one_of(const void *p, std::initializer_list<const void *> others) {
    for (const void *o : others)
        if (p && p == o) return true;
    return false;
}

inline Refusal check_remap(const qtts_paged_pool &p, const int32_t *source, const int32_t *tokens, int32_t window,
                           int32_t sinks, const int32_t *copied) {
    QTTS_REFUSE(check_pool(p));
    if (window < 0 || sinks < 0) return {QTTS_EINVAL, "paged remap: window and sinks must not be negative"};
    if (p.batch == 0) return kAccepted;
    if (!tokens) return {QTTS_EINVAL, "paged remap: null tokens"};
    if (!aligned_to(source, 4) || !aligned_to(tokens, 4) || !aligned_to(copied, 4))
        return {QTTS_EINVAL, "paged remap: misaligned array"};
    if (one_of(copied, {source, tokens, p.slots, p.page_table, p.refs}))
        return {QTTS_EINVAL, "paged remap: copied must be an array of its own"};
    return kAccepted;
}

inline Refusal check_reserve(const qtts_paged_pool &p, const int32_t *starts, const int32_t *ends,
                             const int32_t *lacking) {
    QTTS_REFUSE(check_pool(p));
    if (p.batch == 0) return kAccepted;
    if (!starts || !ends) return {QTTS_EINVAL, "paged reserve: null array"};
    if (!aligned_to(starts, 4) || !aligned_to(ends, 4) || !aligned_to(lacking, 4))
        return {QTTS_EINVAL, "paged reserve: misaligned array"};
    if (one_of(lacking, {p.slots, p.page_table, p.refs}))
        return {QTTS_EINVAL, "paged reserve: lacking must be none of the pool's arrays"};
    return kAccepted;
}

inline Refusal check_compact(const qtts_paged_pool &p, const int32_t *from, const int32_t *to, const int32_t *live) {
    QTTS_REFUSE(check_pool(p));
    if (p.num_pages > 1 && (!from || !to)) return {QTTS_EINVAL, "paged compact: null list"};
    if (!aligned_to(from, 4) || !aligned_to(to, 4) || !aligned_to(live, 4))
        return {QTTS_EINVAL, "paged compact: misaligned array"};
    if (from && from == to) return {QTTS_EINVAL, "paged compact: two lists"};
    return kAccepted;
}

// What it writes beside the pool is arrays of their own.
inline Refusal check_compact_own(const qtts_paged_pool &p, const int32_t *from, const int32_t *to,
                                 const int32_t *live) {
    if (one_of(from, {to, live, p.slots, p.page_table, p.refs}) || one_of(to, {live, p.slots, p.page_table, p.refs}) ||
        one_of(live, {p.slots, p.page_table, p.refs}))
        return {QTTS_EINVAL, "paged compact: from, to and live must be arrays of their own"};
    return kAccepted;
}

inline Refusal check_block_shape(const qtts_paged_kv &kv) {
    if (kv.head_dim != 64 && kv.head_dim != 128) return {QTTS_ESHAPE, "paged cache: head_dim must be 64 or 128"};
    if (kv.page_size != 16 && kv.page_size != 32 && kv.page_size != 64 && kv.page_size != 128)
        return {QTTS_ESHAPE, "paged cache: page_size must be 16, 32, 64 or 128"};
    if (kv.kv_heads < 1 || kv.kv_heads > 1024) return {QTTS_ESHAPE, "paged cache: kv_heads must be 1..1024"};
    return kAccepted;
}

// Blocks of a copy's launch: K's and V's of each pair of pages, and of each pair
// of slots and kv head.
inline Refusal check_copy_pages(const qtts_paged_kv &a, const qtts_paged_kv &b, int32_t n, const int32_t *from,
                                const int32_t *to) {
    QTTS_REFUSE(check_block_shape(a));
    if (a.head_dim != b.head_dim || a.page_size != b.page_size || a.kv_heads != b.kv_heads)
        return {QTTS_ESHAPE, "paged copy: the caches' pages differ in shape"};
    for (const qtts_paged_kv *kv : {&a, &b}) {
        if (kv->num_pages < 1) return {QTTS_ESHAPE, "paged copy: num_pages must be positive"};
        if ((long long)kv->num_pages * kv->kv_heads > (1LL << 31) - 1)
            return {QTTS_ERANGE, "paged cache: more than 2^31 - 1 blocks (pages times kv heads)"};
        if (!kv->k_codes || !kv->v_codes || !kv->k_scales || !kv->v_scales)
            return {QTTS_EINVAL, "paged cache: null buffer"};
        if (!aligned_to(kv->k_codes, 16) || !aligned_to(kv->v_codes, 16) || !aligned_to(kv->k_scales, 4) ||
            !aligned_to(kv->v_scales, 4))
            return {QTTS_EINVAL, "paged cache: buffers must be 16-byte aligned"};
    }
    if (n < 0) return {QTTS_ESHAPE, "paged copy: a negative number of pages"};
    if (2LL * n > kPagedMaxBlocks) return {QTTS_ERANGE, "paged copy: more pages than a launch holds"};
    if (n == 0) return kAccepted;
    if (!from || !to) return {QTTS_EINVAL, "paged copy: null list"};
    if (!aligned_to(from, 4) || !aligned_to(to, 4)) return {QTTS_EINVAL, "paged copy: misaligned list"};
    return kAccepted;
}

inline Refusal check_copy_open(const qtts_paged_kv &kv, int32_t n, const int32_t *from, const int32_t *to,
                               const int32_t *tokens) {
    QTTS_REFUSE(check_block_shape(kv));
    if (kv.num_slots < 1) return {QTTS_ESHAPE, "paged copy: num_slots must be positive"};
    if (!kv.k_open || !kv.v_open) return {QTTS_EINVAL, "paged cache: null buffer"};
    if (!aligned_to(kv.k_open, 16) || !aligned_to(kv.v_open, 16))
        return {QTTS_EINVAL, "paged cache: buffers must be 16-byte aligned"};
    if (n < 0) return {QTTS_ESHAPE, "paged copy: a negative number of slots"};
    if (2LL * n * kv.kv_heads > kPagedMaxBlocks) return {QTTS_ERANGE, "paged copy: more slots than a launch holds"};
    if (n == 0) return kAccepted;
    if (!from || !to || !tokens) return {QTTS_EINVAL, "paged copy: null list"};
    if (!aligned_to(from, 4) || !aligned_to(to, 4) || !aligned_to(tokens, 4))
        return {QTTS_EINVAL, "paged copy: misaligned list"};
    return kAccepted;
}

// A row's source and length after a remap, whatever the device arrays hold.
struct Heir {
    int source;  // -1: none
    int tokens;
};
QTTS_HD Heir heir_of(const qtts_paged_pool &p, const int32_t *source, const int32_t *tokens, int b) {
    const int s = source ? source[b] : b, t = tokens[b], most = p.max_pages * p.page_size;
    if (s < 0 || s >= p.batch) return {-1, 0};
    return {s, t < 0 ? 0 : t > most ? most : t};
}

// Whether a row of `tokens` keeps its source's page j: full ones, and its own
// that is being filled; behind a window those that hold a sink or a token that
// the next row sees.
QTTS_HD bool page_kept(int j, int tokens, bool self, int page_size, int window, int sinks) {
    const int entries = self ? (tokens + page_size - 1) / page_size : tokens / page_size;
    if (j >= entries) return false;
    if (window == 0) return true;
    return (long long)(j + 1) * page_size > (long long)tokens - window + 1 || (long long)j * page_size < sinks;
}

// Entries first .. last - 1 of a row that a reservation looks at; first < 0: the
// row is left out.
struct Span {
    int first, last;
};
QTTS_HD Span reserve_span(const qtts_paged_pool &p, int start, int end) {
    if (start < 0 || end < 0 || end > p.max_pages * p.page_size) return {-1, -1};
    const int last = (end + p.page_size - 1) / p.page_size;
    return {start / p.page_size < last ? start / p.page_size : last, last};
}

}  // namespace qtts
