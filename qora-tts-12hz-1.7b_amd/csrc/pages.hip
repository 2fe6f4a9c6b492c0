// pages.hip — the pages of a paged cache on the device: rows of the page table
// forked, cut and freed with their references counted, pages reserved, the pool
// packed, pages and open rows copied.
//
// Everything that decides an order (which page is given out, where one moves to,
// who keeps a slot) is a rank in index order, found by scans in one block, so
// results do not depend on the order of atomics; those only count.
#include <algorithm>

#include "device_common.h"
#include "pages_plan.h"
#include "serve.h"

namespace qtts {

namespace {

constexpr int kThreads = kRemapThreads, kWaves = kThreads / 64;

// Sum over the lanes up to this one: rows of 16 by shifts, then their last lanes' sums.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}

// Exclusive sum over the block's threads, and the total; `sums`: kWaves ints.
__device__ __forceinline__ int block_rank(int v, int *sums, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int x = wave_scan(v);
    __syncthreads();  // the last call's sums have been read
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        const int s = sums[w];
        before += w < wave ? s : 0;
        all += s;
    }
    total = all;
    return before + x - v;
}

__device__ __forceinline__ bool in_pool(const qtts_paged_pool &p, int id) { return id >= 0 && id < p.num_pages; }

// Slots: a sequence that goes on keeps its own, one that only others go on from
// leaves it to the first of them; the rest take the slots of those that ended, both
// in order.  One block.
struct Slots {
    int heir[kPoolBatch], old[kPoolBatch], ended[kPoolBatch];
    int sums[kWaves];
};

__device__ void hand_on_slots(const RemapParams &A, Slots &S) {
    const int batch = A.pool.batch, tid = threadIdx.x;
    for (int b = tid; b < batch; b += kThreads) S.heir[b] = batch, S.old[b] = A.pool.slots[b];
    __syncthreads();
    for (int b = tid; b < batch; b += kThreads) {
        const Heir h = heir_of(A.pool, A.source, A.tokens, b);
        if (h.source >= 0) atomicMin(&S.heir[h.source], b);
    }
    __syncthreads();
    for (int b = tid; b < batch; b += kThreads)
        if (heir_of(A.pool, A.source, A.tokens, b).source == b) S.heir[b] = b;
    __syncthreads();
    int at = 0;
    for (int b0 = 0; b0 < batch; b0 += kThreads) {
        const int b = b0 + tid;
        const bool ended = b < batch && S.heir[b] == batch;
        int n;
        const int rank = block_rank(ended, S.sums, n);
        if (ended) S.ended[at + rank] = S.old[b];
        at += n;
    }
    __syncthreads();
    at = 0;
    for (int b0 = 0; b0 < batch; b0 += kThreads) {
        const int b = b0 + tid;
        const Heir h = b < batch ? heir_of(A.pool, A.source, A.tokens, b) : Heir{-1, 0};
        const bool first = h.source >= 0 && S.heir[h.source] == b;
        int n;
        const int rank = block_rank(b < batch && !first, S.sums, n);
        if (b < batch) {
            A.pool.slots[b] = first ? S.old[h.source] : S.ended[at + rank];
            if (A.copied)
                A.copied[b] = h.source >= 0 && !first && h.tokens % A.pool.page_size ? S.old[h.source] : -1;
        }
        at += n;
    }
}

// What N entries from `first` on, kThreads apart, become, of a table that has some;
// references change where they do.  Loads of one kind are asked for together, one kind
// after another: what an entry was, its row's heir, the heir's entry.
template <int N>
__device__ __forceinline__ void remapped(const RemapParams &A, int first, int (&now)[N]) {
    const int n = A.pool.batch * A.pool.max_pages, wide = A.pool.max_pages;
    int old[N], from[N];
    Heir h[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int i = min(first + k * kThreads, n - 1);
        old[k] = A.pool.page_table[i];
        h[k] = heir_of(A.pool, A.source, A.tokens, i / wide);
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int i = min(first + k * kThreads, n - 1), b = i / wide, j = i % wide;
        const bool kept = h[k].source >= 0 &&
                          page_kept(j, h[k].tokens, h[k].source == b, A.pool.page_size, A.window, A.sinks);
        from[k] = kept ? h[k].source * wide + j : -1;
        now[k] = A.pool.page_table[max(from[k], 0)];
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        if (from[k] < 0 || !in_pool(A.pool, now[k])) now[k] = -1;
        if (first + k * kThreads < n && old[k] != now[k]) {
            if (in_pool(A.pool, old[k])) atomicSub(A.pool.refs + old[k], 1);
            if (now[k] >= 0) atomicAdd(A.pool.refs + now[k], 1);
        }
    }
}

// Tables of up to kRemapThreads * kRemapEach entries: block 0 reads them all, then
// writes; block 1 hands on the slots.  8 rows of 18: 3.5 us.  (64 of 127 took 13 us this
// way, most of it one CU's atomics.)
__global__ __launch_bounds__(kThreads) void k_paged_remap_one(RemapParams A) {
    __shared__ Slots S;
    if (blockIdx.x == 1) return hand_on_slots(A, S);
    const int n = A.pool.batch * A.pool.max_pages;
    if (n == 0) return;
    int now[kRemapEach];
    remapped(A, threadIdx.x, now);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRemapEach; k++) {
        const int i = k * kThreads + threadIdx.x;
        if (i < n) A.pool.page_table[i] = now[k];
    }
}

// Larger ones: new rows to scratch, block 0 the slots; then scratch to the table: up to
// kRemapStored entries by the block that ends last (64 of 127 4.8 to 5.9 us), more in a launch
// of their own (4.1 + 2.3 us; 64 of 500 5.6 together, 2^20 entries 12.7, 2^22 31).
template <bool LAST>
__global__ __launch_bounds__(kThreads) void k_paged_remap(RemapParams A) {
    __shared__ Slots S;
    __shared__ bool last;
    if (blockIdx.x == 0) return hand_on_slots(A, S);
    const int n = A.pool.batch * A.pool.max_pages, i = (blockIdx.x - 1) * kThreads + threadIdx.x;
    int now[1];
    remapped(A, i, now);
    if (!LAST) {
        if (i < n) A.scratch[i] = now[0];
        return;
    }
    if (i < n) st_dev_i32(A.scratch + i, now[0]);
    wait_stores();
    __syncthreads();
    if (threadIdx.x == 0) {
        last = arrive_dev(A.counter) == gridDim.x - 2;
        if (last) reset_dev(A.counter);
    }
    __syncthreads();
    if (!last) return;
    for (int j = threadIdx.x; j < n; j += 8 * kThreads) {
        int x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = ld_dev_i32(A.scratch + min(j + k * kThreads, n - 1));
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (j + k * kThreads < n) A.pool.page_table[j + k * kThreads] = x[k];
    }
}

__global__ __launch_bounds__(256) void k_paged_remap_store(RemapParams A) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < A.pool.batch * A.pool.max_pages) A.pool.page_table[i] = A.scratch[i];
}

// Sixteen pages' references from page `at` + 16 * thread; behind the pool ones that
// are in use.
__device__ __forceinline__ void load_refs(const qtts_paged_pool &p, int at, int (&r)[16]) {
    const int first = at + 16 * threadIdx.x;
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
        if (first + k + 4 <= p.num_pages) {
            const int4 v = *reinterpret_cast<const int4 *>(p.refs + first + k);
            r[k] = v.x, r[k + 1] = v.y, r[k + 2] = v.z, r[k + 3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) r[k + e] = first + k + e < p.num_pages ? p.refs[first + k + e] : 1;
        }
    }
}

// Pages for each row's span, in order of rows and entries, the lowest free ones
// first; from the first row that cannot be served whole on, none.  16 lanes a row, as
// most rows want a page or two; the pages found lie in LDS as far as they fit.  64
// rows, some of them new with up to 31 pages, of 14046: 8 us, a chain of latencies
// (spans, references, ranks, entries).
constexpr int kFoundLds = 8192;
__global__ __launch_bounds__(kThreads) void k_paged_reserve(ReserveParams A) {
    __shared__ int need[kPoolBatch];
    __shared__ int found_ids[kFoundLds];
    __shared__ int sums[kWaves];
    constexpr int kRows = kThreads / 16;
    const int tid = threadIdx.x, lane = tid & 15, at64 = tid & 48, batch = A.pool.batch;
    int refs[16];
    load_refs(A.pool, 0, refs);
    // whether this lane's entry, j0 + lane of a span, wants a page, and the row's lanes' answers
    auto wants = [&](const int32_t *row, const Span &s, int j0, unsigned &all) {
        const bool want = j0 + lane < s.last && !in_pool(A.pool, row[min(j0 + lane, s.last - 1)]);
        all = (unsigned)(__ballot(want) >> at64) & 0xffffu;
        return want;
    };
    for (int b = tid >> 4; b < batch; b += kRows) {
        const Span s = reserve_span(A.pool, A.starts[b], A.ends[b]);
        const int32_t *row = A.pool.page_table + (size_t)b * A.pool.max_pages;
        int n = 0;
        for (int j0 = s.first; j0 < s.last; j0 += 16) {
            unsigned all;
            wants(row, s, j0, all);
            n += __popc(all);
        }
        if (lane == 0) need[b] = n;
    }
    __syncthreads();
    int total = 0;  // (at most the table's entries)
    for (int b0 = 0; b0 < batch; b0 += kThreads) {
        const int b = b0 + tid;
        int n;
        const int rank = block_rank(b < batch ? need[b] : 0, sums, n);
        if (b < batch) need[b] = total + rank;  // pages of the rows before
        total += n;
    }
    int found = 0;
    for (int at = 0; found < total && at < A.pool.num_pages; at += kPoolChunk) {
        if (at > 0) load_refs(A.pool, at, refs);
        int mine = 0, n;
#pragma unroll
        for (int k = 0; k < 16; k++) mine += refs[k] <= 0;
        int rank = found + block_rank(mine, sums, n);
#pragma unroll
        for (int k = 0; k < 16; k++)
            if (refs[k] <= 0) {
                const int id = at + 16 * tid + k;
                if (rank < kFoundLds) found_ids[rank] = id;
                else if (rank < total) A.scratch[rank] = id;
                rank++;
            }
        found += n;
    }
    found = min(found, total);
    __syncthreads();
    for (int b = tid >> 4; b < batch; b += kRows) {
        const Span s = reserve_span(A.pool, A.starts[b], A.ends[b]);
        const int base = need[b], end = b + 1 < batch ? need[b + 1] : total;
        const bool served = end <= found;
        if (lane == 0 && A.lacking) A.lacking[b] = s.first < 0 ? -1 : served ? 0 : end - base;
        if (!served || base == end) continue;
        int32_t *row = A.pool.page_table + (size_t)b * A.pool.max_pages;
        int rank = base;
        for (int j0 = s.first; j0 < s.last; j0 += 16) {
            unsigned all;
            if (wants(row, s, j0, all)) {
                const int r = rank + __popc(all & ((1u << lane) - 1));
                const int id = r < kFoundLds ? found_ids[r] : A.scratch[r];
                row[j0 + lane] = id;
                A.pool.refs[id] = 1;
            }
            rank += __popc(all);
        }
    }
}

// Which pages move where so that those in use are the pool's first: the i-th in use
// behind that border to the i-th free one before it.  Their new names go to scratch,
// the border to its end.  One block, which renames a smaller table too; the moves of a
// pool of one chunk stay in LDS (12532 pages, 2300 moves, without the renaming: 10.5 us,
// 12.5 by way of the lists).  Larger pools are the one block's to read twice: 65536 pages,
// half of them in use anywhere, 52 us with the renaming, 2^20 0.75 ms, 2^22 3.0 ms.
template <bool ONE>
__global__ __launch_bounds__(kThreads) void k_paged_compact(CompactParams A) {
    __shared__ int sums[kWaves];
    constexpr int kMoves = ONE ? kPoolChunk / 2 : 1;
    __shared__ int from[kMoves], held[kMoves], to[kMoves];  // held: the page's references
    const int tid = threadIdx.x, n = A.pool.num_pages;
    int refs[16], live = 0;
    for (int at = 0; at < n; at += kPoolChunk) {
        load_refs(A.pool, at, refs);
        int mine = 0, m;
#pragma unroll
        for (int k = 0; k < 16; k++) mine += refs[k] > 0 && at + 16 * tid + k < n;
        block_rank(mine, sums, m);
        live += m;
    }
    int moves = 0, holes = 0;
    for (int at = 0; at < n; at += kPoolChunk) {
        if (!ONE) load_refs(A.pool, at, refs);
        const int first = at + 16 * tid;
        int movers = 0, free = 0, m, h;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int id = first + k;
            movers += id < n && id >= live && refs[k] > 0;
            free += id < live && refs[k] <= 0;
        }
        // (a chunk's counts of both in one scan)
        const int both = block_rank(movers << 16 | free, sums, m);
        int rank_m = moves + (both >> 16), rank_h = holes + (both & 0xffff);
        h = m & 0xffff, m >>= 16;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int id = first + k;
            if (id < n && id >= live) {
                if (refs[k] <= 0) A.scratch[id] = id;
                else if (ONE) from[rank_m] = id, held[rank_m++] = refs[k];
                else A.from[rank_m++] = id;
            } else if (id < live && refs[k] <= 0) {
                if (ONE) to[rank_h++] = id;
                else A.to[rank_h++] = id;
            }
        }
        moves += m, holes += h;
    }
    __syncthreads();
    for (int i = tid; i < n / 2; i += kThreads) {
        int a = -1, b = -1;
        if (i < moves) {
            a = ONE ? from[i] : A.from[i], b = ONE ? to[i] : A.to[i];
            A.scratch[a] = b;
            A.pool.refs[b] = ONE ? held[i] : A.pool.refs[a];
            A.pool.refs[a] = 0;
        }
        if (ONE || i >= moves) A.from[i] = a, A.to[i] = b;
    }
    if (tid == 0) {
        A.scratch[n] = live;
        if (A.live) *A.live = live;
    }
    const int entries = A.pool.batch * A.pool.max_pages;
    if (entries > kRenameOne) return;
    __syncthreads();  // the names are there
    for (int i0 = tid; i0 < entries; i0 += 8 * kThreads) {
        int id[8];
#pragma unroll
        for (int k = 0; k < 8; k++) id[k] = A.pool.page_table[min(i0 + k * kThreads, entries - 1)];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const bool moved = i0 + k * kThreads < entries && in_pool(A.pool, id[k]) && id[k] >= live;
            if (moved) A.pool.page_table[i0 + k * kThreads] = A.scratch[id[k]];
        }
    }
}

__global__ __launch_bounds__(256) void k_paged_rename(CompactParams A) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= A.pool.batch * A.pool.max_pages) return;
    const int id = A.pool.page_table[i];
    if (in_pool(A.pool, id) && id >= A.scratch[A.pool.num_pages]) A.pool.page_table[i] = A.scratch[id];
}

// `bytes` from one place to another, 16 a thread and four loads in flight.
__device__ __forceinline__ void copy_bytes(void *to, const void *from, int bytes) {
    const u32x4 *a = reinterpret_cast<const u32x4 *>(from);
    u32x4 *b = reinterpret_cast<u32x4 *>(to);
    const int n = bytes / 16;
    for (int i0 = threadIdx.x; i0 < n; i0 += 4 * blockDim.x) {
        u32x4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i0 + k * (int)blockDim.x < n) x[k] = __builtin_nontemporal_load(glb(a + i0 + k * blockDim.x));
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i0 + k * (int)blockDim.x < n) __builtin_nontemporal_store(x[k], glb(b + i0 + k * blockDim.x));
    }
}

// A block for K or V of each pair of pages.  Bound by memory: 2270 of 131 KB each way,
// 0.6 GB in 100 us (5.9 TB/s), blocks of pairs that are not there among them.
__global__ __launch_bounds__(256) void k_paged_copy_pages(CopyPagesParams A) {
    const int pair = blockIdx.x >> 1, from = A.from[pair], to = A.to[pair], heads = A.a.kv_heads;
    if (from < 0 || from >= A.a.num_pages || to < 0 || to >= A.b.num_pages) return;
    const int bytes = heads * A.a.page_size * A.a.head_dim;
    const bool v = blockIdx.x & 1;
    copy_bytes((v ? A.b.v_codes : A.b.k_codes) + (size_t)to * bytes,
               (v ? A.a.v_codes : A.a.k_codes) + (size_t)from * bytes, bytes);
    const float *sa = (v ? A.a.v_scales : A.a.k_scales) + (size_t)from * heads;
    float *sb = (v ? A.b.v_scales : A.b.k_scales) + (size_t)to * heads;
    for (int h = threadIdx.x; h < heads; h += 256) sb[h] = sa[h];
}

// A block for K or V of each pair of slots and kv head: the rows that the tokens
// behind the last full page take.
__global__ __launch_bounds__(256) void k_paged_copy_open(CopyOpenParams A) {
    const int heads = A.kv.kv_heads, head = blockIdx.x / 2 % heads, pair = blockIdx.x / 2 / heads;
    const int from = A.from[pair], to = A.to[pair], tokens = A.tokens[pair];
    if (from < 0 || from >= A.kv.num_slots || to < 0 || to >= A.kv.num_slots || from == to || tokens < 0) return;
    const int rows = tokens % A.kv.page_size;
    const size_t each = (size_t)A.kv.page_size * A.kv.head_dim;
    float *open = blockIdx.x & 1 ? A.kv.v_open : A.kv.k_open;
    copy_bytes(open + ((size_t)to * heads + head) * each, open + ((size_t)from * heads + head) * each,
               rows * A.kv.head_dim * 4);
}

}  // namespace

void launch_paged_remap(hipStream_t st, const RemapParams &p) {
    const long long n = (long long)p.pool.batch * p.pool.max_pages;
    if (n <= kRemapThreads * kRemapEach) {
        hipLaunchKernelGGL(k_paged_remap_one, dim3(2), dim3(kThreads), 0, st, p);
        return;
    }
    const unsigned blocks = 1 + (unsigned)((n + kThreads - 1) / kThreads);
    if (n <= kRemapStored) {
        hipLaunchKernelGGL(k_paged_remap<true>, dim3(blocks), dim3(kThreads), 0, st, p);
        return;
    }
    hipLaunchKernelGGL(k_paged_remap<false>, dim3(blocks), dim3(kThreads), 0, st, p);
    hipLaunchKernelGGL(k_paged_remap_store, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
}

void launch_paged_reserve(hipStream_t st, const ReserveParams &p) {
    hipLaunchKernelGGL(k_paged_reserve, dim3(1), dim3(kThreads), 0, st, p);
}

void launch_paged_compact(hipStream_t st, const CompactParams &p) {
    if (p.pool.num_pages <= kPoolChunk) hipLaunchKernelGGL(k_paged_compact<true>, dim3(1), dim3(kThreads), 0, st, p);
    else hipLaunchKernelGGL(k_paged_compact<false>, dim3(1), dim3(kThreads), 0, st, p);
    const long long n = (long long)p.pool.batch * p.pool.max_pages;
    if (n > kRenameOne) hipLaunchKernelGGL(k_paged_rename, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
}

void launch_paged_copy_pages(hipStream_t st, const CopyPagesParams &p, int n) {
    hipLaunchKernelGGL(k_paged_copy_pages, dim3(2 * (unsigned)n), dim3(256), 0, st, p);
}

void launch_paged_copy_open(hipStream_t st, const CopyOpenParams &p, int n) {
    hipLaunchKernelGGL(k_paged_copy_open, dim3(2 * (unsigned)n * p.kv.kv_heads), dim3(256), 0, st, p);
}

}  // namespace qtts
