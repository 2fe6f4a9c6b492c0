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

// Exclusive sum over the block's threads, and the total; `sums`: kWaves ints.
__device__ __forceinline__ int block_rank(int v, int *sums, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
    }
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

// What entry i becomes; references change where it does.
__device__ __forceinline__ int remapped(const RemapParams &A, int i) {
    const int b = i / A.pool.max_pages, j = i % A.pool.max_pages;
    const Heir h = heir_of(A.pool, A.source, A.tokens, b);
    const int old = A.pool.page_table[i];
    int now = -1;
    if (h.source >= 0 && page_kept(j, h.tokens, h.source == b, A.pool.page_size, A.window, A.sinks))
        now = h.source == b ? old : A.pool.page_table[(size_t)h.source * A.pool.max_pages + j];
    if (!in_pool(A.pool, now)) now = -1;
    if (old != now) {
        if (in_pool(A.pool, old)) atomicSub(A.pool.refs + old, 1);
        if (now >= 0) atomicAdd(A.pool.refs + now, 1);
    }
    return now;
}

// Tables of up to kRemapThreads * kRemapEach entries: all read, then written.
__global__ __launch_bounds__(kThreads) void k_paged_remap_one(RemapParams A) {
    __shared__ Slots S;
    const int n = A.pool.batch * A.pool.max_pages;
    int now[kRemapEach];
#pragma unroll
    for (int k = 0; k < kRemapEach; k++) {
        const int i = k * kThreads + threadIdx.x;
        now[k] = i < n ? remapped(A, i) : -1;
    }
    hand_on_slots(A, S);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRemapEach; k++) {
        const int i = k * kThreads + threadIdx.x;
        if (i < n) A.pool.page_table[i] = now[k];
    }
}

// Larger ones: new rows to scratch, block 0 the slots; then scratch to the table.
__global__ __launch_bounds__(kThreads) void k_paged_remap(RemapParams A) {
    __shared__ Slots S;
    if (blockIdx.x == 0) return hand_on_slots(A, S);
    const int i = (blockIdx.x - 1) * kThreads + threadIdx.x;
    if (i < A.pool.batch * A.pool.max_pages) A.scratch[i] = remapped(A, i);
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
// first; from the first row that cannot be served whole on, none.
__global__ __launch_bounds__(kThreads) void k_paged_reserve(ReserveParams A) {
    __shared__ int need[kPoolBatch];
    __shared__ int sums[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, batch = A.pool.batch;
    int refs[16];
    load_refs(A.pool, 0, refs);
    for (int b = wave; b < batch; b += kWaves) {
        const Span s = reserve_span(A.pool, A.starts[b], A.ends[b]);
        const int32_t *row = A.pool.page_table + (size_t)b * A.pool.max_pages;
        int n = 0;
        for (int j0 = s.first; j0 < s.last; j0 += 64)
            n += __popcll(__ballot(j0 + lane < s.last && !in_pool(A.pool, row[min(j0 + lane, s.last - 1)])));
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
                if (rank < total) A.scratch[rank] = at + 16 * tid + k;
                rank++;
            }
        found += n;
    }
    found = min(found, total);
    __syncthreads();
    for (int b = wave; b < batch; b += kWaves) {
        const Span s = reserve_span(A.pool, A.starts[b], A.ends[b]);
        const int base = need[b], end = b + 1 < batch ? need[b + 1] : total;
        const bool served = end <= found;
        if (lane == 0 && A.lacking) A.lacking[b] = s.first < 0 ? -1 : served ? 0 : end - base;
        if (!served || base == end) continue;
        int32_t *row = A.pool.page_table + (size_t)b * A.pool.max_pages;
        int rank = base;
        for (int j0 = s.first; j0 < s.last; j0 += 64) {
            const bool want = j0 + lane < s.last && !in_pool(A.pool, row[min(j0 + lane, s.last - 1)]);
            const uint64_t all = __ballot(want);
            if (want) {
                const int id = A.scratch[rank + __popcll(all & ((1ull << lane) - 1))];
                row[j0 + lane] = id;
                A.pool.refs[id] = 1;
            }
            rank += __popcll(all);
        }
    }
}

// Which pages move where so that those in use are the pool's first: the i-th in use
// behind that border to the i-th free one before it.  Their new names go to scratch,
// the border to its end.  One block.
__global__ __launch_bounds__(kThreads) void k_paged_compact(CompactParams A) {
    __shared__ int sums[kWaves];
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
        if (n > kPoolChunk) load_refs(A.pool, at, refs);
        const int first = at + 16 * tid;
        int movers = 0, free = 0, m, h;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int id = first + k;
            movers += id < n && id >= live && refs[k] > 0;
            free += id < live && refs[k] <= 0;
        }
        int rank_m = moves + block_rank(movers, sums, m), rank_h = holes + block_rank(free, sums, h);
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int id = first + k;
            if (id < n && id >= live) {
                if (refs[k] > 0) A.from[rank_m++] = id;
                else A.scratch[id] = id;
            } else if (id < live && refs[k] <= 0) {
                A.to[rank_h++] = id;
            }
        }
        moves += m, holes += h;
    }
    __syncthreads();
    for (int i = tid; i < n / 2; i += kThreads) {
        if (i < moves) {
            const int a = A.from[i], b = A.to[i];
            A.scratch[a] = b;
            A.pool.refs[b] = A.pool.refs[a];
            A.pool.refs[a] = 0;
        } else {
            A.from[i] = A.to[i] = -1;
        }
    }
    if (tid == 0) {
        A.scratch[n] = live;
        if (A.live) *A.live = live;
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

// A block for K or V of each pair of pages.
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
        hipLaunchKernelGGL(k_paged_remap_one, dim3(1), dim3(kThreads), 0, st, p);
        return;
    }
    hipLaunchKernelGGL(k_paged_remap, dim3(1 + (unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, p);
    hipLaunchKernelGGL(k_paged_remap_store, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
}

void launch_paged_reserve(hipStream_t st, const ReserveParams &p) {
    hipLaunchKernelGGL(k_paged_reserve, dim3(1), dim3(kThreads), 0, st, p);
}

void launch_paged_compact(hipStream_t st, const CompactParams &p) {
    hipLaunchKernelGGL(k_paged_compact, dim3(1), dim3(kThreads), 0, st, p);
    const long long n = (long long)p.pool.batch * p.pool.max_pages;
    if (n) hipLaunchKernelGGL(k_paged_rename, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
}

void launch_paged_copy_pages(hipStream_t st, const CopyPagesParams &p, int n) {
    hipLaunchKernelGGL(k_paged_copy_pages, dim3(2 * (unsigned)n), dim3(256), 0, st, p);
}

void launch_paged_copy_open(hipStream_t st, const CopyOpenParams &p, int n) {
    hipLaunchKernelGGL(k_paged_copy_open, dim3(2 * (unsigned)n * p.kv.kv_heads), dim3(256), 0, st, p);
}

}  // namespace qtts
