// sample_rows.hip — a token from each row of logits: temperature, top-k,
// top-p, min-p, given uniform numbers.
//
// Weights w_i = exp((l_i - max) / T) are evaluated in 64 bits and summed as
// integers of 2^-44 of the largest: sums do not depend on their order, and a
// draw next to the border between two tokens falls as the 64-bit definition's
// does.  What is kept is a prefix of the tokens in order (logit down, index up),
// so that it is two numbers: a least key, and how many of those at it, the first
// by index.
//
// Rows of up to kRowVocab logits take a block each, which holds the row's keys
// in LDS (k_sample_row).  Longer rows are read in chunks by as many blocks as
// they have: their maxima (k_sample_max), sums (k_sample_sum) and, where top-p
// cuts without a top-k, the tokens next to the cut (k_sample_near); the row's
// last block joins them and draws (k_sample_draw).
#include <algorithm>

#include "device_common.h"
#include "paged_plan.h"
#include "serve.h"

namespace qtts {

namespace {

typedef unsigned long long u64;
typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr double kUnit = 17592186044416.0;  // 2^44

// Order-preserving integer of a float (no NaN), both zeros alike.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ u64 wave_scan(u64 v) {
    for (int off = 1; off < 64; off <<= 1) {
        const u64 y = (u64)__shfl_up((long long)v, off, 64);
        if ((threadIdx.x & 63) >= (unsigned)off) v += y;
    }
    return v;
}
__device__ __forceinline__ u64 wave_total(u64 v) {
    for (int off = 32; off > 0; off >>= 1) v += (u64)__shfl_xor((long long)v, off, 64);
    return v;
}
__device__ __forceinline__ unsigned wave_top(unsigned v) {
    for (int off = 32; off > 0; off >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, off, 64));
    return v;
}

// Sum over the block's NT threads; every thread gets it.
template <int NT>
__device__ u64 block_total(u64 v, u64 *wsum) {
    v = wave_total(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < NT / 64; w++) all += wsum[w];
    return all;
}

// Inclusive scan over the block; every thread gets the total as well.
template <int NT>
__device__ u64 block_scan(u64 v, u64 *wsum, u64 *total) {
    const int wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) wsum[wave] = v;
    __syncthreads();
    u64 base = 0, all = 0;
    for (int w = 0; w < NT / 64; w++) {
        if (w < wave) base += wsum[w];
        all += wsum[w];
    }
    *total = all;
    return base + v;
}

struct RowSettings {
    float t, top_p, min_p;
    int top_k;  // 0: off
    bool greedy;
    double least;  // min-p's weight
    __device__ __forceinline__ RowSettings(const SampleRowsParams &P, int r) {
        t = P.p.temperature ? P.p.temperature[r] : 1.0f;
        top_k = P.p.top_k ? P.p.top_k[r] : 0;
        top_p = P.p.top_p ? P.p.top_p[r] : 1.0f;
        min_p = P.p.min_p ? P.p.min_p[r] : 0.0f;
        if (top_k < 0 || top_k >= P.vocab) top_k = 0;
        greedy = !(t > 0.0f);
        least = min_p > 0.0f ? (min_p < 1.0f ? (double)min_p : 1.0) : 0.0;
    }
    __device__ __forceinline__ bool cuts_sum() const { return top_p < 1.0f; }
    // Units of `total` whose reaching ends the prefix that top-p keeps: kept
    // are those whose predecessors' sum is below top_p * total.
    __device__ __forceinline__ u64 share_of(u64 total) const {
        const u64 need = (u64)ceil((double)(top_p > 0.0f ? top_p : 0.0f) * (double)total);
        return need < 1 ? 1 : need;
    }
    __device__ __forceinline__ u64 target_of(float u, u64 total) const {
        const u64 x = (u64)((u > 0.0f ? (u < 1.0f ? (double)u : 1.0) : 0.0) * (double)total);
        return x < total ? x : total - 1;
    }
};

// exp((l - max) / T) as 2^(y / 64), y = (l - max) * 64 log2(e) / T: the whole
// part of y from a table of 2^(j/64) and an exponent, the rest (below 0.0055 in
// the exponent of e) by its series to the fifth power, 3e-17 off.  A dozen 64-bit
// operations, a fifth of the library's exp.
constexpr int kBins = 1536;  // of 1/32 octave: weights down to 2^-48
struct Weights {
    float mx;
    double scale;
    const double *tab;
    __device__ __forceinline__ double place(float l) const { return ((double)l - (double)mx) * scale; }
    // nothing below 2^-46 reaches half a unit
    __device__ __forceinline__ bool counts(float l, double y) const {
        return l != -INFINITY && mx != INFINITY && y > -46.0 * 64;
    }
    __device__ __forceinline__ double raised(double y, int by) const {
        const double n = rint(y), r = (y - n) * (0.693147180559945309417 / 64);
        const double p = fma(fma(fma(fma(fma(1.0 / 120, r, 1.0 / 24), r, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0);
        const int k = (int)n;
        return ldexp(tab[k & 63] * p, (k >> 6) + by);
    }
    __device__ __forceinline__ double weight(float l) const {
        if (l == mx) return 1.0;
        const double y = place(l);
        return counts(l, y) ? raised(y, 0) : 0.0;
    }
    // in units, kept by min-p or not
    __device__ __forceinline__ u64 units(float l, double least = 0.0) const {
        if (l == mx) return (u64)kUnit;
        const double y = place(l);
        if (!counts(l, y)) return 0;
        const double w = raised(y, 44);
        if (w < least * kUnit) return 0;
        return __builtin_bit_cast(u64, w + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: to the nearest
    }
    // weights fall with the bin
    __device__ __forceinline__ int bin(float l) const {
        if (l == mx) return 0;
        const double y = place(l);
        return counts(l, y) ? min((int)(y * -0.5), kBins - 1) : kBins - 1;
    }
};

// By the first wave, before a barrier.
__device__ __forceinline__ void fill_table(double *tab) {
    if (threadIdx.x < 64) tab[threadIdx.x] = exp2((double)threadIdx.x / 64);
}
__device__ __forceinline__ Weights weights_of(const RowSettings &S, float mx, const double *tab) {
    return {mx, 64 * 1.44269504088896340736 / (double)S.t, tab};
}

// What is kept of a set: keys above `thr`, and the first `ties` at it.
struct Cut {
    unsigned thr = 0;
    u64 ties = ~0ull;
};

constexpr int kBrute = 256;  // a set this small is ranked by comparing all pairs

struct Space {
    double tab[64];
    u64 hist[256], wsum[16], base;
    unsigned digit, thr, ties, top, bad;
    int token;
};

// The prefix that top-k and top-p keep of n keys, key(i) in the order of their
// indices; `need`: the sum that top-p's prefix reaches, 0: its share of the sum.
// Small sets by comparing all pairs; others by 8 bits of the key at a time,
// counts first and then sums.
template <int NT, class Key>
__device__ Cut cut_of(const Key &key, int n, const RowSettings &S, const Weights &W, u64 need, Space *sp) {
    const int tid = threadIdx.x;
    const bool sums = S.cuts_sum();
    Cut c;
    if (S.top_k == 0 && !sums) return c;
    if (n <= kBrute) {
        u64 *units = sp->hist;
        __syncthreads();
        if (tid == 0) sp->thr = 0xffffffffu, sp->ties = 0;
        const bool in = tid < n;
        const unsigned k = in ? key(tid) : 0;
        const u64 mine = in ? W.units(logit_of(k)) : 0;
        if (in) units[tid] = mine;
        __syncthreads();
        unsigned rank = 0;
        u64 ahead = 0;
        if (in)
            for (int j = 0; j < n; j++) {
                const unsigned o = key(j);
                const bool before = o > k || (o == k && j < tid);
                rank += before;
                ahead += before ? units[j] : 0;
            }
        bool keep = in && (S.top_k == 0 || rank < (unsigned)S.top_k);
        if (sums) {
            if (need == 0) need = S.share_of(block_total<NT>(keep ? mine : 0, sp->wsum));
            keep = keep && ahead < need;
        }
        if (keep) atomicMin(&sp->thr, k);
        __syncthreads();
        c.thr = sp->thr;
        if (keep && k == c.thr) atomicAdd(&sp->ties, 1u);
        __syncthreads();
        c.ties = sp->ties;
        return c;
    }
    auto select = [&](bool by_sum, u64 want, u64 *above) {
        unsigned prefix = 0;
        u64 base = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            for (int i = tid; i < 256; i += NT) sp->hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += NT) {
                const unsigned k = key(i);
                if (k < c.thr || (shift < 24 && k >> (shift + 8) != prefix)) continue;
                const u64 w = by_sum ? W.units(logit_of(k)) : (u64)1;
                if (w) atomicAdd(&sp->hist[(k >> shift) & 255], w);
            }
            __syncthreads();
            if (tid < 64) {  // from the top: a lane has digits 255 - 4 lane and the next three
                u64 h[4], sum = 0;
                for (int j = 0; j < 4; j++) sum += h[j] = sp->hist[255 - 4 * tid - j];
                u64 run = base + wave_scan(sum) - sum;
                const bool mine = run < want && run + sum >= want, none = !__any(mine);
                if (mine || (none && tid == 63)) {
                    int j = 0;
                    for (; j < 3 && run + h[j] < want; j++) run += h[j];
                    sp->digit = 255 - 4 * tid - j;
                    sp->base = run;
                }
            }
            __syncthreads();
            prefix = prefix << 8 | sp->digit;
            base = sp->base;
        }
        *above = base;
        return prefix;
    };
    if (S.top_k > 0) {
        u64 above;
        c.thr = select(false, (u64)S.top_k, &above);
        c.ties = (u64)S.top_k - above;
    }
    if (sums) {
        if (need == 0) {  // of those above thr, and `ties` at it
            u64 sum = 0;
            for (int i = tid; i < n; i += NT) {
                const unsigned k = key(i);
                if (k > c.thr) sum += W.units(logit_of(k));
            }
            sum = block_total<NT>(sum, sp->wsum);
            need = S.share_of(sum + (c.thr ? c.ties * W.units(logit_of(c.thr)) : 0));
        }
        u64 above;
        const unsigned t = select(true, need, &above);
        const u64 w = W.units(logit_of(t)), m = w ? (need - above + w - 1) / w : ~0ull;
        if (t > c.thr || c.thr == 0) c.thr = t, c.ties = m;
        else c.ties = m < c.ties ? m : c.ties;
    }
    return c;
}

// The draw among n tokens in the order of their indices, keys through key(i):
// which one it falls on and the sum it fell in, or -1 in the threads that do not
// find it.  A thread takes a run of consecutive ones.  `tied`: ties before the
// first; `target` ~0: uniform u's place in the sum, else this one.
template <int NT, class Key>
__device__ int draw_of(const Key &key, int n, const Cut &c, const RowSettings &S, const Weights &W, float u, u64 tied,
                       u64 target, u64 *total, Space *sp) {
    const int per = (n + NT - 1) / NT, lo = min((int)threadIdx.x * per, n), hi = min(lo + per, n);
    u64 before = 0, all;
    if (c.ties != ~0ull) {
        u64 count = 0;
        for (int i = lo; i < hi; i++) count += key(i) == c.thr;
        before = tied + block_scan<NT>(count, sp->wsum, &all) - count;
    }
    u64 seen = before;
    auto kept = [&](int i) {
        const unsigned k = key(i);
        if (k < c.thr || (k == c.thr && seen++ >= c.ties)) return (u64)0;
        return W.units(logit_of(k), S.least);
    };
    u64 sum = 0;
    for (int i = lo; i < hi; i++) sum += kept(i);
    const u64 upto = block_scan<NT>(sum, sp->wsum, &all);
    if (target == ~0ull) *total = all, target = S.target_of(u, all);
    if (target < upto - sum || target >= upto) return -1;
    u64 run = upto - sum;
    seen = before;
    for (int i = lo; i < hi; i++) {
        run += kept(i);
        if (run > target) return i;
    }
    return -1;
}

__device__ __forceinline__ void no_token(const SampleRowsParams &P, int r, bool bad) {
    P.tokens[r] = -1;
    if (P.probs) P.probs[r] = bad ? __uint_as_float(0x7fc00000u) : 0.0f;
}
__device__ __forceinline__ void drawn(const SampleRowsParams &P, int r, int token, double weight, u64 total) {
    P.tokens[r] = token;
    if (P.probs) P.probs[r] = (float)(weight * kUnit / (double)total);
}

// The keys of `n` candidates among the row's, at least as large as the k-th
// largest: at most top_k of the maxima of runs are above the k-th largest of
// them, so that what is below it is not among the first k.  Ranked by comparing
// all pairs; with top_k runs or fewer everything stays.
template <int NT>
__device__ unsigned least_of_runs(unsigned mine, int top_k, unsigned *tops, Space *sp) {
    if (top_k >= NT) return 0;
    tops[threadIdx.x] = mine;
    __syncthreads();
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < NT; j++) {
        const unsigned o = tops[j];
        rank += o > mine || (o == mine && j < (int)threadIdx.x);
    }
    if (rank == top_k - 1) sp->thr = mine;
    __syncthreads();
    return sp->thr;
}

constexpr int kRowVocab = 8192;  // with the lists, a block's 64 KB of LDS

template <int NT>
__global__ __launch_bounds__(NT) void k_sample_row(SampleRowsParams P) {
    constexpr int kList = 4 * NT < 2048 ? 4 * NT : 2048;  // candidates
    extern __shared__ unsigned keys[];
    __shared__ Space sp;
    __shared__ unsigned tops[NT], list[kList];
    __shared__ int place[kList];
    const int r = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    if (tid == 0) sp.top = 0, sp.bad = 0, sp.token = V;
    fill_table(sp.tab);
    __syncthreads();
    unsigned top = 0;
    bool bad = false;
    for (int i = tid; i < V; i += NT) {
        const float l = x[i];
        bad |= l != l;
        const unsigned k = key_of(l);
        keys[i] = k;
        top = max(top, k);
    }
    top = wave_top(top);
    if ((tid & 63) == 0) atomicMax(&sp.top, top);
    if (bad) atomicOr(&sp.bad, 1u);
    __syncthreads();
    top = sp.top;
    const float mx = logit_of(top);
    if (sp.bad || mx == -INFINITY) {
        if (tid == 0) no_token(P, r, sp.bad);
        return;
    }
    if (S.greedy) {
        for (int i = tid; i < V; i += NT)
            if (keys[i] == top) {
                atomicMin(&sp.token, i);
                break;
            }
        __syncthreads();
        if (tid == 0) drawn(P, r, sp.token, 1.0, (u64)kUnit);
        return;
    }
    const Weights W = weights_of(S, mx, sp.tab);
    const unsigned *set = keys;
    int n = V;
    bool listed = false;
    if (S.top_k > 0 && V > kBrute) {  // candidates, in the order of their indices
        const int per = (V + NT - 1) / NT, lo = min(tid * per, V), hi = min(lo + per, V);
        unsigned run = 0;
        for (int i = lo; i < hi; i++) run = max(run, keys[i]);
        const unsigned least = least_of_runs<NT>(run, S.top_k, tops, &sp);
        u64 count = 0, total;
        for (int i = lo; i < hi; i++) count += keys[i] >= least;
        int at = (int)(block_scan<NT>(count, sp.wsum, &total) - count);
        if (total <= kList) {
            for (int i = lo; i < hi; i++)
                if (keys[i] >= least) list[at] = keys[i], place[at++] = i;
            set = list, n = (int)total, listed = true;
            __syncthreads();
        }
    }
    auto key = [&](int j) { return set[j]; };
    const Cut c = cut_of<NT>(key, n, S, W, 0, &sp);
    u64 total;
    const int i = draw_of<NT>(key, n, c, S, W, P.u[r], 0, ~0ull, &total, &sp);
    if (i >= 0) drawn(P, r, listed ? place[i] : i, W.weight(logit_of(set[i])), total);
}

// ---------------------------------------------------------------------------
// Rows of more than kRowVocab logits
// ---------------------------------------------------------------------------
constexpr int kChunk = 4096, kGroup = 64;         // logits of a block, of a maximum
constexpr int kNear = 2048;                       // tokens next to a cut that are held
constexpr int kMaxChunks = kSampleRowsMaxVocab / kChunk, kMaxGroups = kSampleRowsMaxVocab / kGroup;

// A row's scratch.
struct RowScratch {
    u64 hist[kBins];                  // top-p without top-k: units by bin
    u64 sum[kMaxChunks];              // kept units of a chunk (of bins before the cut's)
    unsigned top[kMaxChunks];         // its largest key
    int token[kMaxChunks];            // where that is first
    unsigned bad[kMaxChunks];         // a NaN
    unsigned near_at[kMaxChunks];     // its tokens in the cut's bin, in `near`
    unsigned near_n[kMaxChunks];
    unsigned near_all;
    unsigned pad;
    unsigned near[kNear];             // keys
    unsigned group[kMaxGroups];       // the largest key of each kGroup
};

struct RowTop {
    unsigned top;
    bool bad;
};

// The row's largest key, by the chunks'; every thread of the block.
__device__ RowTop row_top(const RowScratch *R, int chunks, Space *sp) {
    const int tid = threadIdx.x;
    if (tid == 0) sp->top = 0, sp->bad = 0;
    __syncthreads();
    if (tid < chunks) {
        atomicMax(&sp->top, R->top[tid]);
        if (R->bad[tid]) atomicOr(&sp->bad, 1u);
    }
    __syncthreads();
    return {sp->top, sp->bad != 0};
}

// Logits lo + 4 i .. of a row into registers, -Inf past the last: 16 bytes a lane
// where the row's start allows it.
__device__ __forceinline__ f32x4 load_logits(const float *x, int i, int V, bool aligned) {
    if (aligned && i + 4 <= V) return *glb(reinterpret_cast<const f32x4 *>(x + i));
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = i + e < V ? x[min(i + e, V - 1)] : -INFINITY;
    return v;
}

__global__ __launch_bounds__(256) void k_sample_max(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ unsigned stop, sbad;
    __shared__ int stoken;
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const bool aligned = ((uintptr_t)x & 15) == 0;
    if (tid == 0) stop = 0, sbad = 0, stoken = V;
    for (int i = chunk * 256 + tid; i < kBins; i += gridDim.x * 256) R->hist[i] = 0;
    if (chunk == 0 && tid == 0) R->near_all = 0;
    __syncthreads();
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = load_logits(x, chunk * kChunk + 1024 * j + 4 * tid, V, aligned);
    unsigned top = 0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        unsigned g = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            bad |= v[j][e] != v[j][e];
            g = max(g, key_of(v[j][e]));
        }
        for (int off = 1; off < 16; off <<= 1) g = max(g, (unsigned)__shfl_xor((int)g, off, 64));
        top = max(top, g);
        const int at = chunk * kChunk + 1024 * j + 4 * tid;
        if ((tid & 15) == 0 && at < V) R->group[at / kGroup] = g;
    }
    top = wave_top(top);
    if ((tid & 63) == 0) atomicMax(&stop, top);
    if (bad) sbad = 1;
    __syncthreads();
    top = stop;
    int first = V;
#pragma unroll
    for (int j = 3; j >= 0; j--)
#pragma unroll
        for (int e = 3; e >= 0; e--)
            if (key_of(v[j][e]) == top) first = chunk * kChunk + 1024 * j + 4 * tid + e;
    if (first < V) atomicMin(&stoken, first);
    __syncthreads();
    if (tid == 0) R->top[chunk] = top, R->bad[chunk] = sbad, R->token[chunk] = stoken;
}

// Rows that top-k does not cut: units by bin where top-p does, else the chunk's
// sum.
__global__ __launch_bounds__(256) void k_sample_sum(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ Space sp;
    __shared__ u64 hist[kBins];
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    if (S.greedy || S.top_k > 0) return;
    const bool sums = S.cuts_sum(), aligned = ((uintptr_t)x & 15) == 0;
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = load_logits(x, chunk * kChunk + 1024 * j + 4 * tid, V, aligned);
    fill_table(sp.tab);
    if (sums)
        for (int i = tid; i < kBins; i += 256) hist[i] = 0;
    const RowTop t = row_top(R, gridDim.x, &sp);
    const float mx = logit_of(t.top);
    if (t.bad || mx == -INFINITY) return;
    const Weights W = weights_of(S, mx, sp.tab);
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float l = v[j][e];
            const u64 w = W.units(l, sums ? 0.0 : S.least);
            if (!sums) sum += w;
            else if (w) atomicAdd(&hist[W.bin(l)], w);
        }
    if (!sums) {
        sum = block_total<256>(sum, sp.wsum);
        if (tid == 0) R->sum[chunk] = sum;
        return;
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += 256)
        if (hist[i]) atomicAdd(&R->hist[i], hist[i]);
}

struct BinCut {
    int bin;    // where the sum reaches top-p's share
    u64 above;  // units of the bins before it
    u64 need;
};

template <int NT>
__device__ BinCut bin_cut(const RowScratch *R, const RowSettings &S, Space *sp) {
    constexpr int N = (kBins + NT - 1) / NT;
    u64 h[N], sum = 0, total;
#pragma unroll
    for (int i = 0; i < N; i++) sum += h[i] = (int)threadIdx.x * N + i < kBins ? R->hist[threadIdx.x * N + i] : 0;
    u64 run = block_scan<NT>(sum, sp->wsum, &total) - sum;
    const u64 need = S.share_of(total);
    if (run < need && run + sum >= need) {
        int i = 0;
        for (; i < N - 1 && run + h[i] < need; i++) run += h[i];
        sp->token = threadIdx.x * N + i;
        sp->base = run;
    }
    __syncthreads();
    return {sp->token, sp->base, need};
}

// Rows that top-p alone cuts: each chunk's kept sum before the cut's bin, and its
// tokens in it, in the order of their indices.
__global__ __launch_bounds__(256) void k_sample_near(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ Space sp;
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    if (S.greedy || S.top_k > 0 || !S.cuts_sum()) return;
    const bool aligned = ((uintptr_t)x & 15) == 0;
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = load_logits(x, chunk * kChunk + 16 * tid + 4 * j, V, aligned);
    fill_table(sp.tab);
    const RowTop t = row_top(R, gridDim.x, &sp);
    const float mx = logit_of(t.top);
    if (t.bad || mx == -INFINITY) return;
    const Weights W = weights_of(S, mx, sp.tab);
    const BinCut b = bin_cut<256>(R, S, &sp);
    u64 sum = 0, near = 0, all;
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int bin = W.bin(v[j][e]);
            if (bin < b.bin) sum += W.units(v[j][e], S.least);
            near += bin == b.bin && chunk * kChunk + 16 * tid + 4 * j + e < V;
        }
    sum = block_total<256>(sum, sp.wsum);
    unsigned at = (unsigned)(block_scan<256>(near, sp.wsum, &all) - near);
    if (tid == 0) {
        R->sum[chunk] = sum;
        R->near_n[chunk] = (unsigned)all;
        sp.digit = all ? atomicAdd(&R->near_all, (unsigned)all) : 0;
        R->near_at[chunk] = sp.digit;
    }
    __syncthreads();
    at += sp.digit;
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (W.bin(v[j][e]) == b.bin && chunk * kChunk + 16 * tid + 4 * j + e < V) {
                if (at < kNear) R->near[at] = key_of(v[j][e]);
                at++;
            }
}

// The row's end: top-k's candidates, or where the chunks' sums say the draw falls.
constexpr int kDrawThreads = 1024, kDrawList = 8192;
static_assert(kDrawList >= kMaxGroups && kDrawList >= kNear, "either lies in LDS");

__global__ __launch_bounds__(kDrawThreads) void k_sample_draw(SampleRowsParams P, RowScratch *scratch, int row0) {
    constexpr int NT = kDrawThreads;
    __shared__ Space sp;
    __shared__ unsigned keys[kDrawList];
    __shared__ int place[kDrawList];
    __shared__ unsigned short list[kMaxGroups];
    __shared__ int offset[kMaxChunks], ties[kMaxChunks];
    const int r = row0 + blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = P.vocab;
    const int chunks = (V + kChunk - 1) / kChunk, groups = (V + kGroup - 1) / kGroup;
    RowScratch *R = scratch + blockIdx.x;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    fill_table(sp.tab);
    const RowTop t = row_top(R, chunks, &sp);
    const float mx = logit_of(t.top);
    if (t.bad || mx == -INFINITY) {
        if (tid == 0) no_token(P, r, t.bad);
        return;
    }
    if (S.greedy) {
        if (tid == 0) sp.token = V;
        __syncthreads();
        if (tid < chunks && R->top[tid] == t.top) atomicMin(&sp.token, R->token[tid]);
        __syncthreads();
        if (tid == 0) drawn(P, r, sp.token, 1.0, (u64)kUnit);
        return;
    }
    const Weights W = weights_of(S, mx, sp.tab);
    const float u = P.u[r];
    auto far_key = [&](int i) { return key_of(x[i]); };
    auto near_key = [&](int i) { return keys[i]; };
    auto whole = [&]() {  // the row by its keys' digits, from memory: many passes
        const Cut c = cut_of<NT>(far_key, V, S, W, 0, &sp);
        u64 total;
        const int i = draw_of<NT>(far_key, V, c, S, W, u, 0, ~0ull, &total, &sp);
        if (i >= 0) drawn(P, r, i, W.weight(x[i]), total);
    };
    u64 total;
    if (S.top_k > 0) {
        // Candidates: as large as the top_k-th largest of the groups' maxima, from
        // the groups that have such (to within a few times top_k tokens; many
        // equal logits, or top_k past a few thousand, take the whole row).
        for (int i = tid; i < groups; i += NT) keys[i] = R->group[i];
        __syncthreads();
        unsigned least = 0;
        if (S.top_k < groups) {
            RowSettings count = S;
            count.top_p = 1.0f;
            least = cut_of<NT>(near_key, groups, count, W, 0, &sp).thr;
        }
        const int per = (groups + NT - 1) / NT, lo = min(tid * per, groups), hi = min(lo + per, groups);
        u64 n = 0, all;
        for (int i = lo; i < hi; i++) n += keys[i] >= least;
        int at = (int)(block_scan<NT>(n, sp.wsum, &all) - n);
        for (int i = lo; i < hi; i++)
            if (keys[i] >= least) list[at++] = (unsigned short)i;
        __syncthreads();
        // a wave's run of those groups, four at a time: counted, then written in
        // the order of their indices
        const int run = ((int)all + NT / 64 - 1) / (NT / 64);
        const int g0 = min(wave * run, (int)all), g1 = min(g0 + run, (int)all);
        auto each = [&](auto take) {
            for (int g = g0; g < g1; g += 4) {
                unsigned k[4];
                int i[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    i[j] = list[min(g + j, g1 - 1)] * kGroup + lane;
                    k[j] = key_of(x[min(i[j], V - 1)]);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) take(i[j], k[j], g + j < g1 && i[j] < V && k[j] >= least);
            }
        };
        u64 mine = 0;
        each([&](int, unsigned, bool in) { mine += __popcll(__ballot(in)); });
        if (lane == 0) sp.wsum[wave] = mine;
        __syncthreads();
        int to = 0, have = 0;
        for (int w = 0; w < NT / 64; w++) {
            if (w < wave) to += (int)sp.wsum[w];
            have += (int)sp.wsum[w];
        }
        if (have > kDrawList) return whole();
        each([&](int i, unsigned k, bool in) {
            const u64 who = __ballot(in);
            if (in) {
                const int p = to + __popcll(who & ((1ull << lane) - 1));
                keys[p] = k, place[p] = i;
            }
            to += __popcll(who);
        });
        __syncthreads();
        const Cut c = cut_of<NT>(near_key, have, S, W, 0, &sp);
        const int i = draw_of<NT>(near_key, have, c, S, W, u, 0, ~0ull, &total, &sp);
        if (i >= 0) drawn(P, r, place[i], W.weight(logit_of(keys[i])), total);
        return;
    }
    Cut c;
    u64 part = tid < chunks ? R->sum[tid] : 0;
    if (S.cuts_sum()) {
        const BinCut b = bin_cut<NT>(R, S, &sp);
        const unsigned mine = tid < chunks ? R->near_n[tid] : 0;
        u64 all;
        const int first = (int)(block_scan<NT>(mine, sp.wsum, &all) - mine);
        if (all > kNear) return whole();  // many equal or nearly equal logits
        if (tid < chunks) offset[tid] = first;
        __syncthreads();
        for (int k = wave; k < chunks; k += NT / 64) {
            const int n = (int)R->near_n[k], from = (int)R->near_at[k];
            for (int j = lane; j < n; j += 64) keys[offset[k] + j] = R->near[from + j];
        }
        __syncthreads();
        c = cut_of<NT>(near_key, (int)all, S, W, b.need - b.above, &sp);
        // each chunk's ties and kept sum
        u64 count = 0, before;
        for (unsigned j = 0; j < mine; j++) count += keys[first + j] == c.thr;
        before = block_scan<NT>(count, sp.wsum, &all) - count;
        if (tid < chunks) ties[tid] = (int)before;
        for (unsigned j = 0; j < mine; j++) {
            const unsigned k = keys[first + j];
            if (k > c.thr || (k == c.thr && before++ < c.ties)) part += W.units(logit_of(k), S.least);
        }
    } else if (tid < chunks) {
        ties[tid] = 0;
    }
    const u64 upto = block_scan<NT>(part, sp.wsum, &total);
    u64 target = S.target_of(u, total);
    if (target >= upto - part && target < upto) sp.token = tid, sp.base = upto - part;
    __syncthreads();
    const int chunk = sp.token, i0 = chunk * kChunk;
    target -= sp.base;
    const int i = draw_of<NT>([&](int j) { return far_key(i0 + j); }, min(kChunk, V - i0), c, S, W, u,
                              (u64)ties[chunk], target, &total, &sp);
    if (i >= 0) drawn(P, r, i0 + i, W.weight(x[i0 + i]), total);
}

}  // namespace

void launch_sample_rows(hipStream_t st, const SampleRowsParams &p) {
    if (p.vocab <= kRowVocab) {
        const unsigned lds = (unsigned)p.vocab * 4;
        if (p.vocab <= 4096) hipLaunchKernelGGL(k_sample_row<256>, dim3((unsigned)p.rows), dim3(256), lds, st, p);
        else hipLaunchKernelGGL(k_sample_row<1024>, dim3((unsigned)p.rows), dim3(1024), lds, st, p);
        return;
    }
    RowScratch *scratch = static_cast<RowScratch *>(p.scratch);
    const int most = (int)std::min<size_t>(p.scratch_bytes / sizeof(RowScratch), 1024);
    const unsigned chunks = (unsigned)((p.vocab + kChunk - 1) / kChunk);
    for (int row0 = 0; row0 < p.rows; row0 += most) {
        const unsigned n = (unsigned)std::min(most, p.rows - row0);
        hipLaunchKernelGGL(k_sample_max, dim3(chunks, n), dim3(256), 0, st, p, scratch, row0);
        hipLaunchKernelGGL(k_sample_sum, dim3(chunks, n), dim3(256), 0, st, p, scratch, row0);
        if (p.p.top_p) hipLaunchKernelGGL(k_sample_near, dim3(chunks, n), dim3(256), 0, st, p, scratch, row0);
        hipLaunchKernelGGL(k_sample_draw, dim3(n), dim3(kDrawThreads), 0, st, p, scratch, row0);
    }
}

}  // namespace qtts
