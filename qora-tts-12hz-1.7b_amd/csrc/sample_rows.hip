// sample_rows.hip — a token from each row of logits: temperature, top-k,
// top-p, min-p, given uniform numbers.
//
// Weights w_i = exp((l_i - max) / T) are evaluated in 64 bits and summed as
// integers of 2^-44 of the largest, each to the nearest: sums do not depend on
// their order, and a draw falls as the 64-bit definition's does but within 2^-45 a
// token of the border between two.  What is kept is a prefix of the tokens in order (logit down, index up),
// so that it is one number, the order of the last.
//
// Rows of up to kRowVocab logits take a block each, which holds the row's keys
// in LDS (k_sample_row).  Longer rows are read in chunks by as many blocks as
// they have: their maxima (k_sample_max); where top-k's candidates end, or the
// sums by weight (k_sample_sum); the candidates next to the cut
// (k_sample_near).  One block a row joins them and draws (k_sample_draw).
//
// Measured: 64 rows of 151936, settings of every kind among them, 14 + 12 + 13
// + 25 us (39 MB, which a copy reads in 8); all at top_k = 50, 14 + 9 + 7 + 10;
// one row 6 + 7 + 4 + 9 us, all of it latency.  Rows of more than kNear candidates
// (top_k past the groups that hold a finite logit, thousands of equal or masked
// but finite ones) are cut from memory by one block: 0.2 to 1.1 ms a row of 151936,
// 0.3 to 1.5 for 64.
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

// The order of a row's tokens: larger logits first, equal ones by index.  What
// top-k and top-p keep is all from some order on, the cut.
__device__ __forceinline__ u64 order_of(unsigned key, int i) { return (u64)key << 32 | (unsigned)~i; }
__device__ __forceinline__ unsigned key_in(u64 order) { return (unsigned)(order >> 32); }
__device__ __forceinline__ int index_in(u64 order) { return (int)~(unsigned)order; }

constexpr int kBrute = 256;  // a set this small is ranked by comparing all pairs

struct Space {
    double tab[64];
    u64 hist[256], wsum[16], near[kBrute], units[kBrute], base, cut;
    unsigned rank[kBrute], digit, count, thr, top, bad;
    int token;
};

__device__ __forceinline__ u64 readlane64(u64 v, int j) {
    return (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, j) |
           (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), j) << 32;
}

// The cut of the n <= kBrute orders in sp->near (as they come), of which the first
// `count` stay (0: all) and then, where `by_sum`, those whose predecessors' sum and
// `above` is below `need` (0: top-p's share of the sum).  A lane holds every 64th
// of them and a wave compares all with its share, which it has in scalar
// registers: two instructions a pair, six with the sum (226 by count 2.8 us, 215 by
// sum 6.2; with each pair read from LDS and the cut by an atomic minimum 7.4 both).
template <int NT>
__device__ u64 rank_near(int n, u64 count, bool by_sum, u64 above, u64 need, const RowSettings &S, const Weights &W,
                         Space *sp) {
    constexpr int J = kBrute / (NT / 64), A = kBrute / 64;
    const int tid = threadIdx.x, lane = tid & 63, j0 = __builtin_amdgcn_readfirstlane(tid >> 6) * J;
    u64 *ahead = sp->hist;
    __syncthreads();
    u64 mine = 0;
    if (tid < n) {
        sp->rank[tid] = 0, ahead[tid] = 0;
        if (by_sum) mine = W.units(logit_of(key_in(sp->near[tid])));
        sp->units[tid] = mine;
    }
    if (tid == 0) sp->cut = 0;
    __syncthreads();
    u64 order[A], sum[A];
    unsigned rank[A];
#pragma unroll
    for (int a = 0; a < A; a++) {
        order[a] = 64 * a + lane < n ? sp->near[64 * a + lane] : ~0ull;
        sum[a] = 0, rank[a] = 0;
    }
    const u64 share = sp->near[min(j0 + lane, kBrute - 1)], weigh = sp->units[min(j0 + lane, kBrute - 1)];
    const int jn = min(J, n - j0);
    if (by_sum) {
        for (int j = 0; j < jn; j++) {
            const u64 o = readlane64(share, j), w = readlane64(weigh, j);
#pragma unroll
            for (int a = 0; a < A; a++) {
                const bool before = o > order[a];
                rank[a] += before;
                sum[a] += before ? w : 0;
            }
        }
    } else {
        for (int j = 0; j < jn; j++) {
            const u64 o = readlane64(share, j);
#pragma unroll
            for (int a = 0; a < A; a++) rank[a] += o > order[a];
        }
    }
    if (jn > 0) {
#pragma unroll
        for (int a = 0; a < A; a++)
            if (64 * a + lane < n) {
                atomicAdd(&sp->rank[64 * a + lane], rank[a]);
                if (by_sum) atomicAdd(&ahead[64 * a + lane], sum[a]);
            }
    }
    __syncthreads();
    const bool keep = tid < n && (count == 0 || sp->rank[tid] < count);
    if (by_sum) {  // the last that stays is where the sum arrives
        const u64 before = tid < n ? above + ahead[tid] : 0;
        if (need == 0) need = S.share_of(block_total<NT>(keep ? mine : 0, sp->wsum));
        if (keep && before < need && before + mine >= need) sp->cut = sp->near[tid];
    } else if (keep && sp->rank[tid] == count - 1) {
        sp->cut = sp->near[tid];
    }
    __syncthreads();
    return sp->cut;
}

// A logit's place among 2^16 equal steps from `hi` down to `lo` (halves, so that
// the difference stays in range; what lies outside goes to the ends).
struct Line {
    float hi, scale;
    __device__ __forceinline__ Line(float from, float to) : hi(from) {
        const float range = 0.5f * from - 0.5f * to;
        scale = range > 0.0f ? 65535.0f / range : 0.0f;
        if (!(scale < INFINITY)) scale = 3e38f;
    }
    __device__ __forceinline__ int operator()(unsigned k) const {
        const float l = logit_of(k);
        return l >= hi ? 0 : (int)fminf((0.5f * hi - 0.5f * l) * scale, 65535.0f);
    }
};

// Where the sums of 256 bins, on top of `base`, reach `want` (the last where they
// don't): sp->digit, and sp->base the sum before it.  By the first wave, for all
// after the barrier.
__device__ __forceinline__ void find_bin(bool down, u64 want, u64 base, Space *sp) {
    const int tid = threadIdx.x;
    if (tid < 64) {
        u64 h[4], sum = 0;
        for (int j = 0; j < 4; j++) sum += h[j] = sp->hist[down ? 255 - 4 * tid - j : 4 * tid + j];
        u64 run = base + wave_scan(sum) - sum;
        const bool mine = run < want && run + sum >= want, none = !__any(mine);
        if (mine || (none && tid == 63)) {
            int j = 0;
            for (; j < 3 && run + h[j] < want; j++) run += h[j];
            sp->digit = down ? 255 - 4 * tid - j : 4 * tid + j;
            sp->base = run;
        }
    }
    __syncthreads();
}

// The order, from `cut` on, at which the count or the sum of n keys reaches
// `want`: by the keys' places on a line, 8 bits at a time, until what shares the
// step is a small set (many equal ones: by the keys' digits, then by index).
// `found`: the first 8 bits are in sp->digit, the sum before them in sp->base.
template <int NT, class Key>
__device__ u64 select(const Key &key, int n, const Line &line, u64 cut, bool by_sum, u64 want, bool found,
                      const RowSettings &S, const Weights &W, Space *sp) {
    const int tid = threadIdx.x;
    u64 base = 0;
    int at = 0;  // the chosen step's first bits
    for (int shift = 8; shift >= 0; shift -= 8) {
        if (!found) {
            __syncthreads();
            for (int i = tid; i < 256; i += NT) sp->hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += NT) {
                const unsigned k = key(i);
                if (order_of(k, i) < cut) continue;
                const int p = line(k);
                if (shift == 0 && p >> 8 != at) continue;
                const u64 w = by_sum ? W.units(logit_of(k)) : (u64)1;
                if (w) atomicAdd(&sp->hist[p >> shift & 255], w);
            }
            __syncthreads();
            find_bin(false, want, base, sp);
        }
        found = false;
        at = at << 8 | (int)sp->digit;
        base = sp->base;
        if (tid == 0) sp->count = 0;
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
            const unsigned k = key(i);
            if (order_of(k, i) < cut || line(k) >> shift != at) continue;
            const unsigned to = atomicAdd(&sp->count, 1u);
            if (to < kBrute) sp->near[to] = order_of(k, i);
        }
        __syncthreads();
        const int all = (int)sp->count;
        if (all <= kBrute)
            return by_sum ? rank_near<NT>(all, 0, true, base, want, S, W, sp)
                          : rank_near<NT>(all, want - base, false, 0, 0, S, W, sp);
    }
    unsigned prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = tid; i < 256; i += NT) sp->hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
            const unsigned k = key(i);
            if (order_of(k, i) < cut || line(k) != at || (shift < 24 && k >> (shift + 8) != prefix)) continue;
            const u64 w = by_sum ? W.units(logit_of(k)) : (u64)1;
            if (w) atomicAdd(&sp->hist[k >> shift & 255], w);
        }
        __syncthreads();
        find_bin(true, want, base, sp);
        prefix = prefix << 8 | sp->digit;
        base = sp->base;
    }
    const u64 w = by_sum ? W.units(logit_of(prefix)) : (u64)1;
    if (w == 0) return order_of(prefix, 0x7fffffff);
    const u64 nth = (want - base + w - 1) / w;  // of those equal to it the last that stays
    const int per = (n + NT - 1) / NT, lo = min(tid * per, n), hi = min(lo + per, n);
    u64 count = 0, all;
    for (int i = lo; i < hi; i++) count += key(i) == prefix;
    u64 seen = block_scan<NT>(count, sp->wsum, &all) - count;
    if (tid == 0) sp->token = 0x7fffffff;
    __syncthreads();
    if (seen < nth && seen + count >= nth)
        for (int i = lo; i < hi; i++)
            if (key(i) == prefix && ++seen == nth) sp->token = i;
    __syncthreads();
    return order_of(prefix, sp->token);
}

// The cut that top-k and top-p make in n keys, key(i) in the order of their
// indices, which lie between lo and hi for the most part (0: none); `need`: the sum
// that top-p's prefix reaches, 0: its share of the sum.  `found`: as for select,
// by line's first 8 bits, for the first that cuts.
template <int NT, class Key>
__device__ u64 cut_of(const Key &key, int n, const Line &line, bool found, const RowSettings &S, const Weights &W,
                      u64 need, Space *sp) {
    const int tid = threadIdx.x;
    const bool counts = S.top_k > 0 && S.top_k < n, sums = S.cuts_sum();
    u64 cut = 0;
    if (!counts && !sums) return cut;
    if (n <= kBrute && !found) {
        __syncthreads();
        if (tid < n) sp->near[tid] = order_of(key(tid), tid);
        return rank_near<NT>(n, counts ? S.top_k : 0, sums, 0, need, S, W, sp);
    }
    if (counts) cut = select<NT>(key, n, line, cut, false, (u64)S.top_k, found, S, W, sp);
    if (!sums) return cut;
    if (need == 0) {
        u64 sum = 0;
        for (int i = tid; i < n; i += NT) {
            const unsigned k = key(i);
            if (order_of(k, i) >= cut) sum += W.units(logit_of(k));
        }
        need = S.share_of(block_total<NT>(sum, sp->wsum));
    }
    const u64 least = select<NT>(key, n, line, cut, true, need, found && !counts, S, W, sp);
    return least > cut ? least : cut;
}

// The draw among n tokens in the order of their indices, keys through key(i), the
// first at `first` in the cut's terms: which one it falls on, or -1 in the threads
// that do not find it.  A thread takes a run of consecutive ones.  `target` ~0:
// uniform u's place in the sum, else this one.
template <int NT, class Key>
__device__ int draw_of(const Key &key, int first, int n, u64 cut, const RowSettings &S, const Weights &W, float u,
                       u64 target, u64 *total, Space *sp) {
    const int per = (n + NT - 1) / NT, lo = min((int)threadIdx.x * per, n), hi = min(lo + per, n);
    auto kept = [&](int i) {
        const unsigned k = key(i);
        return order_of(k, first + i) >= cut ? W.units(logit_of(k), S.least) : (u64)0;
    };
    u64 sum = 0, all;
    for (int i = lo; i < hi; i++) sum += kept(i);
    const u64 upto = block_scan<NT>(sum, sp->wsum, &all);
    if (target == ~0ull) *total = all, target = S.target_of(u, all);
    if (target < upto - sum || target >= upto) return -1;
    u64 run = upto - sum;
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

// The whole end of a row whose candidates are at most a wave: n keys in the order
// of their indices, cut and drawn from without a barrier.  place(i): the index.
template <class Place>
__device__ void finish_wave(const SampleRowsParams &P, int r, unsigned k, int n, const Place &place,
                            const RowSettings &S, const Weights &W, u64 need) {
    const int lane = threadIdx.x & 63;
    const bool in = lane < n, sums = S.cuts_sum();
    const float l = logit_of(k);
    const u64 mine = in ? W.units(l) : 0;
    unsigned rank = 0;
    u64 ahead = 0;
    for (int j = 0; j < n; j++) {
        const unsigned o = (unsigned)__builtin_amdgcn_readlane((int)k, j);
        const u64 w = readlane64(mine, j);
        const bool before = o > k || (o == k && j < lane);
        rank += before;
        ahead += before ? w : 0;
    }
    bool keep = in && (S.top_k == 0 || rank < (unsigned)S.top_k);
    if (sums) {
        if (need == 0) need = S.share_of(wave_total(keep ? mine : 0));
        keep = keep && ahead < need;
    }
    const u64 kept = keep && W.weight(l) >= S.least ? mine : 0;
    const u64 upto = wave_scan(kept), total = (u64)__shfl((long long)upto, 63, 64);
    const u64 target = S.target_of(P.u[r], total);
    if (target >= upto - kept && target < upto) drawn(P, r, place(lane), W.weight(l), total);
}

// Four logits of a row from the i-th, -Inf past the last: 16 bytes a lane where
// the row's start allows it.
__device__ __forceinline__ f32x4 load_logits(const float *x, int i, int V, bool aligned) {
    if (aligned && i + 4 <= V) return *glb(reinterpret_cast<const f32x4 *>(x + i));
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = i + e < V ? x[min(i + e, V - 1)] : -INFINITY;
    return v;
}

// Rows that one block takes, in 48 KB of its LDS: 64 of 12000 logits in 35 us,
// in chunks 61; one in 11 us, in chunks 16.
constexpr int kRowVocab = 12288;

// Bound by its steps' barriers and latencies, not by its bytes (64 rows of 2048:
// 512 KB): 11 us where 50 tokens are kept and a wave finishes them, 16 us where
// top-k and top-p both cut among many.  256 threads a row up to 1024 logits, which
// have no more than four each (64 rows of 300: 11 us, with 1024 threads 12.5; of
// 1500: 17 and 14).
template <int NT>
__global__ __launch_bounds__(NT) void k_sample_row(SampleRowsParams P, int row0) {
    extern __shared__ unsigned keys[];
    __shared__ Space sp;
    __shared__ unsigned sleast;
    __shared__ int place[64];
    const int r = row0 + blockIdx.x, tid = threadIdx.x, V = P.vocab;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    const bool aligned = ((uintptr_t)x & 15) == 0;
    if (tid == 0) sp.top = 0, sp.bad = 0, sp.token = V, sleast = 0xffffffffu;
    fill_table(sp.tab);
    for (int i = tid; i < 256; i += NT) sp.hist[i] = 0;
    __syncthreads();
    unsigned top = 0, least = 0xffffffffu;
    bool bad = false;
    for (int i0 = 4 * tid; i0 < V; i0 += 8 * NT) {  // two loads in flight
        f32x4 v[2];
#pragma unroll
        for (int j = 0; j < 2; j++) v[j] = load_logits(x, i0 + 4 * NT * j, V, aligned);
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = i0 + 4 * NT * j + e;
                bad |= v[j][e] != v[j][e];
                const unsigned k = key_of(v[j][e]);
                if (i < V) keys[i] = k;
                top = max(top, k);
                least = min(least, v[j][e] > -INFINITY ? k : 0xffffffffu);
            }
    }
    top = wave_top(top), least = ~wave_top(~least);
    if ((tid & 63) == 0) atomicMax(&sp.top, top), atomicMin(&sleast, least);
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
    auto key = [&](int j) { return keys[j]; };
    const float lo = logit_of(sleast), far = mx - 32.0f * S.t;  // 46 octaves: no weights past them
    const Line line(mx, S.top_k == 0 && far > lo ? far : lo);
    u64 need = 0, total;
    if (S.top_k > 0 || S.cuts_sum()) {
        // Steps down from the largest to the one where top-k's count or top-p's
        // sum is reached; a wave's worth of tokens ends here.
        const bool by_sum = S.top_k == 0;
        u64 sum = 0;
        for (int i = tid; i < V; i += NT) {
            const unsigned k = keys[i];
            const u64 w = by_sum ? W.units(logit_of(k)) : (u64)1;
            if (w) atomicAdd(&sp.hist[line(k) >> 8], w);
            sum += w;
        }
        if (by_sum) need = S.share_of(block_total<NT>(sum, sp.wsum));
        __syncthreads();
        find_bin(false, by_sum ? need : (u64)S.top_k, 0, &sp);
        const int bin = (int)sp.digit;
        const int per = (V + NT - 1) / NT, lo_i = min(tid * per, V), hi_i = min(lo_i + per, V);
        u64 count = 0, n;
        for (int i = lo_i; i < hi_i; i++) count += line(keys[i]) >> 8 <= bin;
        int at = (int)(block_scan<NT>(count, sp.wsum, &n) - count);
        if (n <= 64) {
            for (int i = lo_i; i < hi_i; i++)
                if (line(keys[i]) >> 8 <= bin) place[at++] = i;
            __syncthreads();
            if (tid < 64)
                finish_wave(P, r, tid < (int)n ? keys[place[tid]] : 0, (int)n, [&](int i) { return place[i]; }, S, W, need);
            return;
        }
    }
    const u64 cut = cut_of<NT>(key, V, line, true, S, W, need, &sp);
    const int i = draw_of<NT>(key, 0, V, cut, S, W, P.u[r], ~0ull, &total, &sp);
    if (i >= 0) drawn(P, r, i, W.weight(logit_of(keys[i])), total);
}

// ---------------------------------------------------------------------------
// Rows of more than kRowVocab logits
// ---------------------------------------------------------------------------
constexpr int kChunk = 4096;                      // logits of a block
constexpr int kNear = 8192;                       // tokens next to a cut that are held
constexpr int kMaxChunks = kSampleRowsMaxVocab / kChunk;
constexpr int kMaxGroups = 8192;

// Logits of a maximum.  A top-k past the number of groups with a finite logit takes
// every such logit for a candidate, and the whole row from memory where those are
// more than are held, so groups are as small as their places allow (64 rows of 32000, top_k =
// 2000 and top-p among the settings: 121 us in groups of 16, 45 of 4).
__host__ __device__ constexpr int group_of(int vocab) {
    return vocab <= 4 * kMaxGroups ? 4 : vocab <= 16 * kMaxGroups ? 16 : 64;
}
static_assert(kSampleRowsMaxVocab <= 64 * kMaxGroups, "the groups fit");

// A row's scratch.
struct RowScratch {
    u64 hist[kBins];                  // top-p without top-k: units by bin
    u64 sum[kMaxChunks];              // kept units of a chunk (of bins before the cut's)
    unsigned top[kMaxChunks];         // its largest key
    int token[kMaxChunks];            // where that is first
    unsigned bad[kMaxChunks];         // a NaN
    unsigned low[kMaxChunks];         // the least of its groups' maxima above -Inf
    unsigned least_key[kMaxChunks];   // and of its logits
    unsigned near_at[kMaxChunks];     // its candidates (of top-p: in the cut's bin), in `near`
    unsigned near_n[kMaxChunks];
    unsigned near_all;
    float least;                      // top-k's candidates are no smaller; +Inf: a NaN in the row
    unsigned near[kNear];             // keys
    int near_i[kNear];                // and indices
    unsigned group[kMaxGroups];       // the largest key of each group
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

// The largest key of each group and chunk, and where the chunk's is first.  Bound
// by memory: one load of the row, 16 bytes a lane and four in flight (64 rows of
// 151936 in 14 us: 2.8 TB/s, from HBM).
template <int G>
__global__ __launch_bounds__(256) void k_sample_max(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ unsigned stop, sbad, slow, sleast;
    __shared__ int stoken;
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const bool aligned = ((uintptr_t)x & 15) == 0;
    if (tid == 0) stop = 0, sbad = 0, slow = sleast = 0xffffffffu, stoken = V;
    for (int i = chunk * 256 + tid; i < kBins; i += gridDim.x * 256) R->hist[i] = 0;
    if (chunk == 0 && tid == 0) R->near_all = 0;
    __syncthreads();
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = load_logits(x, chunk * kChunk + 1024 * j + 4 * tid, V, aligned);
    constexpr int lanes = G / 4;  // of a group
    unsigned top = 0, low = 0xffffffffu, least = 0xffffffffu;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        unsigned g = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            bad |= v[j][e] != v[j][e];
            g = max(g, key_of(v[j][e]));
            least = min(least, v[j][e] > -INFINITY ? key_of(v[j][e]) : 0xffffffffu);
        }
        for (int off = 1; off < lanes; off <<= 1) g = max(g, (unsigned)__shfl_xor((int)g, off, 64));
        top = max(top, g);
        low = min(low, g > key_of(-INFINITY) ? g : 0xffffffffu);
        const int at = chunk * kChunk + 1024 * j + 4 * tid;
        if ((tid & (lanes - 1)) == 0 && at < V) R->group[at / (4 * lanes)] = g;
    }
    top = wave_top(top), low = ~wave_top(~low), least = ~wave_top(~least);
    if ((tid & 63) == 0) atomicMax(&stop, top), atomicMin(&slow, low), atomicMin(&sleast, least);
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
    if (tid == 0) R->top[chunk] = top, R->bad[chunk] = sbad, R->low[chunk] = slow, R->least_key[chunk] = sleast, R->token[chunk] = stoken;
}

// What top-k's candidates are no smaller than: a value that top_k of the groups'
// maxima reach, by 256 steps down from the largest.  A group of -Inf alone holds no
// candidate and is not counted (-Inf is never drawn); where fewer than top_k are
// left, as in rows of which few tokens are allowed, the maxima say nothing of what
// lies behind them in their groups, and it is the least finite logit.
__device__ void find_least(RowScratch *R, const RowSettings &S, int chunks, int groups, Space *sp) {
    constexpr int N = kMaxGroups / 256;  // all in flight, and kept for both passes
    const int tid = threadIdx.x;
    unsigned g[N];
#pragma unroll
    for (int j = 0; j < N; j++) g[j] = R->group[min(tid + j * 256, groups - 1)];
    const int mine = min(tid, chunks - 1);
    const unsigned low_group = R->low[mine], low_logit = R->least_key[mine];
    unsigned *lowest = sp->rank;  // of the logits
    if (tid == 0) sp->thr = 0xffffffffu, sp->count = 0xffffffffu, *lowest = 0xffffffffu;
    sp->hist[tid] = 0;
    const RowTop t = row_top(R, chunks, sp);
    float least = INFINITY;
    if (!t.bad) {
        // (a wave's own least first: an atomic minimum goes through its lanes one by one)
        const unsigned wave_group = ~wave_top(tid < chunks ? ~low_group : 0);
        const unsigned wave_logit = ~wave_top(tid < chunks ? ~low_logit : 0);
        if ((tid & 63) == 0) atomicMin(&sp->thr, wave_group), atomicMin(lowest, wave_logit);
        __syncthreads();
        const Line line(logit_of(t.top), logit_of(sp->thr));
        auto each = [&](auto take) {
#pragma unroll
            for (int j = 0; j < N; j++)
                if (tid + j * 256 < groups) take(g[j]);
        };
        each([&](unsigned k) {
            if (k > key_of(-INFINITY)) atomicAdd(&sp->hist[line(k) >> 8], (u64)1);
        });
        __syncthreads();
        find_bin(false, (u64)S.top_k, 0, sp);
        const int bin = (int)sp->digit;
        if (sp->base + sp->hist[bin] >= (u64)S.top_k) {
            unsigned low = 0xffffffffu;
            each([&](unsigned k) { low = min(low, line(k) >> 8 <= bin && k > key_of(-INFINITY) ? k : 0xffffffffu); });
            low = ~wave_top(~low);
            if ((tid & 63) == 0) atomicMin(&sp->count, low);
            __syncthreads();
            least = logit_of(sp->count);
        } else {
            least = logit_of(*lowest);
        }
    }
    if (tid == 0) R->least = least;
}

// Rows that top-k cuts: where its candidates end.  Others: units by bin where
// top-p cuts them, else the chunk's sum.  Bound by the 64-bit exponentials and,
// by bin, the atomic sums in LDS (20 of 64 rows of 151936: 12 us).
__global__ __launch_bounds__(256) void k_sample_sum(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ Space sp;
    __shared__ u64 hist[kBins];
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    if (S.greedy || (S.top_k > 0 && chunk > 0)) return;
    if (S.top_k > 0) return find_least(R, S, gridDim.x, (V + group_of(V) - 1) / group_of(V), &sp);
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

// A chunk's candidates, in the order of their indices.  For rows that top-k cuts:
// what may be among the first top_k, from the groups whose maximum may.  (By the
// one block that ends the row that took 36 us at 152000 logits and top_k = 2000,
// bound by its instructions; here, beside other rows, 13.)  For rows that top-p
// alone cuts: what shares the cut's bin, and the kept sum before that.
__global__ __launch_bounds__(256) void k_sample_near(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ Space sp;
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    const bool first = S.top_k > 0;
    if (S.greedy || !(first || S.cuts_sum())) return;
    const int i0 = chunk * kChunk + 16 * tid;
    const bool aligned = ((uintptr_t)x & 15) == 0;
    const float least = first ? R->least : 0.0f;
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = -INFINITY;
    unsigned most = 0;  // of the groups that hold the 16
    if (first && i0 < V) {
        const unsigned *g = R->group + i0 / group_of(V);
        if (group_of(V) == 4)
            for (int e = 0; e < 4; e++) most = max(most, g[min(e, (V - i0 + 3) / 4 - 1)]);
        else most = *g;
    }
    if (i0 < V && (!first || most >= key_of(least))) {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = load_logits(x, i0 + 4 * j, V, aligned);
    }
    unsigned in = 0;  // which of the 16
    u64 sum = 0, all;
    if (first) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) in |= (unsigned)(v[j][e] >= least) << (4 * j + e);
    } else {
        fill_table(sp.tab);
        const RowTop t = row_top(R, gridDim.x, &sp);
        const float mx = logit_of(t.top);
        if (t.bad || mx == -INFINITY) return;
        const Weights W = weights_of(S, mx, sp.tab);
        const BinCut b = bin_cut<256>(R, S, &sp);
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int bin = W.bin(v[j][e]);
                if (bin < b.bin) sum += W.units(v[j][e], S.least);
                in |= (unsigned)(bin == b.bin && i0 + 4 * j + e < V) << (4 * j + e);
            }
        sum = block_total<256>(sum, sp.wsum);
    }
    unsigned at = (unsigned)(block_scan<256>((u64)__popc(in), sp.wsum, &all) - __popc(in));
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
            if (in >> (4 * j + e) & 1) {
                if (at < kNear) R->near[at] = key_of(v[j][e]), R->near_i[at] = i0 + 4 * j + e;
                at++;
            }
}

// The row's end: top-k's candidates, or where the chunks' sums say the draw falls.
// A row's few thousand candidates keep one block busy for up to 25 us (top_k =
// 2000 and top-p after it: two cuts of 8 us), a few for 9.
constexpr int kDrawThreads = 1024;

__global__ __launch_bounds__(kDrawThreads) void k_sample_draw(SampleRowsParams P, RowScratch *scratch, int row0) {
    constexpr int NT = kDrawThreads;
    __shared__ Space sp;
    __shared__ unsigned keys[kNear];
    __shared__ int place[kNear];
    __shared__ int offset[kMaxChunks];
    const int r = row0 + blockIdx.x, tid = threadIdx.x, V = P.vocab, chunks = (V + kChunk - 1) / kChunk;
    RowScratch *R = scratch + blockIdx.x;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    // asked for with the first loads, where they are needed or not
    const int mine_at = min(tid, chunks - 1);
    const unsigned near_n = R->near_n[mine_at], near_at = R->near_at[mine_at];
    const float u = P.u[r], least = R->least;
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
    auto far_key = [&](int i) { return key_of(x[i]); };
    auto near_key = [&](int i) { return keys[i]; };
    auto whole = [&]() {  // the row from memory: many passes
        const u64 cut = cut_of<NT>(far_key, V, Line(mx, mx - 32.0f * S.t), false, S, W, 0, &sp);
        u64 total;
        const int i = draw_of<NT>(far_key, 0, V, cut, S, W, u, ~0ull, &total, &sp);
        if (i >= 0) drawn(P, r, i, W.weight(x[i]), total);
    };
    u64 total;
    // Candidates into LDS, in the order of their indices.
    const unsigned mine = tid < chunks ? near_n : 0;
    unsigned first = 0;
    u64 held = 0;
    if (S.top_k > 0 || S.cuts_sum()) {
        first = (unsigned)(block_scan<NT>(mine, sp.wsum, &held) - mine);
        if (held > kNear) return whole();  // many equal logits, or top_k past a few thousand
        if (tid < chunks) offset[tid] = (int)first - (int)near_at;
        __syncthreads();
        for (int j0 = tid; j0 < (int)held; j0 += 4 * NT) {
            unsigned k[4];
            int i[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int at = min(j0 + j * NT, (int)held - 1);
                k[j] = R->near[at], i[j] = R->near_i[at];
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j0 + j * NT < (int)held) {
                    const int at = j0 + j * NT + offset[i[j] / kChunk];
                    keys[at] = k[j], place[at] = i[j];
                }
        }
        __syncthreads();
    }
    if (S.top_k > 0) {
        const int n = (int)held;
        if (n <= 64) {
            if (tid < 64) finish_wave(P, r, tid < n ? keys[tid] : 0, n, [&](int i) { return place[i]; }, S, W, 0);
            return;
        }
        const u64 cut = cut_of<NT>(near_key, n, Line(mx, least), false, S, W, 0, &sp);
        const int i = draw_of<NT>(near_key, 0, n, cut, S, W, u, ~0ull, &total, &sp);
        if (i >= 0) drawn(P, r, place[i], W.weight(logit_of(keys[i])), total);
        return;
    }
    u64 cut = 0, part = tid < chunks ? R->sum[tid] : 0;
    if (S.cuts_sum()) {
        const BinCut b = bin_cut<NT>(R, S, &sp);
        const Line line((float)((double)mx - 2 * b.bin / W.scale), (float)((double)mx - 2 * (b.bin + 1) / W.scale));
        cut = cut_of<NT>(near_key, (int)held, line, false, S, W, b.need - b.above, &sp);
        static_assert(kMaxChunks <= 256, "sums in the histogram");
        for (int i = tid; i < 256; i += NT) sp.hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < (int)held; i += NT)
            if (order_of(keys[i], i) >= cut) atomicAdd(&sp.hist[place[i] / kChunk], W.units(logit_of(keys[i]), S.least));
        __syncthreads();
        if (tid < chunks) part += sp.hist[tid];
        if (cut && index_in(cut) < (int)held) cut = order_of(key_in(cut), place[index_in(cut)]);  // in the row's terms
    }
    const u64 upto = block_scan<NT>(part, sp.wsum, &total);
    u64 target = S.target_of(u, total);
    if (target >= upto - part && target < upto) sp.token = tid, sp.base = upto - part;
    __syncthreads();
    const int chunk = sp.token, i0 = chunk * kChunk;
    target -= sp.base;
    const int i = draw_of<NT>([&](int j) { return far_key(i0 + j); }, i0, min(kChunk, V - i0), cut, S, W, u, target,
                              &total, &sp);
    if (i >= 0) drawn(P, r, i0 + i, W.weight(x[i0 + i]), total);
}

}  // namespace

void launch_sample_rows(hipStream_t st, const SampleRowsParams &p) {
    if (p.vocab <= kRowVocab) {
        const unsigned lds = (unsigned)p.vocab * 4;
        constexpr int most = (1 << 22) - 1;  // a launch's threads are counted in 32 bits
        for (int row0 = 0; row0 < p.rows; row0 += most) {
            const dim3 grid((unsigned)std::min(most, p.rows - row0));
            if (p.vocab <= 1024) hipLaunchKernelGGL(k_sample_row<256>, grid, dim3(256), lds, st, p, row0);
            else hipLaunchKernelGGL(k_sample_row<1024>, grid, dim3(1024), lds, st, p, row0);
            if (p.rows - row0 <= most) break;
        }
        return;
    }
    RowScratch *scratch = static_cast<RowScratch *>(p.scratch);
    const int most = (int)std::min<size_t>(p.scratch_bytes / sizeof(RowScratch), 1024);
    const unsigned chunks = (unsigned)((p.vocab + kChunk - 1) / kChunk);
    for (int row0 = 0; row0 < p.rows; row0 += most) {
        const unsigned n = (unsigned)std::min(most, p.rows - row0);
        const dim3 grid(chunks, n);
        switch (group_of(p.vocab)) {
            case 4: hipLaunchKernelGGL(k_sample_max<4>, grid, dim3(256), 0, st, p, scratch, row0); break;
            case 16: hipLaunchKernelGGL(k_sample_max<16>, grid, dim3(256), 0, st, p, scratch, row0); break;
            default: hipLaunchKernelGGL(k_sample_max<64>, grid, dim3(256), 0, st, p, scratch, row0);
        }
        hipLaunchKernelGGL(k_sample_sum, grid, dim3(256), 0, st, p, scratch, row0);
        if (p.p.top_p || p.p.top_k) hipLaunchKernelGGL(k_sample_near, grid, dim3(256), 0, st, p, scratch, row0);
        hipLaunchKernelGGL(k_sample_draw, dim3(n), dim3(kDrawThreads), 0, st, p, scratch, row0);
    }
}

}  // namespace qtts
