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
    unsigned near[kBrute];
    unsigned digit, thr, ties, top, bad;
    int token;
};

// The prefix of n <= kBrute keys, near(i) in the order of their indices, of which
// the first `count` stay (0: all) and then, where `by_sum`, those whose
// predecessors' sum and `above` is below `need` (0: top-p's share of the sum).
// NT / kBrute threads a key, or one, compare it with the others.
template <int NT, class Key>
__device__ Cut rank_all(const Key &near, int n, u64 count, bool by_sum, u64 above, u64 need, const RowSettings &S,
                        const Weights &W, Space *sp) {
    constexpr int PARTS = NT / kBrute;
    static_assert(PARTS == 1 || PARTS == 4, "quads of lanes");
    u64 *units = sp->hist;
    const int i = threadIdx.x / PARTS, part = threadIdx.x % PARTS;
    __syncthreads();
    if (threadIdx.x == 0) sp->thr = 0xffffffffu, sp->ties = 0;
    const bool in = i < n;
    const unsigned k = in ? near(i) : 0;
    const u64 mine = in && by_sum ? W.units(logit_of(k)) : 0;
    if (in && part == 0) units[i] = mine;
    __syncthreads();
    unsigned rank = 0;
    u64 ahead = 0;
    if (in) {
#pragma unroll 4
        for (int j = part; j < n; j += PARTS) {
            const unsigned o = near(j);
            const bool before = o > k || (o == k && j < i);
            rank += before;
            ahead += before ? units[j] : 0;
        }
    }
    for (int off = 1; off < PARTS; off <<= 1) {
        rank += __shfl_xor((int)rank, off, 64);
        ahead += (u64)__shfl_xor((long long)ahead, off, 64);
    }
    bool keep = in && (count == 0 || rank < count);
    if (by_sum) {
        if (need == 0) need = S.share_of(block_total<NT>(keep && part == 0 ? mine : 0, sp->wsum));
        keep = keep && above + ahead < need;
    }
    if (keep) atomicMin(&sp->thr, k);
    __syncthreads();
    Cut c;
    c.thr = sp->thr;
    if (keep && part == 0 && k == c.thr) atomicAdd(&sp->ties, 1u);
    __syncthreads();
    c.ties = sp->ties;
    return c;
}

// The prefix that top-k and top-p keep of n keys, key(i) in the order of their
// indices; `need`: the sum that top-p's prefix reaches, 0: its share of the sum.
// Small sets at once.  Others by the logit's place on a line of 2^16 steps from
// the largest down, 8 bits at a time, counts first and then sums, until what
// shares the cut's step is a small set (many equal ones: by the key's digits).
template <int NT, class Key>
__device__ Cut cut_of(const Key &key, int n, const RowSettings &S, const Weights &W, u64 need, Space *sp) {
    const int tid = threadIdx.x;
    const bool sums = S.cuts_sum();
    Cut c;
    if (S.top_k == 0 && !sums) return c;
    if (n <= kBrute) return rank_all<NT>(key, n, S.top_k, sums, 0, need, S, W, sp);
    // the least finite logit, and the line's scale
    unsigned least = 0xffffffffu;
    for (int i = tid; i < n; i += NT) {
        const unsigned k = key(i);
        least = min(least, k > key_of(-INFINITY) ? k : 0xffffffffu);
    }
    for (int off = 32; off > 0; off >>= 1) least = min(least, (unsigned)__shfl_xor((int)least, off, 64));
    __syncthreads();
    if (tid == 0) sp->thr = 0xffffffffu;
    __syncthreads();
    if ((tid & 63) == 0) atomicMin(&sp->thr, least);
    __syncthreads();
    const float lo = logit_of(sp->thr);
    __syncthreads();
    float scale = 0;
    auto line = [&](unsigned k) {  // halves, so that the difference stays in range
        const float l = logit_of(k);
        return l == W.mx ? 0 : (int)fminf((0.5f * W.mx - 0.5f * l) * scale, 65535.0f);
    };
    auto scan_digits = [&](bool down, u64 want, u64 base) {  // by the first wave: where the sum reaches `want`
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
    };
    auto select = [&](bool by_sum, u64 want) {
        const float range = 0.5f * W.mx - 0.5f * lo;
        const float far = by_sum ? 16.0f * S.t : INFINITY;  // half of 46 octaves: no weights past them
        const float span = range < far ? range : far;
        scale = span > 0.0f ? 65535.0f / span : 0.0f;
        if (!(scale < INFINITY)) scale = 3e38f;
        u64 base = 0;
        int at = 0;  // the chosen steps' first digits
        for (int round = 0; round < 2; round++) {
            for (int i = tid; i < 256; i += NT) sp->hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += NT) {
                const unsigned k = key(i);
                if (k < c.thr) continue;
                const int p = line(k);
                if (round == 1 && p >> 8 != at) continue;
                const u64 w = by_sum ? W.units(logit_of(k)) : (u64)1;
                if (w) atomicAdd(&sp->hist[round == 0 ? p >> 8 : p & 255], w);
            }
            __syncthreads();
            scan_digits(false, want, base);
            at = at << 8 | (int)sp->digit;
            base = sp->base;
            // what shares them, in order, if that is few
            const int shift = round == 0 ? 8 : 0;
            const int per = (n + NT - 1) / NT, lo_i = min(tid * per, n), hi_i = min(lo_i + per, n);
            u64 have = 0, all;
            for (int i = lo_i; i < hi_i; i++) {
                const unsigned k = key(i);
                have += k >= c.thr && line(k) >> shift == at;
            }
            int to = (int)(block_scan<NT>(have, sp->wsum, &all) - have);
            if (all <= kBrute) {
                for (int i = lo_i; i < hi_i; i++) {
                    const unsigned k = key(i);
                    if (k >= c.thr && line(k) >> shift == at) sp->near[to++] = k;
                }
                auto near = [&](int i) { return sp->near[i]; };
                return by_sum ? rank_all<NT>(near, (int)all, 0, true, base, want, S, W, sp)
                              : rank_all<NT>(near, (int)all, want - base, false, 0, 0, S, W, sp);
            }
        }
        unsigned prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            for (int i = tid; i < 256; i += NT) sp->hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += NT) {
                const unsigned k = key(i);
                if (k < c.thr || line(k) != at || (shift < 24 && k >> (shift + 8) != prefix)) continue;
                const u64 w = by_sum ? W.units(logit_of(k)) : (u64)1;
                if (w) atomicAdd(&sp->hist[(k >> shift) & 255], w);
            }
            __syncthreads();
            scan_digits(true, want, base);
            prefix = prefix << 8 | sp->digit;
            base = sp->base;
        }
        __syncthreads();
        const u64 w = by_sum ? W.units(logit_of(prefix)) : (u64)1;
        Cut d;
        d.thr = prefix;
        d.ties = w ? (want - base + w - 1) / w : ~0ull;
        return d;
    };
    if (S.top_k > 0) c = select(false, (u64)S.top_k);
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
        __syncthreads();
        const Cut d = select(true, need);
        if (d.thr > c.thr) c = d;
        else c.ties = d.ties < c.ties ? d.ties : c.ties;
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
        const u64 w = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)mine, j) |
                      (u64)(unsigned)__builtin_amdgcn_readlane((int)(mine >> 32), j) << 32;
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

// The first of 256 bins in `hist` (in LDS) where the sum from bin 0 reaches
// `want`: by the first wave, for all after the barrier.
__device__ __forceinline__ void first_bin(u64 want, Space *sp) {
    if (threadIdx.x < 64) {
        u64 h[4], sum = 0;
        for (int j = 0; j < 4; j++) sum += h[j] = sp->hist[4 * threadIdx.x + j];
        u64 run = wave_scan(sum) - sum;
        const bool mine = run < want && run + sum >= want, none = !__any(mine);
        if (mine || (none && threadIdx.x == 63)) {
            int j = 0;
            for (; j < 3 && run + h[j] < want; j++) run += h[j];
            sp->digit = 4 * threadIdx.x + j;
        }
    }
    __syncthreads();
}

// A logit's place among 256 equal steps from the largest, down to `lo` (halves,
// so that the difference stays in range).
struct Line {
    float mx, scale;
    __device__ __forceinline__ Line(float top, float lo) : mx(top) {
        const float range = 0.5f * top - 0.5f * lo;
        scale = range > 0.0f ? 255.0f / range : 0.0f;
        if (!(scale < INFINITY)) scale = 3e38f;
    }
    __device__ __forceinline__ int operator()(unsigned k) const {
        const float l = logit_of(k);
        return l == mx ? 0 : (int)fminf((0.5f * mx - 0.5f * l) * scale, 255.0f);
    }
};

// Four logits of a row from the i-th, -Inf past the last: 16 bytes a lane where
// the row's start allows it.
__device__ __forceinline__ f32x4 load_logits(const float *x, int i, int V, bool aligned) {
    if (aligned && i + 4 <= V) return *glb(reinterpret_cast<const f32x4 *>(x + i));
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = i + e < V ? x[min(i + e, V - 1)] : -INFINITY;
    return v;
}

constexpr int kRowVocab = 8192;  // with the lists, a block's 64 KB of LDS

template <int NT>
__global__ __launch_bounds__(NT) void k_sample_row(SampleRowsParams P) {
    constexpr int kList = 2048;  // candidates
    extern __shared__ unsigned keys[];
    __shared__ Space sp;
    __shared__ unsigned list[kList], sleast;
    __shared__ unsigned short place[kList];
    const int r = blockIdx.x, tid = threadIdx.x, V = P.vocab;
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
    const unsigned *set = keys;
    int n = V;
    u64 need = 0;
    bool listed = false;
    if (S.top_k > 0 || S.cuts_sum()) {
        // Candidates, in the order of their indices: by steps down from the
        // largest, up to the one where top-k's count or top-p's sum is reached.
        const bool by_sum = S.top_k == 0;
        const float lo = logit_of(sleast), far = mx - 32.0f * S.t;  // 46 octaves: no weights past them
        const Line line(mx, by_sum && far > lo ? far : lo);
        u64 sum = 0;
        for (int i = tid; i < V; i += NT) {
            const unsigned k = keys[i];
            const u64 w = by_sum ? W.units(logit_of(k)) : (u64)1;
            if (w) atomicAdd(&sp.hist[line(k)], w);
            sum += w;
        }
        if (by_sum) need = S.share_of(block_total<NT>(sum, sp.wsum));
        __syncthreads();
        first_bin(by_sum ? need : (u64)S.top_k, &sp);
        const int bin = (int)sp.digit;
        const int per = (V + NT - 1) / NT, lo_i = min(tid * per, V), hi_i = min(lo_i + per, V);
        u64 count = 0, total;
        for (int i = lo_i; i < hi_i; i++) count += line(keys[i]) <= bin;
        int at = (int)(block_scan<NT>(count, sp.wsum, &total) - count);
        if (total <= kList) {
            for (int i = lo_i; i < hi_i; i++)
                if (line(keys[i]) <= bin) list[at] = keys[i], place[at++] = (unsigned short)i;
            set = list, n = (int)total, listed = true;
            __syncthreads();
            if (n <= 64) {
                if (tid < 64)
                    finish_wave(P, r, tid < n ? list[tid] : 0, n, [&](int i) { return (int)place[i]; }, S, W, need);
                return;
            }
        }
    }
    auto key = [&](int j) { return set[j]; };
    const Cut c = cut_of<NT>(key, n, S, W, need, &sp);
    u64 total;
    const int i = draw_of<NT>(key, n, c, S, W, P.u[r], 0, ~0ull, &total, &sp);
    if (i >= 0) drawn(P, r, listed ? place[i] : i, W.weight(logit_of(set[i])), total);
}

// ---------------------------------------------------------------------------
// Rows of more than kRowVocab logits
// ---------------------------------------------------------------------------
constexpr int kChunk = 4096, kGroup = 64;         // logits of a block, of a maximum
constexpr int kNear = 8192;                       // tokens next to a cut that are held
constexpr int kMaxChunks = kSampleRowsMaxVocab / kChunk, kMaxGroups = kSampleRowsMaxVocab / kGroup;

// A row's scratch.
struct RowScratch {
    u64 hist[kBins];                  // top-p without top-k: units by bin
    u64 sum[kMaxChunks];              // kept units of a chunk (of bins before the cut's)
    unsigned top[kMaxChunks];         // its largest key
    int token[kMaxChunks];            // where that is first
    unsigned bad[kMaxChunks];         // a NaN
    unsigned low[kMaxChunks];         // the least of its groups' maxima above -Inf
    unsigned near_at[kMaxChunks];     // its candidates (of top-p: in the cut's bin), in `near`
    unsigned near_n[kMaxChunks];
    unsigned near_all;
    float least;                      // top-k's candidates are no smaller; +Inf: a NaN in the row
    unsigned near[kNear];             // keys
    int near_i[kNear];                // and indices
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

__global__ __launch_bounds__(256) void k_sample_max(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ unsigned stop, sbad, slow;
    __shared__ int stoken;
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const bool aligned = ((uintptr_t)x & 15) == 0;
    if (tid == 0) stop = 0, sbad = 0, slow = 0xffffffffu, stoken = V;
    for (int i = chunk * 256 + tid; i < kBins; i += gridDim.x * 256) R->hist[i] = 0;
    if (chunk == 0 && tid == 0) R->near_all = 0;
    __syncthreads();
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = load_logits(x, chunk * kChunk + 1024 * j + 4 * tid, V, aligned);
    unsigned top = 0, low = 0xffffffffu;
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
        low = min(low, g > key_of(-INFINITY) ? g : 0xffffffffu);
        const int at = chunk * kChunk + 1024 * j + 4 * tid;
        if ((tid & 15) == 0 && at < V) R->group[at / kGroup] = g;
    }
    top = wave_top(top), low = ~wave_top(~low);
    if ((tid & 63) == 0) atomicMax(&stop, top), atomicMin(&slow, low);
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
    if (tid == 0) R->top[chunk] = top, R->bad[chunk] = sbad, R->low[chunk] = slow, R->token[chunk] = stoken;
}

// What top-k's candidates are no smaller than: a value that top_k of the groups'
// maxima reach, by 256 steps down from the largest; every finite logit where
// there are not that many groups.  (-Inf is never drawn, so it is no candidate.)
__device__ void find_least(RowScratch *R, const RowSettings &S, int chunks, int groups, Space *sp) {
    constexpr int N = 16;  // loads in flight: a row of 262144 in one step, kept for both passes
    const int tid = threadIdx.x;
    unsigned g[N];
#pragma unroll
    for (int j = 0; j < N; j++) g[j] = R->group[min(tid + j * 256, groups - 1)];
    if (tid == 0) sp->thr = 0xffffffffu, sp->ties = 0xffffffffu;
    sp->hist[tid] = 0;
    const RowTop t = row_top(R, chunks, sp);
    float least = t.bad ? INFINITY : -3.402823466e38f;
    if (S.top_k < groups && !t.bad) {
        if (tid < chunks) atomicMin(&sp->thr, R->low[tid]);
        __syncthreads();
        const Line line(logit_of(t.top), logit_of(sp->thr));
        auto each = [&](auto take) {
#pragma unroll
            for (int j = 0; j < N; j++)
                if (tid + j * 256 < groups) take(g[j]);
            for (int i = tid + N * 256; i < groups; i += 256) take(R->group[i]);
        };
        each([&](unsigned k) { atomicAdd(&sp->hist[line(k)], (u64)1); });
        __syncthreads();
        first_bin((u64)S.top_k, sp);
        const int bin = (int)sp->digit;
        unsigned low = 0xffffffffu;
        each([&](unsigned k) { low = min(low, line(k) <= bin ? k : 0xffffffffu); });
        low = ~wave_top(~low);
        if ((tid & 63) == 0) atomicMin(&sp->ties, low);
        __syncthreads();
        least = fmaxf(least, logit_of(sp->ties));
    }
    if (tid == 0) R->least = least;
}

// Rows that top-k cuts: where its candidates end.  Others: units by bin where
// top-p cuts them, else the chunk's sum.
__global__ __launch_bounds__(256) void k_sample_sum(SampleRowsParams P, RowScratch *scratch, int row0) {
    __shared__ Space sp;
    __shared__ u64 hist[kBins];
    const int r = row0 + blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    RowScratch *R = scratch + blockIdx.y;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S(P, r);
    if (S.greedy || (S.top_k > 0 && chunk > 0)) return;
    if (S.top_k > 0) return find_least(R, S, gridDim.x, (V + kGroup - 1) / kGroup, &sp);
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
    if (i0 < V && (!first || R->group[i0 / kGroup] >= key_of(least))) {
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
constexpr int kDrawThreads = 1024;

__global__ __launch_bounds__(kDrawThreads) void k_sample_draw(SampleRowsParams P, RowScratch *scratch, int row0) {
    constexpr int NT = kDrawThreads;
    __shared__ Space sp;
    __shared__ unsigned keys[kNear];
    __shared__ int place[kNear];
    __shared__ int offset[kMaxChunks], ties[kMaxChunks];
    const int r = row0 + blockIdx.x, tid = threadIdx.x, V = P.vocab, chunks = (V + kChunk - 1) / kChunk;
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
    // Candidates into LDS, in the order of their indices.
    const unsigned mine = tid < chunks ? R->near_n[tid] : 0;
    unsigned first = 0;
    u64 held = 0;
    if (S.top_k > 0 || S.cuts_sum()) {
        first = (unsigned)(block_scan<NT>(mine, sp.wsum, &held) - mine);
        if (held > kNear) return whole();  // many equal logits, or top_k past a few thousand
        if (tid < chunks) offset[tid] = (int)first - (int)R->near_at[tid];
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
        const Cut c = cut_of<NT>(near_key, n, S, W, 0, &sp);
        const int i = draw_of<NT>(near_key, n, c, S, W, u, 0, ~0ull, &total, &sp);
        if (i >= 0) drawn(P, r, place[i], W.weight(logit_of(keys[i])), total);
        return;
    }
    Cut c;
    u64 part = tid < chunks ? R->sum[tid] : 0;
    if (S.cuts_sum()) {
        const BinCut b = bin_cut<NT>(R, S, &sp);
        c = cut_of<NT>(near_key, (int)held, S, W, b.need - b.above, &sp);
        // each chunk's ties before it and kept sum
        static_assert(kMaxChunks <= 256, "sums in the histogram");
        for (int i = tid; i < 256; i += NT) sp.hist[i] = 0;
        if (tid < chunks) ties[tid] = 0;
        const int per = ((int)held + NT - 1) / NT, lo = min(tid * per, (int)held), hi = min(lo + per, (int)held);
        u64 count = 0, all;
        for (int i = lo; i < hi; i++) count += keys[i] == c.thr;
        u64 seen = block_scan<NT>(count, sp.wsum, &all) - count;  // with the barrier
        for (int i = lo; i < hi; i++) {
            const unsigned k = keys[i];
            const int at = place[i] / kChunk;
            if (k == c.thr) atomicAdd(&ties[at], 1);
            if (k > c.thr || (k == c.thr && seen++ < c.ties)) atomicAdd(&sp.hist[at], W.units(logit_of(k), S.least));
        }
        __syncthreads();
        if (tid < chunks) part += sp.hist[tid], count = (u64)ties[tid];
        else count = 0;
        const u64 upto = block_scan<NT>(count, sp.wsum, &all);
        if (tid < chunks) ties[tid] = (int)(upto - count);
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
        if (p.vocab <= 1024) hipLaunchKernelGGL(k_sample_row<256>, dim3((unsigned)p.rows), dim3(256), lds, st, p);
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
        if (p.p.top_p || p.p.top_k) hipLaunchKernelGGL(k_sample_near, dim3(chunks, n), dim3(256), 0, st, p, scratch, row0);
        hipLaunchKernelGGL(k_sample_draw, dim3(n), dim3(kDrawThreads), 0, st, p, scratch, row0);
    }
}

}  // namespace qtts
