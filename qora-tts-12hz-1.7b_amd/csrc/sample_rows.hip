// sample_rows.hip — a token from each row of logits: temperature, top-k,
// top-p, min-p, given uniform numbers.
//
// Weights w_i = exp((l_i - max) / T) are evaluated in 64 bits and summed as
// integers of 2^-44 of the largest: sums do not depend on their order (one
// row's partial sums come from many waves through atomics), and a draw next to
// the border between two tokens falls as the 64-bit definition's does.
#include "device_common.h"
#include "serve.h"

namespace qtts {

namespace {

typedef unsigned long long u64;
constexpr int kT = 1024;
constexpr double kUnit = 17592186044416.0;  // 2^44

// Order-preserving integer of a float (no NaN), both zeros alike.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ u64 shfl_up64(u64 v, int off) {
    return (u64)__shfl_up((long long)v, off, 64);
}

// Inclusive scan over the block; every thread gets the total as well.
__device__ u64 block_scan(u64 v, u64 *wsum, u64 *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int off = 1; off < 64; off <<= 1) {
        const u64 y = shfl_up64(v, off);
        if (lane >= off) v += y;
    }
    __syncthreads();
    if (lane == 63) wsum[wave] = v;
    __syncthreads();
    u64 base = 0, all = 0;
    for (int w = 0; w < kT / 64; w++) {
        if (w < wave) base += wsum[w];
        all += wsum[w];
    }
    *total = all;
    return base + v;
}

struct RowSettings {
    float t, top_p, min_p;
    int top_k;
};

__device__ __forceinline__ RowSettings settings_of(const SampleRowsParams &P, int r) {
    RowSettings s;
    s.t = P.p.temperature ? P.p.temperature[r] : 1.0f;
    s.top_k = P.p.top_k ? P.p.top_k[r] : 0;
    s.top_p = P.p.top_p ? P.p.top_p[r] : 1.0f;
    s.min_p = P.p.min_p ? P.p.min_p[r] : 0.0f;
    return s;
}

__device__ __forceinline__ double weight_of(float l, float mx, double t) {
    return l == mx ? 1.0 : l == -INFINITY || mx == INFINITY ? 0.0 : exp(((double)l - (double)mx) / t);
}

__device__ __forceinline__ u64 units_of(double w) { return (u64)rint(w * kUnit); }

// One block per row; the row is read from memory at each pass.
__global__ __launch_bounds__(kT) void k_sample_rows(SampleRowsParams P) {
    __shared__ u64 wsum[kT / 64], hist[256];
    __shared__ unsigned smax, sthr, snan;
    __shared__ u64 sbase;
    __shared__ int stoken;
    const int r = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    const float *x = P.logits + (size_t)r * P.ld;
    const RowSettings S = settings_of(P, r);
    if (tid == 0) smax = 0, snan = 0, stoken = V;
    __syncthreads();
    unsigned top = 0, bad = 0;
    for (int i = tid; i < V; i += kT) {
        const float l = x[i];
        bad |= l != l;
        top = max(top, key_of(l));
    }
    if (bad) atomicOr(&snan, 1u);
    atomicMax(&smax, top);
    __syncthreads();
    top = smax;
    const float mx = __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
    if (snan || mx == -INFINITY) {
        if (tid == 0) {
            P.tokens[r] = -1;
            if (P.probs) P.probs[r] = snan ? __uint_as_float(0x7fc00000u) : 0.0f;
        }
        return;
    }
    if (!(S.t > 0.0f)) {
        for (int i = tid; i < V; i += kT)
            if (key_of(x[i]) == top) {
                atomicMin(&stoken, i);
                break;
            }
        __syncthreads();
        if (tid == 0) {
            P.tokens[r] = stoken;
            if (P.probs) P.probs[r] = 1.0f;
        }
        return;
    }
    const double T = S.t;
    // The kept ones are those above `thr` and the first `ties` at it.
    unsigned thr = 0;
    u64 ties = (u64)V;
    // Finds the largest key whose count (or sum) with all above reaches
    // `need` (count: >= need; sum: >= need), by 8 bits at a time; `above`:
    // what lies above it.
    auto select = [&](bool by_sum, u64 need, u64 *above) {
        unsigned prefix = 0;
        u64 base = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i0 = 0; i0 < V; i0 += kT) {
                const int i = i0 + tid;
                const float l = i < V ? x[i] : -INFINITY;
                const unsigned k = key_of(l);
                bool in = i < V && k >= thr;
                if (in && shift < 24) in = (k >> (shift + 8)) == prefix;
                if (in) {
                    if (by_sum) atomicAdd(&hist[(k >> shift) & 255], units_of(weight_of(l, mx, T)));
                    else atomicAdd(&hist[(k >> shift) & 255], (u64)1);
                }
            }
            __syncthreads();
            if (tid == 0) {
                u64 run = base;
                int d = 255;
                for (; d > 0; d--) {
                    if (run + hist[d] >= need) break;
                    run += hist[d];
                }
                sthr = (unsigned)d;
                sbase = run;
            }
            __syncthreads();
            prefix = prefix << 8 | sthr;
            base = sbase;
        }
        *above = base;
        return prefix;
    };
    if (S.top_k > 0 && S.top_k < V) {
        u64 above;
        thr = select(false, (u64)S.top_k, &above);
        ties = (u64)S.top_k - above;
    }
    // The sum over the first k: those above thr and `ties` of its own weight.
    if (S.top_p < 1.0f) {
        u64 sum = 0, total;
        const float lt = __uint_as_float(thr & 0x80000000u ? thr & 0x7fffffffu : ~thr);
        const u64 wt = units_of(weight_of(lt, mx, T));
        for (int i = tid; i < V; i += kT)
            if (key_of(x[i]) > thr) sum += units_of(weight_of(x[i], mx, T));
        block_scan(sum, wsum, &total);
        if (thr) total += ties * wt;
        // kept: predecessors' sum < top_p * total, so sums up to (and with)
        // the last kept one reach that; the key where that happens:
        const double want = (double)(S.top_p > 0.0f ? S.top_p : 0.0f) * (double)total;
        u64 need = (u64)ceil(want);
        if (need < 1) need = 1;
        u64 above;
        const unsigned t2 = select(true, need, &above);
        if (t2 > thr || thr == 0) {
            const float l2 = __uint_as_float(t2 & 0x80000000u ? t2 & 0x7fffffffu : ~t2);
            const u64 w2 = units_of(weight_of(l2, mx, T));
            thr = t2;
            ties = w2 ? (need - above + w2 - 1) / w2 : (u64)V;
        } else {
            const u64 n = wt ? (need - above + wt - 1) / wt : ties;
            ties = n < ties ? n : ties;
        }
    }
    const double least = S.min_p > 0.0f ? (S.min_p < 1.0f ? (double)S.min_p : 1.0) : 0.0;
    // The kept sum, then the token: a pass in index order.  Rows whose first
    // `ties` at thr are kept count those in index order as they go.
    u64 target = 0, kept_sum = 0;
    for (int pass = 0; pass < 2; pass++) {
        u64 run = 0, tied = 0;
        for (int i0 = 0; i0 < V; i0 += kT) {
            const int i = i0 + tid;
            const float l = i < V ? x[i] : -INFINITY;
            const unsigned k = key_of(l);
            u64 all, w = 0;
            const bool at = i < V && k == thr;
            const u64 order = tied + block_scan(at ? 1 : 0, wsum, &all);
            tied += all;
            if (i < V && (k > thr || (at && order <= ties))) {
                const double e = weight_of(l, mx, T);
                if (e >= least) w = units_of(e);
            }
            const u64 upto = run + block_scan(w, wsum, &all);
            if (pass == 1 && w && upto > target && upto - w <= target) {
                P.tokens[r] = i;
                if (P.probs) P.probs[r] = (float)(weight_of(l, mx, T) * kUnit / (double)kept_sum);
            }
            run += all;
        }
        if (pass == 0) {
            kept_sum = run;
            const float u = P.u[r];
            const double want = (u > 0.0f ? (u < 1.0f ? (double)u : 1.0) : 0.0) * (double)run;
            target = (u64)want;
            if (target >= run) target = run - 1;
        }
    }
}

}  // namespace

void launch_sample_rows(hipStream_t st, const SampleRowsParams &p) {
    hipLaunchKernelGGL(k_sample_rows, dim3((unsigned)p.rows), dim3(kT), 0, st, p);
}

}  // namespace qtts
