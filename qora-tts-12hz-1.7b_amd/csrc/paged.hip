// paged.hip — the paged 8-bit cache: rotated append, attention, reading back.
//
// A block is one page of one kv head: P tokens x HD values in int8 with one
// f32 scale, K as [P][HD], V as [HD][P] (the product with the probabilities
// contracts over tokens).  The page a sequence is filling lies in f32 in its
// slot's open rows, so every block is rounded once, when it is full.
#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "paged_plan.h"
#include "serve.h"

namespace qtts {

namespace {

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, 0xF, 0xF, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over groups of 8 or 16 lanes, the same in each.
template <int WIDTH>
__device__ __forceinline__ double group_sum(double v) {
    v += dpp64<kDppXor1>(v);
    v += dpp64<kDppXor2>(v);
    v += dpp64<kDppHalfMirror>(v);
    if (WIDTH == 16) v += dpp64<kDppMirror>(v);
    return v;
}

// 1 / sqrt(x): the hardware's estimate and two steps of Newton's method.
__device__ __forceinline__ double inv_sqrt(double x) {
    if (!(x > 0.0 && x < (double)INFINITY)) return 1.0 / sqrt(x);
    double y = __builtin_amdgcn_rsq(x);
    y *= 1.5 - 0.5 * x * y * y;
    y *= 1.5 - 0.5 * x * y * y;
    return y;
}

// One head's vector spread over HD / 8 lanes: lane g of them holds elements
// 4g..4g+3 of both halves, the pairs that the rotation mixes.
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 load4(const float *p) { return *glb(reinterpret_cast<const f32x4 *>(p)); }
__device__ __forceinline__ void store4(float *p, f32x4 v) { *glb(reinterpret_cast<f32x4 *>(p)) = v; }

struct Pairs {
    f32x4 lo, hi;
    __device__ __forceinline__ void load(const float *p, int g, int half) {
        lo = load4(p + 4 * g);
        hi = load4(p + half + 4 * g);
    }
    __device__ __forceinline__ void store(float *p, int g, int half) const {
        store4(p + 4 * g, lo);
        store4(p + half + 4 * g, hi);
    }
};

// A position's cosines and sines, lane g's four.
struct Turn {
    f32x4 c, s;
    __device__ __forceinline__ void load(const qtts_paged_rows &r, int pos, int g, int half) {
        c = load4(r.rope_cos + (size_t)pos * half + 4 * g);
        s = load4(r.rope_sin + (size_t)pos * half + 4 * g);
    }
};

// Norm and rotation in 64 bits, rounded to f32 once: codes at the border
// between two steps then agree with the definition's.  The vector units run
// 64-bit products at the f32 rate, and the kernel waits for memory.
template <int HD>
__device__ __forceinline__ Pairs norm_rotate(const Pairs &x, const Turn &t, const uint16_t *norm, float eps, bool rope,
                                             int g) {
    double a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) a[i] = x.lo[i], b[i] = x.hi[i];
    if (norm) {
        double ss = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) ss += a[i] * a[i] + b[i] * b[i];
        const double inv = inv_sqrt(group_sum<HD / 8>(ss) * (1.0 / HD) + (double)eps);
        const uint2 na = *reinterpret_cast<const uint2 *>(norm + 4 * g);
        const uint2 nb = *reinterpret_cast<const uint2 *>(norm + HD / 2 + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            a[i] *= (double)f16_to_f32((uint16_t)((i < 2 ? na.x : na.y) >> 16 * (i & 1))) * inv;
            b[i] *= (double)f16_to_f32((uint16_t)((i < 2 ? nb.x : nb.y) >> 16 * (i & 1))) * inv;
        }
    }
    Pairs r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double y = rope ? a[i] * (double)t.c[i] - b[i] * (double)t.s[i] : a[i];
        const double z = rope ? b[i] * (double)t.c[i] + a[i] * (double)t.s[i] : b[i];
        r.lo[i] = (float)y, r.hi[i] = (float)z;
    }
    return r;
}

// max |x| as bits; an Inf or NaN is the largest.
__device__ __forceinline__ unsigned top_bits(f32x4 x, unsigned m) {
#pragma unroll
    for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}

// A block's scale and what its codes are made with: rne(127 x / top).  The
// f32 quotient is good to 2^-22 of its value; next to a border between two
// codes, and where 127 / top leaves f32's range, the quotient is a 64-bit one.
struct Quantizer {
    float top, inv;
    bool none;  // zeros, or not finite
    __device__ __forceinline__ explicit Quantizer(unsigned bits) {
        top = __uint_as_float(bits);
        none = bits == 0 || bits >= 0x7f800000u;
        inv = 127.0f / top;
    }
    __device__ __forceinline__ float scale() const {
        return __float_as_uint(top) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : top / 127.0f;
    }
    __device__ __forceinline__ int code(float x) const {
        if (none) return 0;
        const float t = x * inv, r = rintf(t);
        if (fabsf(t - r) < 0.4999f && top > 1e-30f) return (int)r;
        return (int)rint((double)x * 127.0 / (double)top);
    }
    __device__ __forceinline__ unsigned code4(float a, float b, float c, float d) const {
        return (unsigned)(code(a) & 255) | (unsigned)(code(b) & 255) << 8 | (unsigned)(code(c) & 255) << 16 |
               (unsigned)code(d) << 24;
    }
};

// A block for each (sequence, kv head, page that its rows touch, K or V), and for
// NT / (HD / 8) groups of four query heads.  Bound by memory: rows are read once,
// in 16-byte pieces all asked for before the first is used; a full page's codes
// are written from registers, V's across (by way of LDS) in whole lines.  4
// prompts of 2000 rows, 16 + 8 + 8 heads of 128: 46 us for 213 MB (4.6 TB/s, a
// copy's 5.1), 7 of them the norm's; 64 single rows 7 us, one 3.4, all latency.
template <int HD, int P>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppendParams A) {
    constexpr int L = HD / 8, H = HD / 2;                 // lanes of one head's vector, its half
    constexpr int NT = P * L < 256 ? P * L : 256;         // threads
    constexpr int V = NT / L, PASS = P / V;               // K: vectors a pass
    constexpr int D4 = HD / 4, TG = NT / D4;              // V: 4 dimensions of 4 tokens a thread
    constexpr int VPASS = P / 4 > TG ? P / 4 / TG : 1;
    constexpr int W = P / 4 + 1;                          // words of a dimension's row in LDS
    __shared__ unsigned tops[NT / 64];
    __shared__ unsigned vt[HD * W];
    const qtts_paged_kv &kv = A.kv;
    const int kv_blocks = 2 * A.kv_items * kv.kv_heads, per_seq = kv_blocks + A.q_items;
    const int b = blockIdx.x / per_seq, item = blockIdx.x % per_seq;
    const PagedSeq q = load_seq(A.s, b, kv.num_slots, A.cap);
    if (!q.ok || q.rows == 0) return;
    const int tid = threadIdx.x, g = tid % L, v = tid / L;
    const bool rope = A.r.rope_cos != nullptr;
    if (item >= kv_blocks) {  // queries: four heads of a row in each group of lanes
        const int groups = (A.r.heads + 3) / 4;
        const int at = (item - kv_blocks) * V + v;
        if (at >= q.rows * groups) return;
        const int row = at / groups, h0 = at % groups * 4, n = min(4, A.r.heads - h0);
        const float *from = A.r.q + (size_t)(q.row0 + row) * A.r.ld_q + (size_t)h0 * HD;
        float *to = A.r.q_out + (size_t)(q.row0 + row) * A.r.ld_q_out + (size_t)h0 * HD;
        Pairs x[4];
        Turn t;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i].load(from + min(i, n - 1) * HD, g, H);
        if (rope) t.load(A.r, q.start + row, g, H);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < n) norm_rotate<HD>(x[i], t, A.r.q_norm, A.r.eps, rope, g).store(to + i * HD, g, H);
        return;
    }
    const bool is_v = item & 1;
    const int head = item / 2 % kv.kv_heads, j = item / 2 / kv.kv_heads;
    const int end = q.start + q.rows, page = q.start / P + j;
    if (page * P >= end) return;
    float *open = (is_v ? kv.v_open : kv.k_open) + ((size_t)q.slot * kv.kv_heads + head) * P * HD;
    const float *rows = (is_v ? A.r.v : A.r.k) + (size_t)head * HD;
    const int ld = is_v ? A.r.ld_v : A.r.ld_k;
    auto row_at = [&](int pos) {  // what the cache holds or takes at a position
        return pos < q.start ? open + pos % P * HD : rows + (size_t)(q.row0 + pos - q.start) * ld;
    };
    auto open_rows = [&](int from, int to) {  // new rows of the page left open
        for (int pos = from + v; pos < to; pos += V) {
            Pairs x;
            Turn t;
            x.load(row_at(pos), g, H);
            if (!is_v) {
                if (rope) t.load(A.r, pos, g, H);
                x = norm_rotate<HD>(x, t, A.r.k_norm, A.r.eps, rope, g);
            }
            x.store(open + pos % P * HD, g, H);
        }
    };
    // The rows left open go over the open rows of the page that was begun
    // before: the block that reads those writes them, after reading.
    const bool begun = q.start % P != 0;
    if ((page + 1) * P > end) {
        if (j == 0 || !begun) open_rows(max(q.start, page * P), end);
        return;
    }
    const int id = q.pages[page];
    const bool in = id >= 0 && id < kv.num_pages;
    const size_t block = (size_t)(in ? id : 0) * kv.kv_heads + head;
    auto block_top = [&](unsigned top) {
        for (int off = 32; off > 0; off >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, off, 64));
        if (tid % 64 == 0) tops[tid / 64] = top;
        __syncthreads();
        for (int w = 0; w < NT / 64; w++) top = max(top, tops[w]);
        return top;
    };
    unsigned top = 0;
    if (!is_v) {
        Pairs x[PASS];
        Turn t[PASS];
#pragma unroll
        for (int i = 0; i < PASS; i++) {
            const int pos = page * P + i * V + v;
            x[i].load(row_at(pos), g, H);
            if (rope) t[i].load(A.r, pos, g, H);
        }
#pragma unroll
        for (int i = 0; i < PASS; i++) {
            if (page * P + i * V + v >= q.start) x[i] = norm_rotate<HD>(x[i], t[i], A.r.k_norm, A.r.eps, rope, g);
            top = top_bits(x[i].hi, top_bits(x[i].lo, top));
        }
        const Quantizer z(block_top(top));
        if (in) {
            if (tid == 0) kv.k_scales[block] = z.scale();
            unsigned *codes = reinterpret_cast<unsigned *>(kv.k_codes + block * P * HD);
#pragma unroll
            for (int i = 0; i < PASS; i++) {
                unsigned *to = codes + (i * V + v) * (HD / 4) + g;
                to[0] = z.code4(x[i].lo[0], x[i].lo[1], x[i].lo[2], x[i].lo[3]);
                to[HD / 8] = z.code4(x[i].hi[0], x[i].hi[1], x[i].hi[2], x[i].hi[3]);
            }
        }
    } else {
        f32x4 x[VPASS][4];
        const int d4 = tid % D4, tg = tid / D4;
        const bool part = P / 4 >= TG || tg < P / 4;
        if (part)
#pragma unroll
            for (int i = 0; i < VPASS; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[i][e] = load4(row_at(page * P + 4 * (i * TG + tg) + e) + 4 * d4);
        if (part)
#pragma unroll
            for (int i = 0; i < VPASS; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) top = top_bits(x[i][e], top);
        const Quantizer z(block_top(top));
        if (in) {
            if (tid == 0) kv.v_scales[block] = z.scale();
            if (part)
#pragma unroll
                for (int i = 0; i < VPASS; i++) {
                    unsigned *to = vt + 4 * d4 * W + i * TG + tg;
#pragma unroll
                    for (int e = 0; e < 4; e++) to[e * W] = z.code4(x[i][0][e], x[i][1][e], x[i][2][e], x[i][3][e]);
                }
            __syncthreads();
            uint4 *codes = reinterpret_cast<uint4 *>(kv.v_codes + block * P * HD);
#pragma unroll
            for (int i = tid; i < P * HD / 16; i += NT) {
                const unsigned *from = vt + i / (P / 16) * W + i % (P / 16) * 4;
                codes[i] = make_uint4(from[0], from[1], from[2], from[3]);
            }
        }
    }
    if (j == 0 && begun && end % P != 0) open_rows(end / P * P, end);
}

// ---------------------------------------------------------------------------
// Attention.  Scores are computed transposed, S^T = K Q^T, and so is the
// output, O^T = V^T P^T: the columns of every product are query rows (a row of
// the call and one of the heads that share the kv head, "columns" below), and
// the lane that holds a probability after the first product is the one that
// feeds it to the second, with no exchange between lanes.  The order of tokens
// in a contraction is free, so the pages are read 16 bytes a lane in an order
// that makes it so.
//
// Weights of V's products are p times the page's scale of V, whose logarithm
// joins the score (t = s + log2 scale): the largest weight fills the operand's
// range whatever V's size is, and t is rounded at its size (by some 2^-17 of a
// weight where scales are 2^100 or 2^-100, 2^-21 where they are ordinary).  The
// sum of probabilities has a reference of its own and is taken from the weights
// (over the scale) where they hold it.
// ---------------------------------------------------------------------------
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;

// Eight int8 codes as binary16: byte u = code + 128 becomes 1024 + u, whose
// mantissa it is, minus 1152.
__device__ __forceinline__ f16x8 codes_f16(unsigned w0, unsigned w1) {
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    union {
        f16x8 v;
        f16x2 h[4];
    } r;
    w0 ^= 0x80808080u, w1 ^= 0x80808080u;
    r.h[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) + off;
    r.h[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) + off;
    r.h[2] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) + off;
    r.h[3] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) + off;
    return r.v;
}

// Byte `digit` of four integers' balanced base-256 digits (-128 .. 127 but for
// the highest): adding 128 to the lower digits carries, and taking it off each
// is flipping its top bit.  `pick` selects the byte (digit | (digit + 4) << 8).
__device__ __forceinline__ int digits4(int a, int b, int c, int d, unsigned pick, unsigned flip) {
    const unsigned lo = __builtin_amdgcn_perm((unsigned)b + 0x808080u, (unsigned)a + 0x808080u, pick);
    const unsigned hi = __builtin_amdgcn_perm((unsigned)d + 0x808080u, (unsigned)c + 0x808080u, pick);
    return (int)((lo | hi << 16) ^ flip);
}

// Maximum and sum over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float rows4_max(float v) {
    v = halves_max(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float rows4_sum(float v) {
    v = halves_sum(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The other row of 16 lanes in a half of the wave.
__device__ __forceinline__ float dpp_row_pair(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return (threadIdx.x & 16) ? __uint_as_float(r[0]) : __uint_as_float(r[1]);
}

// Sum over the lanes l + 4 k of a row of 16, the same bits in each.
__device__ __forceinline__ float digits_sum(float v) {
    v += dpp<0x128>(v);  // row_ror:8
    return v + dpp<0x124>(v);
}

// A weight's integer, the nearest to it and to what the last one's rounding left,
// which it hands on: thousands of weights below half a unit, or all alike, beside a
// large one then sum up to what they are (30000 of 2^-28, 1e-4 of the sum: rounded
// each for itself, to units of 2^-27, all of them were lost).  Each is off by a unit
// at most, and not below 0, as a rest is -1/2 at least.
__device__ __forceinline__ int nearest(float x, float scale, float &rest) {
    const float y = fmaf(x, scale, rest), n = rintf(y);
    rest = y - n;
    return (int)n;
}

// log2 of the scale that a row or block of zeros takes: below all others, so that
// it leaves the reference to them.
constexpr float kZeroScale = -200.0f;
// An open row's values are taken times 2^60 below this and 2^-60 above that: their
// weights are 2^-120 of the probabilities beside values of 2^127, where the next
// ones would fall below f32.
constexpr float kSmallRow = -80.0f, kLargeRow = 80.0f;

// The same of an open row, by its largest value's exponent.
__device__ __forceinline__ float row_scale(float x) {
    return x == 0.0f ? kZeroScale : (float)((int)((__float_as_uint(x) >> 23) & 255) - 127);
}

// Columns of one kv head over one chunk of the tokens: a block of four waves,
// each every fourth step of 64 tokens (32 with 32 columns); chunks are joined by
// the block that ends last.  16 loads of 16 bytes a lane are in flight per step,
// K's for the next step from when this step's scores are done and V's from when
// its output is.
//
// Few columns are bound by reading the pages: 64 sequences of up to 8000 tokens,
// 8 kv heads of 128, 798 MB in 153 us (5.2 TB/s; a copy moves 5.1); 4 of 32760 in
// 47 us (4.7); 16 of 2064 in 21 us (2.6), of which 10 are a block's first loads
// and the joining, as one sequence of 1064 tokens takes 12 us.  Many are bound by
// vector instructions, codes to binary16 (160 of 440 a step) and the softmax: 1064
// rows of two heads behind 2000 tokens 76 us, 0.29 PFLOP/s (0.58 as hi + lo), of
// which vector instructions take 35 and products 18, with two waves a SIMD to
// cover one by the other.
//
// Of a step's 64 tokens, lane (r = lane % 16, G = lane / 16) has scores of
// tokens 16G + 4t + i in register i of tile t, and feeds them to the output's
// contraction as its slots of group G, which V's rows hold in that order.  K's
// tile t therefore holds token 16 (r / 4) + 4t + r % 4 in row r.
//
// I8: up to 4 columns, on int8 products: the codes go in as they are read.  A
// query value (scaled to the column's largest) and a weight are 30-bit
// integers, whose four base-256 digits take four operand columns: lane r holds
// digit r / 4 of column r % 4.  Integer sums are exact; they join the f32 ones
// when the running maximum rises.  Vector instructions a step: about half of the
// f16 form's, which a chunk of one token's attention is bound by otherwise.
//
// Otherwise 16 or 32 columns on binary16 products: codes are exact in it, a query
// value and a weight are split hi + lo: 22 bits, and no fewer than binary16's least
// step leaves, 2^-38 of a column's largest query value and 2^-35 of its largest
// weight.
//
// Three blocks of 64 dimensions fit a CU's registers (tiles of 32 columns, 8
// sequences of 500 rows, a window of 72: 33 us, 38 with two), two of 128.
//
// SINKS: with a window, the first tokens stay visible.  The tokens that a tile sees
// are then two stretches, the sinks' and the window's, each begun at a multiple of
// 64: they are numbered through, chunks and steps divide that numbering, and a
// step, which never lies in both, adds the hole between them to its tokens.
template <int HD, int MODE, bool SINKS>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void k_paged_attn(PagedAttnParams A) {
    constexpr bool I8 = MODE == kAttnI8;
    constexpr int S = MODE == kAttn32 ? 32 : 16;  // side of a product's tile
    constexpr int NG = 64 / S, NR = S * S / 64;   // lane groups, registers of a tile
    constexpr int CT = I8 ? 4 : S;                // columns
    constexpr int ST = 16 * NG, RT = 4 * ST;      // tokens of a wave's step, of the block's
    constexpr int NT = ST / S;                    // token tiles of a step
    constexpr int NK = HD / ST, ND = HD / S;      // 16-byte pieces of a K row in a lane; dimension tiles
    // Weights are 2^(t - m); the reference m is set so that the largest is
    // 2^kRoom, and again when one would pass 2^kLimit.  Integers take them times
    // 2^28, so that t - m is small, and its rounding too, where the weight is large
    // (binary16 would take a product each).
    constexpr int kRoom = I8 ? 0 : 11, kLimit = I8 ? 2 : 15, kUnits = I8 ? 28 : 0;
    constexpr int kFlush = 1024;                  // steps that int32 sums hold: 64 * 128 * 127 each
    typedef float Acc __attribute__((ext_vector_type(NR)));
    __shared__ float so[4][CT][HD + 4];
    __shared__ float sm[4][CT], sl[4][CT];
    __shared__ int sk[4][CT];
    __shared__ float srow[S == 32 ? 128 : 1];  // the open rows' largest |v|
    __shared__ unsigned sarrived;
    static_assert(4 * (HD + 4) >= kPagedMaxSplits, "the parts' factors take so's place");
    static_assert(kPagedPartFloats >= 3LL * kPagedRound / 2 * CT * part_floats(HD), "the parts fit");
    const int P = A.kv.page_size, sh = __builtin_ctz(P), kvh = A.kv.kv_heads, group = A.heads / kvh;
    // Consecutive blocks lie on different XCDs.  Tiles of 32 share their pages:
    // with kv heads innermost one head's are read through few caches, and the
    // last rows, which see the most, go first.  Few columns read every page
    // once, and faster with a pair's chunks spread (4 sequences of 32760: 48 us,
    // 54 with heads innermost).
    // Pairs past the plan's whole ones are divided over nsplit blocks.
    int id = blockIdx.x, head, b, split = 0, tile, shared = 0, nsplit = 1;
    if (id >= A.whole) {
        shared = (id - A.whole) / A.nsplit, split = (id - A.whole) % A.nsplit;
        id = A.whole + shared, nsplit = A.nsplit;
    }
    if (S == 32) {
        head = id % kvh, id /= kvh;
        b = id % A.s.batch, tile = A.tiles - 1 - id / A.s.batch;
    } else {
        tile = id % A.tiles, id /= A.tiles;
        head = id % kvh, b = id / kvh;
    }
    const int lane = threadIdx.x & 63, r = lane % S, G = lane / S;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the token (of a step's) in row r of K's tile 0: see above
    const int krow = S == 16 ? 16 * (r >> 2) + (r & 3) : 16 * (r >> 2 & 1) + 8 * (r >> 4) + 4 * (r >> 3 & 1) + (r & 3);
    auto group_max = [&](float v) { return NG == 4 ? rows4_max(v) : halves_max(v); };
    auto group_add = [&](float v) { return NG == 4 ? rows4_sum(v) : halves_sum(v); };
    // row of a product's tile that register i of this lane holds
    auto row_of = [&](int i) { return S == 16 ? 4 * G + i : 8 * (i / 4) + 4 * G + i % 4; };
    auto mma = [&](f16x8 x, f16x8 y, Acc c) {
        if constexpr (S == 16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
    };
    auto mma1 = [&](float x, float y, Acc c) {
        if constexpr (S == 16) return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x2f32(x, y, c, 0, 0, 0);
    };
    const PagedSeq q = load_seq(A.s, b, A.kv.num_slots, A.cap);
    const int left = (int)min((long long)q.rows * group - (long long)tile * CT, (long long)CT);
    if (left <= 0) return;
    auto out_of = [&](int n) {  // column n's place in the output
        const int c = tile * CT + n;
        return A.out + (size_t)(q.row0 + c / group) * A.ld_out + (size_t)(head * group + c % group) * HD;
    };
    if (!q.ok) {
        if (split == 0)
            for (int i = threadIdx.x; i < left * HD; i += 256) out_of(i / HD)[i % HD] = 0.0f;
        return;
    }
    // What the columns see, tokens low .. high - 1, in equal chunks of whole
    // steps: by this sequence's own length, not by its page table's.
    const int row_a = tile * CT / group, row_b = (tile * CT + left - 1) / group;
    const int high = q.start + row_b + 1;
    int low = A.window > 0 ? max(0, q.start + row_a - A.window + 1) : 0, from = low & ~63;
    // Numbers from `edge` on are `hole` below their tokens.  (Where there is a hole
    // the sinks lie in full pages: they end 64 tokens before the window begins.)
    const SeenHole gap = SINKS ? seen_hole(low, high, A.sinks) : SeenHole{0, 0};
    const int hole = gap.hole, edge = gap.edge;
    if (SINKS) from = 0, low = hole ? low : 0;
    const int chunk = chunk_of(high - hole - from, nsplit, attn_least(CT));
    const int parts = (high - hole - from + chunk - 1) / chunk;
    if (split >= parts) return;
    const int c0 = from + split * chunk;
    const int end = q.start + q.rows, full = end >> sh << sh;
    auto token_of = [&](int number) { return SINKS ? number + (number >= edge ? hole : 0) : number; };
    auto in_window = [&](int token, int pos) {
        return A.window == 0 || token > pos - A.window || (SINKS && token < A.sinks);
    };

    // this lane's column
    const int n = I8 ? r & 3 : r, digit = I8 ? r >> 2 : 0;
    const bool real = n < left;
    const int col = tile * CT + (real ? n : 0);
    const int pos = q.start + col / group;
    const float *qr = A.q + (size_t)(q.row0 + col / group) * A.ld_q + (size_t)(head * group + col % group) * HD;

    // --- full pages: the first step's loads ---
    const int stop = SINKS && hole ? min(c0 + chunk, max(edge, min(full, high) - hole)) : min(min(c0 + chunk, full), high);
    int base = c0 + ST * wave;
    u32x4 kr[NT][NK], vr[ND];
    // Loads come back in the order they are issued, so each is issued behind
    // what is needed before it, and none hangs on a branch (which would make a
    // wait for any of them a wait for all): past the last token, and for an
    // absent page, they read the pool's first page, whose tokens are masked.
    auto page_at = [&](int token) {
        const int pg = q.pages[token_of(min(token, stop - 1)) >> sh];
        return token < stop && pg >= 0 && pg < A.kv.num_pages ? pg : -1;
    };
    auto block_of = [&](int pg) { return (unsigned)(max(pg, 0) * kvh + head); };
    constexpr int kHdShift = HD == 64 ? 6 : 7;
    auto load_k = [&](int at, int pg) {
        const int8_t *p = A.kv.k_codes + ((size_t)block_of(pg) << (sh + kHdShift)) +
                          (((at + krow) & (P - 1)) << kHdShift) + 16 * G;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int h = 0; h < NK; h++)
                kr[t][h] = *glb(reinterpret_cast<const u32x4 *>(p + 4 * t * HD + ST * h));
    };
    auto load_v = [&](int at, int pg) {
        const int8_t *p = A.kv.v_codes + ((size_t)block_of(pg) << (sh + kHdShift)) + (r << sh) + ((at + 16 * G) & (P - 1));
#pragma unroll
        for (int d = 0; d < ND; d++) vr[d] = *glb(reinterpret_cast<const u32x4 *>(p + ((S * d) << sh)));
    };
    const bool any = base < stop;
    int pk = -1, pv = -1, pkn = -1, pvn = -1;  // this step's pages and the next one's
    float ks_ = 0, vs_ = 0, ksn, vsn;
    if (any) {
        pk = page_at(base + krow), pv = page_at(base + 16 * G);
        pkn = page_at(base + RT + krow), pvn = page_at(base + RT + 16 * G);
    }
    float x[NK][16];
#pragma unroll
    for (int h = 0; h < NK; h++)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 a = *reinterpret_cast<const float4 *>(qr + ST * h + 16 * G + j);
            x[h][j] = a.x, x[h][j + 1] = a.y, x[h][j + 2] = a.z, x[h][j + 3] = a.w;
        }
    auto load_first = [&]() {
        if (any) {
            load_k(token_of(base), pk);
            ks_ = A.kv.k_scales[block_of(pv)], vs_ = A.kv.v_scales[block_of(pv)];
            load_v(token_of(base), pv);
        }
    };
    if (S == 16) load_first();

    // --- the queries ---
    i32x4 qi[NK];                  // I8: digits of dimensions ST h + 16 G + 0 .. 15
    f16x8 qh[2 * NK], ql[2 * NK];  // else: hi and lo of ST h + 16 G + 8 u + 0 .. 7 at 2 h + u
    float qscale, qsize, qrest;
    const unsigned pick = (unsigned)(digit | (digit + 4) << 8) | 0x0c0c0000u;
    const unsigned flip = digit == 3 ? 0u : 0x80808080u;
    {
        unsigned bits = 0;
#pragma unroll
        for (int h = 0; h < NK; h++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                if (!real) x[h][j] = 0.0f;
                bits = max(bits, __float_as_uint(x[h][j]) & 0x7fffffffu);
            }
        // an Inf or NaN anywhere makes the column NaN
        const bool odd = group_max(bits >= 0x7f800000u ? 1.0f : 0.0f) > 0.0f;
        const float top = group_max(__uint_as_float(min(bits, 0x7f7fffffu)));
        int e = (int)(__float_as_uint(top) >> 23) - 127;
        e = e < -126 ? -126 : e;
#pragma unroll
        for (int h = 0; h < NK; h++) {
            if (I8) {
                int v[16];
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = odd ? 0 : (int)rintf(ldexpf(x[h][j], 29 - e));
#pragma unroll
                for (int j = 0; j < 4; j++)
                    qi[h][j] = digits4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], pick, flip);
            } else {
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float y = odd ? 0.0f : ldexpf(x[h][j], 14 - e);
                    const _Float16 a = (_Float16)y;
                    qh[2 * h + j / 8][j % 8] = a;
                    ql[2 * h + j / 8][j % 8] = (_Float16)(y - (float)a);
                }
            }
        }
        // What an operand is to be multiplied by, in two factors: in one, a query of
        // 2^-110 would leave it below f32's least normal value, and beside open keys of
        // 2^113 an operand of 2^15 would leave f32 (tiles of 32 take it times qsize).
        const int size = I8 ? e - 29 + 8 * digit : e - 14, h = max(size, -60);
        qsize = ldexpf(1.0f, h), qrest = ldexpf(1.0f, size - h);
        qscale = odd ? __uint_as_float(0x7fc00000u) : A.scale * kLog2e;
    }

    // Weights of V are 2^(t - m); the sum of probabilities l is held relative to
    // 2^(m - k), which stays within 2^60 of the largest: V's size, which is in t
    // and m, takes nothing from it.
    float m = -INFINITY, l = 0;
    int k = 0;
    constexpr float kFar = 60.0f;
    Acc o[ND] = {};
    i32x4 oi[I8 ? ND : 1] = {};
    int held = 0;  // steps in oi
    float rest[I8 ? 4 : 1] = {};  // of weights' integers, every fourth token's

    auto flush = [&]() {
        if constexpr (I8) {
            if (held) {
#pragma unroll
                for (int d = 0; d < ND; d++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) o[d][i] += (float)oi[d][i];
                    oi[d] = i32x4{0, 0, 0, 0};
                }
                held = 0;
            }
        }
    };
    // l's reference up to a probability of 2^rel of it, where that is far.
    auto lift = [&](float rel) {
        const int by = rel > kFar ? (int)rintf(rel) : 0;
        k -= by;
        l = ldexpf(l, -by);
    };
    // A new reference where a column's largest t asks for it, and what was
    // summed under the last one; `prob`: the largest probability's logarithm, of
    // top's.  Scores may lie farther apart than an int holds, and top - kRoom is top
    // where f32's steps are larger: what becomes a whole number is a difference.
    auto raise = [&](float top, float prob) {
        const bool first = m == -INFINITY, need = top > (first ? -INFINITY : m + kLimit);
        if (__any(need)) {
            const float mn = need ? top - kRoom : m;
            const float down = first ? 0.0f : fmaxf(m - mn, -4096.0f);  // 2^-4096 is nothing
            const float c = first ? 0.0f : __builtin_amdgcn_exp2f(down);
            const float most = prob + (top - mn);  // of this reference
            const float at = most == most ? fminf(fmaxf(most, -1024.0f), 1024.0f) : 0.0f;
            flush();
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= c;
            const int by = (int)rintf(down);
            l *= __builtin_amdgcn_exp2f(down - (float)by);
#pragma unroll
            for (int e = 0; e < (I8 ? 4 : 0); e++) rest[e] *= c;
            k = first && need ? -(int)rintf(at) : k - by;
            m = mn;
            if (need) lift(at + (float)k);
        }
    };

    // --- the open page's rows, in f32 products, S tokens a step and a wave ---
    // Tiles of 16 read them to registers (while the first step's pages are on
    // their way); with tiles of 32, which have none to spare, the block brings
    // K's and then V's to LDS, in the place of its result.
    const int open_lo = max(max(full, low), c0 + hole), open_hi = min(min(end, c0 + chunk + hole), high);
    const float *k_open = A.kv.k_open + ((size_t)q.slot * kvh + head) * P * HD;
    const float *v_open = A.kv.v_open + ((size_t)q.slot * kvh + head) * P * HD;
    float(*rows)[HD + 4] = so[0];  // S == 32: row t - open_lo of the open page, 128 at most
    // V's are staged as the products take them: what is not finite as 0, small rows
    // times 2^60, large ones 2^-60, their largest values in srow; returns whether something is
    // not finite.
    auto stage = [&](const float *from, bool values) {
        const int count = (open_hi - open_lo) * (HD / 4);
        bool bad = false;
        for (int i0 = threadIdx.x; i0 < count; i0 += 1024) {  // four loads in flight
            f32x4 y[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = min(i0 + 256 * j, count - 1), t = open_lo + i / (HD / 4);
                y[j] = *glb(reinterpret_cast<const f32x4 *>(from + (t & (P - 1)) * HD + 4 * (i % (HD / 4))));
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = min(i0 + 256 * j, count - 1);
                if (values) {
                    float top = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool finite = fabsf(y[j][e]) < INFINITY;
                        bad |= !finite;
                        y[j][e] = finite ? y[j][e] : 0.0f;
                        top = fmaxf(top, fabsf(y[j][e]));
                    }
                    top = row16_max(top);
                    if (HD == 128) top = fmaxf(top, dpp_row_pair(top));
                    y[j] *= row_scale(top) < kSmallRow ? 0x1p60f : row_scale(top) > kLargeRow ? 0x1p-60f : 1.0f;
                    if (i0 + 256 * j < count) srow[i / (HD / 4)] = top;
                }
                if (i0 + 256 * j < count) *reinterpret_cast<f32x4 *>(&rows[i / (HD / 4)][4 * (i % (HD / 4))]) = y[j];
            }
        }
        return bad;
    };
    auto open_tile = [&](int t0) {
        const bool mine = t0 < open_hi;  // S == 32: others only take part in the staging
        Acc s = {}, s1 = {};
        float v[S == 16 ? NR : 1][ND];
        bool odd = false;
        if (S == 16) {
            const int kt = t0 + r;  // K: row r of the tile
            const float *kp = k_open + ((kt < open_hi ? kt : open_lo) & (P - 1)) * HD + 4 * G;
            // V: dimension S d + r of the token of register i
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const int token = t0 + row_of(i);
                const bool in = token < open_hi;
                const float *vp = v_open + ((in ? token : open_lo) & (P - 1)) * HD + r;
#pragma unroll
                for (int d = 0; d < ND; d++) v[S == 16 ? i : 0][d] = vp[S * d];
#pragma unroll
                for (int d = 0; d < ND; d++) v[S == 16 ? i : 0][d] = in ? v[S == 16 ? i : 0][d] : 0.0f;
            }
#pragma unroll
            for (int c = 0; c < HD / (4 * NG); c++) {
                const float4 y = *reinterpret_cast<const float4 *>(kp + 4 * NG * c);
                float4 z = *reinterpret_cast<const float4 *>(qr + 4 * NG * c + 4 * G);
                if (!real || digit) z = make_float4(0, 0, 0, 0);
                s = mma1(y.x, z.x, s);
                s1 = mma1(y.y, z.y, s1);
                s = mma1(y.z, z.z, s);
                s1 = mma1(y.w, z.w, s1);
            }
            s += s1;
        } else {
            stage(k_open, false);
            __syncthreads();
            if (mine) {
                const float *kp = rows[min(t0 + r, open_hi - 1) - open_lo] + 16 * G;
#pragma unroll
                for (int h = 0; h < NK; h++)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const f32x4 y = *reinterpret_cast<const f32x4 *>(kp + ST * h + j);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int at = 2 * h + (j + i) / 8;
                            s = mma1(y[i], ((float)qh[at][(j + i) % 8] + (float)ql[at][(j + i) % 8]) * qsize, s);
                        }
                    }
            }
            __syncthreads();
            odd = stage(v_open, true);
            __syncthreads();
        }
        // What is not finite is left out of V's products (0 * Inf would reach
        // rows that do not see it) and added by itself below.
        float p[NR];
        if (mine) {
            float mx = -INFINITY, prob = -INFINITY;
            unsigned zeros = 0, smalls = 0, larges = 0;  // of the rows here
            float tops[S == 16 ? NR : 1];
            // (qscale is NaN where the query is not finite: -Inf is no score)
            const float by = S == 16 ? qscale : qscale * qrest;
            auto size_of = [&](int i) {  // the logarithm of a row's V
                return row_scale(S == 32 ? srow[min(t0 + row_of(i), open_hi - 1) - open_lo] : tops[S == 16 ? i : 0]);
            };
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const int token = t0 + row_of(i);
                if (S == 16) {
                    float top = 0;
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const float y = fabsf(v[S == 16 ? i : 0][d]);
                        odd |= !(y < INFINITY);
                        top = fmaxf(top, y < INFINITY ? y : 0.0f);
                    }
                    tops[S == 16 ? i : 0] = row16_max(top);
                }
                const bool seen = token <= pos && token < open_hi && in_window(token, pos);
                // (the other digits' products are of zeros: none, or NaN with an Inf)
                p[i] = seen ? (I8 ? digits_sum(digit ? 0.0f : s[i]) : s[i]) * by : -INFINITY;
                const float big = size_of(i);
                zeros |= (unsigned)(big == kZeroScale) << i;
                smalls |= (unsigned)(big < kSmallRow) << i, larges |= (unsigned)(big > kLargeRow) << i;
                mx = fmaxf(mx, p[i] + big - 7.0f);  // as a page's, whose codes go to 127
            }
            const float top = group_max(mx);
            // Where f32's steps are whole units, a score is rounded as the reference
            // is, with V's size, and p is taken from there on.
            const bool coarse = fabsf(top) >= 0x1p24f && fabsf(top) < INFINITY;
            if (__any(coarse)) {
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    const float big = size_of(i);
                    p[i] = coarse ? (p[i] + big - 7.0f - top) + (7.0f - big) : p[i];
                }
            }
#pragma unroll
            for (int i = 0; i < NR; i++) prob = fmaxf(prob, p[i]);
            prob = group_max(prob);
            raise(top, coarse ? prob : prob - top);
            const float ms = (m == -INFINITY ? 0.0f : m) - (coarse ? top : 0.0f);
            lift(prob - ms + (float)k);
#pragma unroll
            for (int i = 0; i < NR; i++) {
                l += __builtin_amdgcn_exp2f(p[i] - ms + (float)k);
                // 2^60 of a small row's weight goes over to its values, of a large one's
                // values to its weight, and zeros have none
                const float over = zeros >> i & 1    ? kZeroScale
                                   : smalls >> i & 1 ? -60.0f
                                   : larges >> i & 1 ? 60.0f
                                                     : 0.0f;
                p[i] = digit ? 0.0f : __builtin_amdgcn_exp2f(p[i] - ms + over) * (float)(1 << kUnits);
            }
            if (S == 32) {
#pragma unroll
                for (int i0 = 0; i0 < NR; i0 += 4) {  // four tokens' values ahead of their products
                    float y[4][ND];
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int d = 0; d < ND; d++)
                            y[j][d] = rows[min(t0 + row_of(i0 + j), open_hi - 1) - open_lo][S * d + r];
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int d = 0; d < ND; d++) o[d] = mma1(y[j][d], p[i0 + j], o[d]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NR; i++)
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const float y = v[S == 16 ? i : 0][d];
                        const float by = smalls >> i & 1 ? 0x1p60f : larges >> i & 1 ? 0x1p-60f : 1.0f;
                        o[d] = mma1(fabsf(y) < INFINITY ? y * by : 0.0f, p[i], o[d]);
                    }
            }
        }
        // (with tiles of 32 the block decides, as V's rows give way to the weights)
        if (S == 32 ? __syncthreads_or(odd) : __any(odd)) {
            if (mine) {
                float *weight = &so[wave][0][0];  // [S tokens][S columns]
#pragma unroll
                for (int i = 0; i < NR; i++) weight[row_of(i) * S + r] = p[i];
#pragma unroll 1
                for (int token = t0; token < min(t0 + S, open_hi); token++) {
                    const float w = fmaxf(weight[(token - t0) * S + r], 0x1p-126f);
                    const bool seen = token <= pos && in_window(token, pos) && !digit;
                    const float *vp = v_open + (token & (P - 1)) * HD;
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int i = 0; i < NR; i++) {
                            const float y = vp[S * d + row_of(i)];
                            if (seen && !(fabsf(y) < INFINITY)) o[d][i] += w * y;
                            if (i % 4 == 3) asm volatile("" ::: "memory");  // as above
                        }
                }
            }
        }
        if (S == 32) __syncthreads();
    };
    if (S == 16) {
        for (int t0 = open_lo + S * wave; t0 < open_hi; t0 += 4 * S) open_tile(t0);
    } else if (open_lo < open_hi) {
        open_tile(open_lo + S * wave);
    }

    // --- full pages ---
    if (S == 32) load_first();  // no registers to spare for them before
    auto step = [&](auto more) {  // more: another one follows, whose pages are asked for
        const int next = base + RT;
        float p[16];
        const bool there = pv >= 0;
        if constexpr (I8) {
            i32x4 s[4] = {};
#pragma unroll
            for (int h = 0; h < NK; h++)
#pragma unroll
                for (int t = 0; t < 4; t++)
                    s[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, kr[t][h]), qi[h], s[t], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 16; j++) p[j] = (float)s[j / 4][j % 4];
        } else {
            Acc s[NT] = {};
#pragma unroll
            for (int h = 0; h < NK; h++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const f16x8 c = codes_f16(kr[t][h][2 * u], kr[t][h][2 * u + 1]);
                        s[t] = mma(c, qh[2 * h + u], s[t]);
                        s[t] = mma(c, ql[2 * h + u], s[t]);
                    }
#pragma unroll
            for (int j = 0; j < 16; j++) p[j] = s[j / NR][j % NR];
        }
        int pk2 = -1, pv2 = -1;
        if constexpr (more) {
            pk2 = page_at(next + RT + krow), pv2 = page_at(next + RT + 16 * G);
            load_k(token_of(next), pkn);
            ksn = A.kv.k_scales[block_of(pvn)], vsn = A.kv.v_scales[block_of(pvn)];
        }
        const float kq = qscale * qsize * ks_ * qrest;
        // The page's scale of V joins the scores as its logarithm, and leaves
        // the sum of probabilities as its inverse.
        const bool small = vs_ < 0x1p-64f, zero = !there || vs_ == 0.0f;
        const float vc = small ? vs_ * 0x1p64f : vs_;
        const float lg = zero ? kZeroScale : __builtin_amdgcn_logf(vc) - (small ? 64.0f : 0.0f);
        const float ms = m == -INFINITY ? 0.0f : m;
        const float off = digit ? 0.0f : lg - ms;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            p[j] = fmaf(p[j], kq, off);
            if (I8) p[j] = digits_sum(p[j]);
        }
        // every column sees all of the step's tokens unless the step passes
        // the first column's position, the window's edge or an absent page
        const int at = token_of(base);
        const bool plain = at + ST - 1 <= q.start + row_a && base + ST <= stop && (SINKS || base >= low) &&
                           (A.window == 0 || at > high - 1 - A.window || (SINKS && at + ST <= A.sinks)) && __all(there);
        if (!plain) {
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int token = at + 16 * G + j;
                const bool seen = there && token <= pos && base + 16 * G + j < stop && in_window(token, pos);
                p[j] = seen ? p[j] : -INFINITY;
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; j++) mx = fmaxf(mx, p[j]);
        if (__any(mx > (m == -INFINITY ? -INFINITY : (float)kLimit))) {
            const float top = group_max(mx);
            raise(top + ms, group_max(mx - lg) - top);
            const float mr = m == -INFINITY ? 0.0f : m, by = ms - mr;
            const bool coarse = fmaxf(fabsf(ms), fabsf(mr)) >= 0x1p24f;
            if (__any(coarse)) {
                // Where f32's steps are whole units, p holds what a score's rounding
                // leaves: the score is rounded as the reference is, and stays below it.
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    p[j] = coarse ? (p[j] + ms) - mr : p[j] + by;
                    p[j] = p[j] > kLimit ? (float)kLimit : p[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; j++) p[j] += by;
            }
        }
        // weights of a V that is so much smaller than the others' hold no
        // probabilities: these are then taken by themselves
        const bool apart = __any(there && (vs_ == 0.0f || (float)k - lg >= kFar));
        if (apart) {
            float prob = -INFINITY;
#pragma unroll
            for (int j = 0; j < 16; j++) prob = fmaxf(prob, p[j]);
            lift(group_max(prob - lg) + (float)k);
            // (a lane whose page is of scale NaN and masked has a NaN lg and no p)
#pragma unroll
            for (int j = 0; j < 16; j++) l += p[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(p[j] - lg + (float)k);
        }
        float sum = 0;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            p[j] = __builtin_amdgcn_exp2f(p[j]);
            sum += p[j];
        }
        // (the sum is 0 where a lane's page is absent or all is masked, as a NaN scale)
        if (!apart && sum != 0.0f) l = fmaf(sum, ldexpf(__builtin_amdgcn_rcpf(vc), small ? k + 64 : k), l);
        if constexpr (I8) {
            i32x4 w;
#pragma unroll
            for (int j = 0; j < 4; j++)
                w[j] = digits4(nearest(p[4 * j], 0x1p28f, rest[0]), nearest(p[4 * j + 1], 0x1p28f, rest[1]),
                               nearest(p[4 * j + 2], 0x1p28f, rest[2]), nearest(p[4 * j + 3], 0x1p28f, rest[3]), pick,
                               flip);
#pragma unroll
            for (int d = 0; d < ND; d++)
                oi[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, vr[d]), w, oi[d], 0, 0, 0);
            if (++held == kFlush) flush();
        } else {
            f16x8 ph[2], pl[2];
#pragma unroll
            for (int j = 0; j < 16; j += 2) {  // lo holds the rest; both to the nearest
                const f16x2 a = __builtin_convertvector(f32x2{p[j], p[j + 1]}, f16x2);
                const f16x2 c = __builtin_convertvector(f32x2{p[j] - (float)a[0], p[j + 1] - (float)a[1]}, f16x2);
                ph[j / 8][j % 8] = a[0], ph[j / 8][j % 8 + 1] = a[1];
                pl[j / 8][j % 8] = c[0], pl[j / 8][j % 8 + 1] = c[1];
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const f16x8 v = codes_f16(vr[d][2 * u], vr[d][2 * u + 1]);
                    o[d] = mma(v, ph[u], o[d]);
                    o[d] = mma(v, pl[u], o[d]);
                }
        }
        if constexpr (more) {
            load_v(token_of(next), pvn);
            pv = pvn, pkn = pk2, pvn = pv2;
            ks_ = ksn, vs_ = vsn;
        }
    };
    if (any) {
        for (; base + RT < stop; base += RT) step(std::true_type{});
        step(std::false_type{});
    }

    // --- the block's four waves ---
    flush();
    l = group_add(l);
    const bool writes = !I8 || digit == 0;
    if (G == 0 && writes) sm[wave][n] = m, sl[wave][n] = l, sk[wave][n] = k;
    const float weight = ldexpf(1.0f, 8 * digit - kUnits);
#pragma unroll
    for (int d = 0; d < ND; d++) {
        Acc z = o[d];
        if (I8)
#pragma unroll
            for (int i = 0; i < NR; i++) z[i] = digits_sum(z[i] * weight);
        if (writes)
#pragma unroll
            for (int i = 0; i < NR; i += 4)
                *reinterpret_cast<f32x4 *>(&so[wave][n][S * d + row_of(i)]) = f32x4{z[i], z[i + 1], z[i + 2], z[i + 3]};
    }
    __syncthreads();
    // Joining, of waves and of parts: outputs relative to the largest reference,
    // sums to the one whose power of two is nearest to the largest of theirs.
    constexpr int PW = part_floats(HD);
    float *part = A.part + (size_t)shared * nsplit * CT * PW;
    if ((int)threadIdx.x < left) {
        const int c = threadIdx.x;
        float mx = -INFINITY, far = -INFINITY, sum = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) mx = fmaxf(mx, sm[w][c]);
        const float ms = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int w = 0; w < 4; w++) far = fmaxf(far, sm[w][c] - ms - (float)sk[w][c]);
        const int kj = far == -INFINITY ? 0 : -(int)rintf(far);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float d = sm[w][c] - ms;
            sum += sl[w][c] == 0.0f ? 0.0f : sl[w][c] * __builtin_amdgcn_exp2f(d == -INFINITY ? 0.0f : d + (float)(kj - sk[w][c]));
            sm[w][c] = __builtin_amdgcn_exp2f(d);
        }
        if (parts == 1) {
            sl[0][c] = sum, sk[0][c] = kj;
        } else {
            float *to = part + ((size_t)split * CT + c) * PW + HD;
            st_dev(to, mx), st_dev(to + 1, sum), st_dev(to + 2, (float)kj);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < left * (HD / 4); i += 256) {
        const int c = i / (HD / 4), d = 4 * (i % (HD / 4));
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) acc += sm[w][c] * *reinterpret_cast<const f32x4 *>(&so[w][c][d]);
        if (parts == 1) {
            const float sum = sl[0][c];
            acc = sum == 0.0f ? f32x4{0, 0, 0, 0} : acc / sum;
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = ldexpf(acc[j], sk[0][c]);
            *reinterpret_cast<f32x4 *>(out_of(c) + d) = acc;
        } else {
            float *to = part + ((size_t)split * CT + c) * PW + d;
#pragma unroll
            for (int j = 0; j < 4; j += 2)
                st_dev_u64(reinterpret_cast<uint64_t *>(to + j),
                           __float_as_uint(acc[j]) | (uint64_t)__float_as_uint(acc[j + 1]) << 32);
        }
    }
    if (parts == 1) return;
    wait_stores();
    __syncthreads();
    if (threadIdx.x == 0) {
        sarrived = arrive_dev(A.counters + shared);
        if (sarrived == (unsigned)parts - 1) reset_dev(A.counters + shared);
    }
    __syncthreads();
    if (sarrived != (unsigned)parts - 1) return;
    // The parts' rows, two values a load and 16 loads in flight; the first ones
    // while the maxima and sums become every part's factor.
    constexpr int MI = CT * HD > 512 ? CT * HD / 512 : 1, U = MI > 8 ? 1 : 16 / MI;
    float *fac = &so[0][0][0];
    uint64_t y[U][MI];
    const int pairs = left * (HD / 2);  // of values
    auto load_parts = [&](int k0) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < MI; i++) {
                const int at = min((int)threadIdx.x + 256 * i, pairs - 1), k = min(k0 + u, parts - 1);
                const float *from = part + ((size_t)k * CT + at / (HD / 2)) * PW + 2 * (at % (HD / 2));
                y[u][i] = ld_dev_u64(reinterpret_cast<const uint64_t *>(from));
            }
    };
    load_parts(0);
    for (int c = wave; c < left; c += 4) {
        constexpr int N = kPagedMaxSplits / 64;
        float pm[N], ps[N], pk[N], mx = -INFINITY, far = -INFINITY, sum = 0;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float *from = part + ((size_t)min(lane + 64 * j, parts - 1) * CT + c) * PW + HD;
            const uint64_t z = ld_dev_u64(reinterpret_cast<const uint64_t *>(from));
            pk[j] = ld_dev(from + 2);
            pm[j] = lane + 64 * j < parts ? __uint_as_float((unsigned)z) : -INFINITY;
            ps[j] = lane + 64 * j < parts ? __uint_as_float((unsigned)(z >> 32)) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < N; j++) mx = fmaxf(mx, pm[j]);
        mx = wave_max(mx);
        const float ms = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int j = 0; j < N; j++) far = fmaxf(far, pm[j] - ms - pk[j]);
        far = wave_max(far);
        const float kj = far == -INFINITY ? 0.0f : -rintf(far);
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float d = pm[j] - ms;
            if (lane + 64 * j < parts) fac[c * parts + lane + 64 * j] = __builtin_amdgcn_exp2f(d);
            sum += ps[j] == 0.0f ? 0.0f : ps[j] * __builtin_amdgcn_exp2f(d == -INFINITY ? 0.0f : d + (kj - pk[j]));
        }
        sum = wave_sum(sum);
        if (lane == 0) sl[0][c] = sum, sk[0][c] = (int)kj;
    }
    __syncthreads();
    float acc[MI][2] = {};
    for (int k0 = 0; k0 < parts; k0 += U) {
        if (k0) load_parts(k0);
#pragma unroll
        for (int i = 0; i < MI; i++) {
            const int c = min((int)threadIdx.x + 256 * i, pairs - 1) / (HD / 2);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float f = k0 + u < parts ? fac[c * parts + k0 + u] : 0.0f;
                acc[i][0] = fmaf(f, __uint_as_float((unsigned)y[u][i]), acc[i][0]);
                acc[i][1] = fmaf(f, __uint_as_float((unsigned)(y[u][i] >> 32)), acc[i][1]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MI; i++) {
        const int at = threadIdx.x + 256 * i, c = at / (HD / 2);
        if (at >= pairs) break;
        const float sum = sl[0][c];
        *reinterpret_cast<float2 *>(out_of(c) + 2 * (at % (HD / 2))) =
            sum == 0.0f ? make_float2(0, 0)
                        : make_float2(ldexpf(acc[i][0] / sum, sk[0][c]), ldexpf(acc[i][1] / sum, sk[0][c]));
    }
}

// A block of each (sequence, kv head, page that its positions touch): 4 tokens x
// 4 dimensions a thread, so that V's codes, which lie across, are turned in
// registers and every row is written 16 bytes a lane in a row.  Bound by writing:
// 8000 tokens of 8 heads of 128, 82 MB in 16 us (5.1 TB/s).
template <int HD>
__global__ __launch_bounds__(256) void k_paged_read(PagedReadParams A, int items) {
    constexpr int D4 = HD / 4;
    const int P = A.kv.page_size, sh = __builtin_ctz(P), kvh = A.kv.kv_heads;
    const int head = blockIdx.x % kvh, item = blockIdx.x / kvh % items, b = blockIdx.x / kvh / items;
    const PagedSeq q = load_seq(A.s, b, A.kv.num_slots, A.cap);
    const int len = A.lens ? A.lens[b] : q.start + q.rows;
    const bool ok = q.ok && len <= A.cap;
    // positions of this block, by pages where they have any
    const int first = ok ? q.start >> sh << sh : 0;
    const int lo = max(first + item * P, ok ? q.start : 0);
    const int hi = min(first + (item + 1) * P, ok ? q.start + q.rows : q.rows);
    if (lo >= hi) return;
    const int row0 = q.row0 - (ok ? q.start : 0);  // of position 0
    const int full = ok ? len >> sh << sh : 0;
    const int page = lo >> sh;
    const int id = ok && lo < full ? q.pages[page] : -1;
    const bool closed = id >= 0 && id < A.kv.num_pages;
    const size_t block = (size_t)(closed ? id : 0) * kvh + head;
    const float ks = closed ? A.kv.k_scales[block] : 0.0f, vs = closed ? A.kv.v_scales[block] : 0.0f;
    const float *k_open = A.kv.k_open + ((size_t)(ok ? q.slot : 0) * kvh + head) * P * HD;
    const float *v_open = A.kv.v_open + ((size_t)(ok ? q.slot : 0) * kvh + head) * P * HD;
    const int8_t *kc = A.kv.k_codes + block * P * HD, *vc = A.kv.v_codes + block * P * HD;
    const int t_lo = lo & ~3, parts = ((hi - t_lo + 3) >> 2) * D4;
    auto byte = [](unsigned w, int i) { return (float)(int8_t)(w >> 8 * i); };
    for (int i = threadIdx.x; i < parts; i += 256) {
        const int d = 4 * (i % D4), t0 = t_lo + 4 * (i / D4);  // 4 tokens from t0, in one page
        unsigned kw[4], vw[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            kw[e] = *reinterpret_cast<const unsigned *>(kc + (((t0 + e) & (P - 1)) * HD) + d);
            vw[e] = *reinterpret_cast<const unsigned *>(vc + ((d + e) << sh) + (t0 & (P - 1)));
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int t = t0 + e;
            if (t < lo || t >= hi) continue;
            f32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
            if (closed) {
                k = f32x4{byte(kw[e], 0), byte(kw[e], 1), byte(kw[e], 2), byte(kw[e], 3)} * ks;
                v = f32x4{byte(vw[0], e), byte(vw[1], e), byte(vw[2], e), byte(vw[3], e)} * vs;
            } else if (ok && t >= full && t < len) {
                k = load4(k_open + (t & (P - 1)) * HD + d);
                v = load4(v_open + (t & (P - 1)) * HD + d);
            }
            if (A.k_out) store4(A.k_out + (size_t)(row0 + t) * A.ld_k + head * HD + d, k);
            if (A.v_out) store4(A.v_out + (size_t)(row0 + t) * A.ld_v + head * HD + d, v);
        }
    }
}

template <int HD>
void append_of(hipStream_t st, const PagedAppendParams &p, unsigned blocks) {
    auto go = [&](auto page) {
        constexpr int P = decltype(page)::value;
        constexpr int NT = P * HD / 8 < 256 ? P * HD / 8 : 256;
        hipLaunchKernelGGL((k_paged_append<HD, P>), dim3(blocks), dim3(NT), 0, st, p);
    };
    switch (p.kv.page_size) {
        case 16: return go(std::integral_constant<int, 16>{});
        case 32: return go(std::integral_constant<int, 32>{});
        case 64: return go(std::integral_constant<int, 64>{});
        default: return go(std::integral_constant<int, 128>{});
    }
}

template <int HD, bool SINKS>
void attn_of(hipStream_t st, const PagedAttnParams &p, AttnMode mode, unsigned blocks) {
    if (mode == kAttnI8) hipLaunchKernelGGL((k_paged_attn<HD, kAttnI8, SINKS>), dim3(blocks), dim3(256), 0, st, p);
    else if (mode == kAttn16) hipLaunchKernelGGL((k_paged_attn<HD, kAttn16, SINKS>), dim3(blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_paged_attn<HD, kAttn32, SINKS>), dim3(blocks), dim3(256), 0, st, p);
}

template <bool SINKS>
void attn_dims(hipStream_t st, const PagedAttnParams &p, AttnMode mode, unsigned blocks) {
    if (p.kv.head_dim == 64) attn_of<64, SINKS>(st, p, mode, blocks);
    else attn_of<128, SINKS>(st, p, mode, blocks);
}

}  // namespace

void launch_paged_append(hipStream_t st, const PagedAppendParams &in) {
    PagedAppendParams p = in;
    const AppendPlan plan = append_plan(p.kv, p.s, p.r);
    p.kv_items = plan.kv_items;
    p.q_items = (int)plan.q_items;
    if (p.kv.head_dim == 64) append_of<64>(st, p, (unsigned)plan.blocks);
    else append_of<128>(st, p, (unsigned)plan.blocks);
}

void launch_paged_attention(hipStream_t st, const PagedAttnParams &in) {
    PagedAttnParams p = in;
    const bool sinks = p.sinks > 0 && p.window > 0;
    const AttnShape shape = attn_shape(p.kv, p.s, p.heads, sinks ? seen_span(p.window, p.sinks) : 0);
    p.tiles = shape.tiles;
    p.whole = shape.whole;
    p.nsplit = shape.nsplit;
    if (sinks) attn_dims<true>(st, p, shape.mode, (unsigned)shape.blocks);
    else attn_dims<false>(st, p, shape.mode, (unsigned)shape.blocks);
}

void launch_paged_read(hipStream_t st, const PagedReadParams &p) {
    const int items = read_items(p.kv, p.s);
    const unsigned blocks = (unsigned)read_blocks(p.kv, p.s);
    if (p.kv.head_dim == 64) hipLaunchKernelGGL(k_paged_read<64>, dim3(blocks), dim3(256), 0, st, p, items);
    else hipLaunchKernelGGL(k_paged_read<128>, dim3(blocks), dim3(256), 0, st, p, items);
}

}  // namespace qtts
