// paged.hip — the paged 8-bit cache: rotated append, attention, reading back.
//
// A block is one page of one kv head: P tokens x HD values in int8 with one
// f32 scale, K as [P][HD], V as [HD][P] (the product with the probabilities
// contracts over tokens).  The page a sequence is filling lies in f32 in its
// slot's open rows, so every block is rounded once, when it is full.
#include "device_common.h"
#include "paged_plan.h"
#include "serve.h"

namespace qtts {

namespace {

__device__ __forceinline__ double group_sum(double v, int width) {
    for (int off = width / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, width);
    return v;
}

// One head's vector spread over HD / 8 lanes: lane g of them holds elements
// 4g..4g+3 of both halves, the pairs that the rotation mixes.
template <int HD>
struct Pairs {
    float lo[4], hi[4];
    __device__ __forceinline__ void load(const float *p, int g) {
        const float4 a = *reinterpret_cast<const float4 *>(p + 4 * g);
        const float4 b = *reinterpret_cast<const float4 *>(p + HD / 2 + 4 * g);
        lo[0] = a.x, lo[1] = a.y, lo[2] = a.z, lo[3] = a.w;
        hi[0] = b.x, hi[1] = b.y, hi[2] = b.z, hi[3] = b.w;
    }
    __device__ __forceinline__ void store(float *p, int g) const {
        *reinterpret_cast<float4 *>(p + 4 * g) = make_float4(lo[0], lo[1], lo[2], lo[3]);
        *reinterpret_cast<float4 *>(p + HD / 2 + 4 * g) = make_float4(hi[0], hi[1], hi[2], hi[3]);
    }
    __device__ __forceinline__ void zero() {
        for (int i = 0; i < 4; i++) lo[i] = hi[i] = 0.0f;
    }
    // Norm and rotation in 64 bits, rounded to f32 once: codes at the border
    // between two steps then agree with the definition's.  The vector units
    // run 64-bit products at the f32 rate, and the kernel waits for memory.
    __device__ __forceinline__ void norm_rotate(const qtts_paged_rows &r, const uint16_t *norm, int pos, int g) {
        double a[4], b[4];
        for (int i = 0; i < 4; i++) a[i] = lo[i], b[i] = hi[i];
        if (norm) {
            double ss = 0;
            for (int i = 0; i < 4; i++) ss += a[i] * a[i] + b[i] * b[i];
            ss = group_sum(ss, HD / 8);
            const double inv = 1.0 / sqrt(ss / HD + (double)r.eps);
            for (int i = 0; i < 4; i++) {
                a[i] *= (double)f16_to_f32(norm[4 * g + i]) * inv;
                b[i] *= (double)f16_to_f32(norm[HD / 2 + 4 * g + i]) * inv;
            }
        }
        if (r.rope_cos) {
            const float *cs = r.rope_cos + (size_t)pos * (HD / 2) + 4 * g;
            const float *sn = r.rope_sin + (size_t)pos * (HD / 2) + 4 * g;
            for (int i = 0; i < 4; i++) {
                const double c = cs[i], s = sn[i];
                const double x = a[i] * c - b[i] * s, y = b[i] * c + a[i] * s;
                a[i] = x, b[i] = y;
            }
        }
        for (int i = 0; i < 4; i++) lo[i] = (float)a[i], hi[i] = (float)b[i];
    }
    // max |x|; an Inf or NaN gives NaN or Inf (the integer order of |x|).
    __device__ __forceinline__ unsigned top_bits() const {
        unsigned m = 0;
        for (int i = 0; i < 4; i++) {
            m = max(m, __float_as_uint(lo[i]) & 0x7fffffffu);
            m = max(m, __float_as_uint(hi[i]) & 0x7fffffffu);
        }
        return m;
    }
};

// rne(127 x / top), the quotient's border cases settled in 64 bits.
__device__ __forceinline__ int quantize(float x, float top, float inv) {
    const float t = x * inv;
    const float r = rintf(t);
    if (fabsf(t - r) < 0.4999f && top > 1e-30f) return (int)r;
    return (int)rint((double)x * 127.0 / (double)top);
}

template <int HD, int P>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppendParams A) {
    constexpr int L = HD / 8;                                  // lanes of one head's vector
    constexpr int NT = P * L < 256 ? P * L : 256;              // threads
    constexpr int V = NT / L;                                  // vectors a pass
    constexpr int PASS = P / V;
    __shared__ unsigned tops[2][NT / 64];
    const int per_seq = A.kv_items * A.kv.kv_heads + A.q_items;
    const int b = blockIdx.x / per_seq, item = blockIdx.x % per_seq;
    const PagedSeq q = load_seq(A.s, b, A.kv.num_slots, A.cap);
    if (!q.ok || q.rows == 0) return;
    const int g = threadIdx.x % L, v = threadIdx.x / L;
    if (item >= A.kv_items * A.kv.kv_heads) {  // queries
        const long long units = (long long)q.rows * A.r.heads;
        const long long u0 = (long long)(item - A.kv_items * A.kv.kv_heads) * 64;
        for (long long u = u0 + v; u < min(u0 + 64, units); u += V) {
            const int row = (int)(u / A.r.heads), h = (int)(u % A.r.heads);
            Pairs<HD> x;
            x.load(A.r.q + (size_t)(q.row0 + row) * A.r.ld_q + (size_t)h * HD, g);
            x.norm_rotate(A.r, A.r.q_norm, q.start + row, g);
            x.store(A.r.q_out + (size_t)(q.row0 + row) * A.r.ld_q_out + (size_t)h * HD, g);
        }
        return;
    }
    const int head = item % A.kv.kv_heads, j = item / A.kv.kv_heads;
    const int end = q.start + q.rows, first = q.start / P, page = first + j;
    if (page * P >= end) return;
    const size_t open = ((size_t)q.slot * A.kv.kv_heads + head) * P * HD;
    auto row_of = [&](const float *x, int ld, int pos) {
        return x + (size_t)(q.row0 + pos - q.start) * ld + (size_t)head * HD;
    };
    auto open_rows = [&](int from, int to) {  // new rows of the page left open
        for (int pos = from + v; pos < to; pos += V) {
            Pairs<HD> k, x;
            k.load(row_of(A.r.k, A.r.ld_k, pos), g);
            k.norm_rotate(A.r, A.r.k_norm, pos, g);
            k.store(A.kv.k_open + open + (size_t)(pos % P) * HD, g);
            x.load(row_of(A.r.v, A.r.ld_v, pos), g);
            x.store(A.kv.v_open + open + (size_t)(pos % P) * HD, g);
        }
    };
    // The rows left open go over the open rows of the page that was begun
    // before: the block that reads those writes them, after reading.
    const bool begun = q.start % P != 0;
    if ((page + 1) * P > end) {
        if (j == 0 || !begun) open_rows(max(q.start, page * P), end);
        return;
    }
    Pairs<HD> k[PASS], x[PASS];
    unsigned top_k = 0, top_v = 0;
#pragma unroll
    for (int i = 0; i < PASS; i++) {
        const int pos = page * P + i * V + v;
        if (pos < q.start) {
            k[i].load(A.kv.k_open + open + (size_t)(pos % P) * HD, g);
            x[i].load(A.kv.v_open + open + (size_t)(pos % P) * HD, g);
        } else {
            k[i].load(row_of(A.r.k, A.r.ld_k, pos), g);
            k[i].norm_rotate(A.r, A.r.k_norm, pos, g);
            x[i].load(row_of(A.r.v, A.r.ld_v, pos), g);
        }
        top_k = max(top_k, k[i].top_bits());
        top_v = max(top_v, x[i].top_bits());
    }
    for (int off = 32; off > 0; off >>= 1) {
        top_k = max(top_k, (unsigned)__shfl_xor((int)top_k, off, 64));
        top_v = max(top_v, (unsigned)__shfl_xor((int)top_v, off, 64));
    }
    if (threadIdx.x % 64 == 0) tops[0][threadIdx.x / 64] = top_k, tops[1][threadIdx.x / 64] = top_v;
    __syncthreads();
    for (int w = 0; w < NT / 64; w++) top_k = max(top_k, tops[0][w]), top_v = max(top_v, tops[1][w]);
    const int id = q.pages[page];
    if (id >= 0 && id < A.kv.num_pages) {
        const size_t block = (size_t)id * A.kv.kv_heads + head;
        const bool fin_k = top_k < 0x7f800000u, fin_v = top_v < 0x7f800000u;
        const float tk = __uint_as_float(top_k), tv = __uint_as_float(top_v);
        const float ik = 127.0f / tk, iv = 127.0f / tv;
        if (threadIdx.x == 0) {
            A.kv.k_scales[block] = fin_k ? tk / 127.0f : __uint_as_float(0x7fc00000u);
            A.kv.v_scales[block] = fin_v ? tv / 127.0f : __uint_as_float(0x7fc00000u);
        }
        int8_t *kc = A.kv.k_codes + block * P * HD, *vc = A.kv.v_codes + block * P * HD;
        const bool zk = !fin_k || top_k == 0, zv = !fin_v || top_v == 0;
#pragma unroll
        for (int i = 0; i < PASS; i++) {
            const int t = i * V + v;
            for (int e = 0; e < 4; e++) {
                kc[t * HD + 4 * g + e] = zk ? 0 : quantize(k[i].lo[e], tk, ik);
                kc[t * HD + HD / 2 + 4 * g + e] = zk ? 0 : quantize(k[i].hi[e], tk, ik);
                vc[(4 * g + e) * P + t] = zv ? 0 : quantize(x[i].lo[e], tv, iv);
                vc[(HD / 2 + 4 * g + e) * P + t] = zv ? 0 : quantize(x[i].hi[e], tv, iv);
            }
        }
    }
    if (j == 0 && begun && end % P != 0) open_rows(end / P * P, end);
}

// One block of four waves per (row, head): each wave takes every fourth token,
// a lane HD / 64 of its dimensions.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_attn_row(PagedAttnParams A) {
    constexpr int E = HD / 64;
    __shared__ float part[4][HD + 2];
    const int P = A.kv.page_size, kvh = A.kv.kv_heads;
    const int h = blockIdx.x % A.heads;
    const int i = blockIdx.x / A.heads % A.s.max_rows, b = blockIdx.x / A.heads / A.s.max_rows;
    const PagedSeq q = load_seq(A.s, b, A.kv.num_slots, (long long)A.s.max_pages * P);
    if (i >= q.rows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head = h / (A.heads / kvh);
    const float *qr = A.q + (size_t)(q.row0 + i) * A.ld_q + (size_t)h * HD;
    float m = -INFINITY, l = 0, o[E] = {}, x[E];
    for (int e = 0; e < E; e++) x[e] = qr[lane + 64 * e];
    if (q.ok) {
        const int end = q.start + q.rows, full = end / P * P, pos = q.start + i;
        const int low = A.window > 0 && pos - A.window >= 0 ? pos - A.window + 1 : 0;
        for (int t = low + wave; t <= pos; t += 4) {
            float s = 0, y[E];
            if (t < full) {
                const int id = q.pages[t / P];
                if (id < 0 || id >= A.kv.num_pages) continue;
                const size_t block = (size_t)id * kvh + head;
                for (int e = 0; e < E; e++) {
                    s += x[e] * (float)A.kv.k_codes[(block * P + t % P) * HD + lane + 64 * e];
                    y[e] = (float)A.kv.v_codes[(block * HD + lane + 64 * e) * P + t % P] * A.kv.v_scales[block];
                }
                s *= A.kv.k_scales[block];
            } else {
                const size_t row = (((size_t)q.slot * kvh + head) * P + t % P) * HD;
                for (int e = 0; e < E; e++) {
                    s += x[e] * A.kv.k_open[row + lane + 64 * e];
                    y[e] = A.kv.v_open[row + lane + 64 * e];
                }
            }
            s = wave_sum(s) * A.scale;
            const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
            l = l * c + p;
            for (int e = 0; e < E; e++) o[e] = o[e] * c + p * y[e];
            m = mn;
        }
    }
    for (int e = 0; e < E; e++) part[wave][lane + 64 * e] = o[e];
    if (lane == 0) part[wave][HD] = m, part[wave][HD + 1] = l;
    __syncthreads();
    if (threadIdx.x < HD) {
        float mx = -INFINITY, sum = 0, acc = 0;
        for (int w = 0; w < 4; w++) mx = fmaxf(mx, part[w][HD]);
        for (int w = 0; w < 4; w++) {
            if (part[w][HD + 1] == 0.0f) continue;
            const float c = expf(part[w][HD] - mx);
            sum += c * part[w][HD + 1];
            acc += c * part[w][threadIdx.x];
        }
        A.out[(size_t)(q.row0 + i) * A.ld_out + (size_t)h * HD + threadIdx.x] = sum == 0.0f ? 0.0f : acc / sum;
    }
}

__global__ __launch_bounds__(256) void k_paged_read(PagedReadParams A, int tiles) {
    const int P = A.kv.page_size, kvh = A.kv.kv_heads, hd = A.kv.head_dim, width = kvh * hd;
    const int b = blockIdx.x / tiles, tile = blockIdx.x % tiles;
    const PagedSeq q = load_seq(A.s, b, A.kv.num_slots, (long long)A.s.max_pages * P);
    const int len = A.lens ? A.lens[b] : q.start + q.rows;
    const bool ok = q.ok && (long long)len <= (long long)A.s.max_pages * P;
    for (int r = tile * 8; r < min(tile * 8 + 8, q.rows); r++) {
        const int pos = q.start + r;
        const bool have = ok && pos < len, open = have && pos >= len / P * P;
        const int id = have && !open ? q.pages[pos / P] : -1;
        for (int d = threadIdx.x; d < width; d += 256) {
            const int head = d / hd, e = d % hd;
            float k = 0, v = 0;
            if (open) {
                const size_t at = (((size_t)q.slot * kvh + head) * P + pos % P) * hd + e;
                k = A.kv.k_open[at], v = A.kv.v_open[at];
            } else if (id >= 0 && id < A.kv.num_pages) {
                const size_t block = (size_t)id * kvh + head;
                k = (float)A.kv.k_codes[(block * P + pos % P) * hd + e] * A.kv.k_scales[block];
                v = (float)A.kv.v_codes[(block * hd + e) * P + pos % P] * A.kv.v_scales[block];
            }
            if (A.k_out) A.k_out[(size_t)(q.row0 + r) * A.ld_k + d] = k;
            if (A.v_out) A.v_out[(size_t)(q.row0 + r) * A.ld_v + d] = v;
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

}  // namespace

bool launch_paged_append(hipStream_t st, const PagedAppendParams &in) {
    PagedAppendParams p = in;
    const int P = p.kv.page_size;
    p.kv_items = (int)(((long long)p.s.max_rows + P - 2) / P + 1);
    p.q_items = p.r.q ? (int)(((long long)p.s.max_rows * p.r.heads + 63) / 64) : 0;
    const long long blocks = p.s.batch * ((long long)p.kv_items * p.kv.kv_heads + p.q_items);
    if ((long long)p.s.max_rows * p.r.heads > kPagedMaxBlocks || blocks > kPagedMaxBlocks) return false;
    if (p.kv.head_dim == 64) append_of<64>(st, p, (unsigned)blocks);
    else append_of<128>(st, p, (unsigned)blocks);
    return true;
}

bool launch_paged_attention(hipStream_t st, const PagedAttnParams &p) {
    const long long blocks = (long long)p.s.batch * p.s.max_rows * p.heads;
    if (blocks > kPagedMaxBlocks) return false;
    if (p.kv.head_dim == 64) hipLaunchKernelGGL(k_paged_attn_row<64>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(k_paged_attn_row<128>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    return true;
}

bool launch_paged_read(hipStream_t st, const PagedReadParams &p) {
    const int tiles = (p.s.max_rows + 7) / 8;
    const long long blocks = (long long)p.s.batch * tiles;
    if (blocks > kPagedMaxBlocks) return false;
    hipLaunchKernelGGL(k_paged_read, dim3((unsigned)blocks), dim3(256), 0, st, p, tiles);
    return true;
}

}  // namespace qtts
