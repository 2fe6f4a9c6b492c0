// fp8.hip — products on weights in 8-bit floats (e4m3) with a scale for each
// block of 128 x 128: y = sum over blocks b of s_w[b] (W_b x_b).
//
// The rows of x are brought to 8 bits on the way, with a power of two for each
// 128 values: the least with which they stay within 448, e4m3's largest.  The
// division is then exact, and what a value stands for is exact in bfloat16 (4
// bits of mantissa, f32's exponents), power of two included; so is a weight's
// code.  The products are taken on bfloat16 matrix instructions, whose sums keep
// 2^-23 of the largest term.  The instructions on 8-bit floats would be twice as
// fast, but within each eight products they drop what is 2^-13 below the largest
// (measured term by term, with and without their scaling): 2.3e-5 of a result on
// ordinary values, where f32 sums are at 1e-7.
#include <algorithm>

#include "device_common.h"
#include "fp8_plan.h"
#include "serve.h"

namespace qtts {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 load4(const float *p) { return *glb(reinterpret_cast<const f32x4 *>(p)); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The scale of a block whose largest magnitude has these bits, 2^(e - 127): 448
// is 0.875 * 2^9.  2^-110 at least, where the least code's value still is a normal
// bfloat16; 255 where a value is not finite.
__device__ __forceinline__ int scale_exponent(unsigned top) {
    if (top >= 0x7f800000u) return 255;
    const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);
    return e < 17 ? 17 : e;
}
__device__ __forceinline__ float power_of(int e) { return __uint_as_float((unsigned)e << 23); }

// Four values as e4m3 under a block's scale, to the nearest, ties to even; codes 0
// where the block is not finite.  Under 2^120 the code 256 would stand for 2^128: f32
// ends at 240.
__device__ __forceinline__ int codes4(f32x4 x, int e) {
    if (e == 255) return 0;
    x *= power_of(254 - e);
    if (e == 247)
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = fminf(fmaxf(x[i], -240.0f), 240.0f);
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
}

// Eight codes times a power of two.
__device__ __forceinline__ bf16x8 values8(int lo, int hi, float power) {
    union {
        bf16x8 v;
        bf16x2 h[4];
    } r;
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true);
    return r.v;
}

__device__ __forceinline__ unsigned top4(f32x4 x, unsigned m) {
#pragma unroll
    for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}

// Largest over 32 lanes, of magnitudes as bits (as integers: a NaN is the largest).
__device__ __forceinline__ unsigned half_max(unsigned v) {
    for (int off = 16; off > 0; off >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, off, 32));
    return v;
}

// Rows of x as the products take them, [rows][kb * 128] with zeros behind k.  32
// lanes a block of 128.
__global__ __launch_bounds__(256) void k_fp8_rows(Fp8Params A) {
    const int lane = threadIdx.x & 31;
    const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), blocks = (long long)A.rows * A.kb;
    if (at >= blocks) return;
    const int row = (int)(at / A.kb), b = (int)(at % A.kb), col = b * kFp8Block + 4 * lane;
    f32x4 x = {0, 0, 0, 0};
    if (col < A.w.k) x = load4(A.x + (size_t)row * A.ld_x + col);
    const int e = scale_exponent(half_max(top4(x, 0)));
    const int c = codes4(x, e);
    const float s = e == 255 ? 1.0f : power_of(e);
    int lo = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, s, false));
    int hi = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, s, true));
    if (e == 255) lo = hi = 0x7fc07fc0;
    reinterpret_cast<int2 *>(A.xc)[(size_t)at * 32 + lane] = make_int2(lo, hi);
}

// A weight in 8 bits, a block of 128 x 128 each: the same scales.
__global__ __launch_bounds__(256) void k_fp8_weight(const float *src, int ld_src, qtts_fp8_weight w, int kb) {
    __shared__ unsigned tops[4];
    const int b = blockIdx.x % kb, nb = blockIdx.x / kb, c = b * kFp8Block + 4 * (threadIdx.x & 31);
    const int r0 = nb * kFp8Block + (threadIdx.x >> 5);
    f32x4 x[16];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        x[i] = f32x4{0, 0, 0, 0};
        if (c < w.k && r0 + 8 * i < w.n) x[i] = load4(src + (size_t)(r0 + 8 * i) * ld_src + c);
        top = top4(x[i], top);
    }
    for (int off = 32; off > 0; off >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, off, 64));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    const int e = scale_exponent(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    uint8_t *codes = const_cast<uint8_t *>(w.codes);
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (c < w.k && r0 + 8 * i < w.n)
            *reinterpret_cast<int *>(codes + (size_t)(r0 + 8 * i) * w.ld + c) = codes4(x[i], e);
    if (threadIdx.x == 0)
        const_cast<float *>(w.scales)[(size_t)nb * kb + b] = e == 255 ? __uint_as_float(0x7fc00000u) : power_of(e);
}

// A weight's scale in two factors: a power of two that its codes take as they
// become bfloat16, within 2^-110 and 2^110, and the rest, for the block's sum.  A
// sum then is of the result's size: a large x beside a small scale does not leave f32.
struct Scale {
    float power, rest;
    __device__ __forceinline__ explicit Scale(float s) {
        const int e = (int)(__float_as_uint(s) >> 23 & 255), c = e == 255 ? 127 : min(max(e, 17), 237);
        power = power_of(c);
        rest = s * power_of(254 - c);
    }
};

// 16 weight rows by 16 rows of x, 32 of the contraction.  Lane (r = lane % 16, G =
// lane / 16) holds 8 values of row r of either operand and the result's rows 4 G..
// of column r.  Which 8 of a block's 128 is free; step q = 2 h + u takes 64 h + 16 G
// + 8 u and on, so that a lane reads codes 16 bytes at a time.
__device__ __forceinline__ f32x4 mma(bf16x8 w, bf16x8 x, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0);
}

__device__ __forceinline__ void fma4(f32x4 &acc, float s, f32x4 p) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = fmaf(s, p[i], acc[i]);
}

// Four columns of a row of y.
__device__ __forceinline__ void put(const Fp8Params &A, int row, int n, f32x4 v) {
    float *to = A.y + (size_t)row * A.ld_y + n;
    const float *add = A.add + (size_t)row * A.ld_add + n;
    if (n + 4 <= A.w.n) {
        if (A.add) v += load4(add);
        *glb(reinterpret_cast<f32x4 *>(to)) = v;
    } else {
        for (int i = 0; n + i < A.w.n; i++) to[i] = A.add ? v[i] + add[i] : v[i];
    }
}

// BN weight rows by BM rows of x a block, WN by WM waves; both operands' blocks
// of 128 come to LDS directly, the next ones while these are used.
template <int BN, int BM, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM, 2) void k_fp8_tile(Fp8Params A) {
    constexpr int W = WN * WM, NF = BN / WN / 16, MF = BM / WM / 16;
    static_assert(BN / WN <= kFp8Block && kFp8Block % (BN / WN) == 0, "one scale a wave");
    constexpr int LA = BN / 8 / W, LB = BM / 4 / W;  // loads of 1 KB a wave
    __shared__ __align__(16) uint8_t sa[2][BN * 128], sb[2][BM * 256];
    const int lane = threadIdx.x & 63, r = lane & 15, G = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN;
    int id = blockIdx.x;
    const int split = id % A.splits;
    id /= A.splits;
    const int n0 = id % A.tiles_n * BN, m0 = id / A.tiles_n * BM;
    const int first = split * A.each, last = min(first + A.each, A.kb);
    // A load brings 8 rows of codes or 4 of x.  A row's 16-byte pieces lie in LDS at
    // their number exclusive-or the row's (half of it for codes, whose rows are half
    // as long), so that 16 rows' same piece is in different banks.
    const uint8_t *wa[LA], *xb[LB];
    int pa[LA];
#pragma unroll
    for (int i = 0; i < LA; i++) {
        const int row = (wave * LA + i) * 8 + (lane >> 3);
        wa[i] = A.w.codes + (size_t)min(n0 + row, A.w.n - 1) * A.w.ld;
        pa[i] = 16 * ((lane & 7) ^ (row >> 1 & 7));
    }
#pragma unroll
    for (int i = 0; i < LB; i++) {
        const int row = (wave * LB + i) * 4 + (lane >> 4);
        xb[i] = A.xc + (size_t)(m0 + row) * A.kb * 256 + 16 * ((lane & 15) ^ (row & 15));
    }
    typedef __attribute__((address_space(1))) void gvoid;
    typedef __attribute__((address_space(3))) void lvoid;
    auto load = [&](int to, int b) {
#pragma unroll
        for (int i = 0; i < LA; i++) {
            // behind k a row's first piece: x has zeros there
            const int at = b * 128 + pa[i];
            __builtin_amdgcn_global_load_lds((gvoid *)(wa[i] + (at < A.w.k ? at : b * 128)),
                                             (lvoid *)(sa[to] + (wave * LA + i) * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < LB; i++)
            __builtin_amdgcn_global_load_lds((gvoid *)(xb[i] + (size_t)b * 256),
                                             (lvoid *)(sb[to] + (wave * LB + i) * 1024), 16, 0, 0);
    };
    const float *ws = A.w.scales + (size_t)(min(n0 + wn * NF * 16, A.w.n - 1) / kFp8Block) * A.kb;
    f32x4 acc[NF][MF] = {};
    load(first & 1, first);
    __syncthreads();
    for (int b = first; b < last; b++) {
        const Scale s(ws[b]);
        if (b + 1 < last) load((b + 1) & 1, b + 1);
        bf16x8 w[NF][4];
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = (wn * NF + i) * 16 + r;
                const i32x4 c = *reinterpret_cast<const i32x4 *>(sa[b & 1] + row * 128 + 16 * ((4 * h + G) ^ (row >> 1 & 7)));
                w[i][2 * h] = values8(c[0], c[1], s.power);
                w[i][2 * h + 1] = values8(c[2], c[3], s.power);
            }
#pragma unroll
        for (int j = 0; j < MF; j++) {
            const uint8_t *row = sb[b & 1] + ((wm * MF + j) * 16 + r) * 256;
            f32x4 p[NF] = {};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const bf16x8 x = *reinterpret_cast<const bf16x8 *>(row + 16 * ((8 * (q >> 1) + 2 * G + (q & 1)) ^ r));
#pragma unroll
                for (int i = 0; i < NF; i++) p[i] = mma(w[i][q], x, p[i]);
            }
#pragma unroll
            for (int i = 0; i < NF; i++) fma4(acc[i][j], s.rest, p[i]);
        }
        __syncthreads();
    }
    if (A.splits > 1) {
        // parts: [tile][split][fragment][lane], joined in order by the last
        float *part = A.part + (size_t)id * A.splits * BN * BM;
        float *mine = part + (size_t)split * BN * BM + wave * NF * MF * 256 + lane * 4;
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int j = 0; j < MF; j++)
#pragma unroll
                for (int h = 0; h < 4; h += 2)
                    st_dev_u64(reinterpret_cast<uint64_t *>(mine + (i * MF + j) * 256 + h),
                               __float_as_uint(acc[i][j][h]) | (uint64_t)__float_as_uint(acc[i][j][h + 1]) << 32);
        __shared__ unsigned arrived;
        wait_stores();
        __syncthreads();
        if (threadIdx.x == 0) {
            arrived = arrive_dev(A.counters + id);
            if (arrived == (unsigned)A.splits - 1) reset_dev(A.counters + id);
        }
        __syncthreads();
        if (arrived != (unsigned)A.splits - 1) return;
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int j = 0; j < MF; j++) acc[i][j] = f32x4{0, 0, 0, 0};
        for (int k = 0; k < A.splits; k++) {
            const float *from = part + (size_t)k * BN * BM + wave * NF * MF * 256 + lane * 4;
#pragma unroll
            for (int i = 0; i < NF; i++)
#pragma unroll
                for (int j = 0; j < MF; j++)
#pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        const uint64_t v = ld_dev_u64(reinterpret_cast<const uint64_t *>(from + (i * MF + j) * 256 + h));
                        acc[i][j][h] += __uint_as_float((unsigned)v);
                        acc[i][j][h + 1] += __uint_as_float((unsigned)(v >> 32));
                    }
        }
    }
#pragma unroll
    for (int j = 0; j < MF; j++) {
        const int row = m0 + (wm * MF + j) * 16 + r;
#pragma unroll
        for (int i = 0; i < NF; i++) {
            const int n = n0 + (wn * NF + i) * 16 + 4 * G;
            if (row < A.rows && n < A.w.n) put(A, row, n, acc[i][j]);
        }
    }
}

// Up to 16 rows: 32 weight rows a block, whose blocks of 128 its four waves take
// in turn, straight from memory to registers.  The lane that feeds x to the matrix
// instruction brings it to 8 bits itself.
__global__ __launch_bounds__(256, 2) void k_fp8_few(Fp8Params A) {
    constexpr int NF = 2;
    __shared__ f32x4 so[4][NF][64];
    const int lane = threadIdx.x & 63, r = lane & 15, G = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.x % A.splits, id = blockIdx.x / A.splits, n0 = id * 16 * NF;
    const int first = split * A.each, last = min(first + A.each, A.kb);
    const uint8_t *wr[NF];
#pragma unroll
    for (int i = 0; i < NF; i++) wr[i] = A.w.codes + (size_t)min(n0 + 16 * i + r, A.w.n - 1) * A.w.ld;
    const float *xr = A.x + (size_t)min(r, A.rows - 1) * A.ld_x;
    const float *ws = A.w.scales + (size_t)(n0 / kFp8Block) * A.kb;
    f32x4 acc[NF] = {};
    for (int b = first + wave; b < last; b += 4) {
        i32x4 w[NF][2];
        f32x4 x[8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int at = b * 128 + 64 * h + 16 * G, to = at < A.w.k ? at : b * 128;
#pragma unroll
            for (int i = 0; i < NF; i++) w[i][h] = *glb(reinterpret_cast<const i32x4 *>(wr[i] + to));
#pragma unroll
            for (int j = 0; j < 4; j++) x[4 * h + j] = load4(xr + to + 4 * j);
#pragma unroll
            for (int j = 0; j < 4; j++) x[4 * h + j] = at < A.w.k ? x[4 * h + j] : f32x4{0, 0, 0, 0};
        }
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) top = top4(x[j], top);
        for (int off = 16; off < 64; off <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, off, 64));
        const int e = scale_exponent(top);
        const float sx = e == 255 ? __uint_as_float(0x7fc00000u) : 1.0f;  // a row that is not finite
        const Scale s(ws[b]);
        f32x4 p[NF] = {};
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const bf16x8 v = values8(codes4(x[2 * q], e), codes4(x[2 * q + 1], e), e == 255 ? 1.0f : power_of(e));
#pragma unroll
            for (int i = 0; i < NF; i++)
                p[i] = mma(values8(w[i][q >> 1][2 * (q & 1)], w[i][q >> 1][2 * (q & 1) + 1], s.power), v, p[i]);
        }
#pragma unroll
        for (int i = 0; i < NF; i++) fma4(acc[i], s.rest * sx, p[i]);
    }
#pragma unroll
    for (int i = 0; i < NF; i++) so[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= NF) return;
    f32x4 v = so[0][wave][lane];
#pragma unroll
    for (int k = 1; k < 4; k++) v += so[k][wave][lane];
    const int n = n0 + 16 * wave + 4 * G;
    if (A.splits > 1) {
        // each wave joins its own 16 columns
        float *part = A.part + ((size_t)id * NF + wave) * A.splits * 256;
        float *mine = part + split * 256 + lane * 4;
        for (int h = 0; h < 4; h += 2)
            st_dev_u64(reinterpret_cast<uint64_t *>(mine + h),
                       __float_as_uint(v[h]) | (uint64_t)__float_as_uint(v[h + 1]) << 32);
        wait_stores();
        unsigned arrived = 0;
        unsigned *counter = A.counters + id * NF + wave;
        if (lane == 0) {
            arrived = arrive_dev(counter);
            if (arrived == (unsigned)A.splits - 1) reset_dev(counter);
        }
        arrived = __builtin_amdgcn_readfirstlane(arrived);
        if (arrived != (unsigned)A.splits - 1) return;
        v = f32x4{0, 0, 0, 0};
        for (int k = 0; k < A.splits; k++)
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
                const uint64_t z = ld_dev_u64(reinterpret_cast<const uint64_t *>(part + k * 256 + lane * 4 + h));
                v[h] += __uint_as_float((unsigned)z);
                v[h + 1] += __uint_as_float((unsigned)(z >> 32));
            }
    }
    if (r < A.rows && n < A.w.n) put(A, r, n, v);
}

}  // namespace

void launch_fp8_gemm(hipStream_t st, const Fp8Params &in) {
    const int most = fp8_rows_at_once(in.w.k);
    for (int at = 0; at < in.rows; at += most) {
        Fp8Params p = in;
        p.x += (size_t)at * p.ld_x;
        p.y += (size_t)at * p.ld_y;
        if (p.add) p.add += (size_t)at * p.ld_add;
        p.rows = std::min(in.rows - at, most);
        p.kb = fp8_blocks(p.w.k);
        const Fp8Plan plan = fp8_plan(p.rows, p.w.n, p.w.k);
        p.tiles_n = plan.tiles_n;
        p.splits = plan.splits;
        p.each = (p.kb + plan.splits - 1) / plan.splits;
        const unsigned blocks = (unsigned)plan.tiles_n * plan.tiles_m * plan.splits;
        if (plan.bm <= 16) {
            hipLaunchKernelGGL(k_fp8_few, dim3(blocks), dim3(256), 0, st, p);
            continue;
        }
        const long long rows_blocks = ((long long)p.rows * p.kb + 7) / 8;
        hipLaunchKernelGGL(k_fp8_rows, dim3((unsigned)rows_blocks), dim3(256), 0, st, p);
        hipLaunchKernelGGL((k_fp8_tile<256, 128, 4, 2>), dim3(blocks), dim3(512), 0, st, p);
    }
}

void launch_fp8_quantize(hipStream_t st, const float *src, int ld_src, const qtts_fp8_weight &w) {
    const int kb = fp8_blocks(w.k), nb = (w.n + kFp8Block - 1) / kFp8Block;
    hipLaunchKernelGGL(k_fp8_weight, dim3((unsigned)nb * kb), dim3(256), 0, st, src, ld_src, w, kb);
}

}  // namespace qtts
