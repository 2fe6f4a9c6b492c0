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
// (measured term by term, with and without their scaling): over 128 products of normal
// values 1.5e-5 of the result, of values of many sizes 5e-5, where the bfloat16 ones have
// 9e-9 and 2.6e-8.
#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "fp8_plan.h"
#include "serve.h"

namespace qtts {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
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

template <int CTRL>
__device__ __forceinline__ unsigned dpp_bits(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}

// Largest over 16 lanes, of magnitudes as bits (as integers: a NaN is the largest).
__device__ __forceinline__ unsigned row_max(unsigned v) {
    v = max(v, dpp_bits<kDppXor1>(v));
    v = max(v, dpp_bits<kDppXor2>(v));
    v = max(v, dpp_bits<kDppHalfMirror>(v));
    return max(v, dpp_bits<kDppMirror>(v));
}

// Where a row's 16-byte pieces lie in LDS, of four: at place_of(piece) exclusive-or a
// quarter of the row's number.  A read of 16 bytes a lane takes lanes 0-3, 12-15 and
// 20-27 together, then 4-11, 16-19 and 28-31: their pieces, of two kinds, are then in
// different banks (with the piece's own number they meet in pairs, and a read takes
// twice as long).
__device__ __forceinline__ int place_of(int piece) { return (piece & 1 ? 3 : 0) ^ (piece >> 1); }

// 128 values of a row as the products take them, in 8 bits and back: eight a lane of 16.
__device__ __forceinline__ u32x4 block_values(f32x4 x, f32x4 y) {
    const int e = scale_exponent(row_max(top4(y, top4(x, 0))));
    const float s = e == 255 ? 1.0f : power_of(e);
    const bf16x8 v = values8(codes4(x, e), codes4(y, e), s);
    return e == 255 ? u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u} : __builtin_bit_cast(u32x4, v);
}

// Rows lie in pieces of 1 KB, 16 of them and half of 64 of the contraction (of every 16
// the first 8, or the others), as they are to lie in LDS.
// All rows to scratch, [row / 16][k / 64][half], zeros behind k.  A wave a block of 128
// of four rows, kRowsAhead blocks one after another whose loads are in flight together.
// Bound by memory: 8192 rows of 2048, 101 MB, in 27 us; 2100 of 6144 12.6 (four blocks a
// wave 13.6); small ones by latency, 17 of 6144 3.4 us (4.2).
//
// The blocks behind those of the rows find how the tiles' unit changes along k
// (Fp8Params::changes), a wave a row of the weight's scales, 64 at a time: 40 rows of 33
// blocks 3.8 us, 3.6 without them, and no more where there are more rows.  (A factor found
// in the tiles themselves, its rounding carried on, took their step 2 to 5 % longer.)
constexpr int kRowsAhead = 2;
__device__ void unit_changes(const Fp8Params &A, int nb) {
    const int lane = threadIdx.x & 63;
    if (nb * kFp8Block >= A.w.n) return;
    const float *ws = A.w.scales + (size_t)nb * A.kb;
    int carried = 0;
    for (int b0 = 0; b0 < A.kb; b0 += 64) {
        const int b = min(b0 + lane, A.kb - 1);
        const unsigned scale = __float_as_uint(*glb(ws + b)), last = __float_as_uint(*glb(ws + max(b - 1, 0)));
        const float from = __uint_as_float(fp8_unit(last)), to = __uint_as_float(fp8_unit(scale));
        const Fp8Change c = fp8_change(from, to, __builtin_amdgcn_rcpf(from), __builtin_amdgcn_rcpf(to));
        // Carried from lane to lane of 16, a block in each turn, and from 16 to 16 what the
        // last of them has left (a product of factors is so within 2^-23).
        int factor = c.quotient, before = 0;
        if (carried != 0 || __any(c.left != 0)) {
#pragma unroll
            for (int turn = 0; turn < 15; turn++)  // row_shr:1, the first gets 0
                before = __builtin_amdgcn_update_dpp(0, fp8_carry(c, before), 0x111, 0xF, 0xF, true);
            factor += fp8_step(c, before);
            const unsigned long long apart = __ballot(fp8_apart(c.quotient));
            const int after = fp8_carry(c, before);
#pragma unroll
            for (int row = 0; row < 4; row++) {
                const unsigned at = (unsigned)(apart >> 16 * row) & 0xffffu;
                carried += __builtin_amdgcn_readlane(after, 16 * row + 15);
                if (at == 0) continue;
                const int l = 16 * row + 31 - __builtin_clz(at);
                const Fp8Change all{0, 0, __builtin_amdgcn_readlane(c.half, l)};
                const int step = fp8_step(all, carried);
                factor += lane == l ? step : 0;
                carried = fp8_carry(all, carried);
            }
        }
        if (b0 + lane < A.kb) A.changes[(size_t)nb * A.kb + b0 + lane] = {(int)fp8_power(scale), factor};
    }
}

__host__ __device__ __forceinline__ int rows_blocks(int rows, int kb) {
    return (int)(((rows + 3) / 4 * (long long)kb + 4 * kRowsAhead - 1) / (4 * kRowsAhead));
}

template <bool TILES>
__global__ __launch_bounds__(256) void k_fp8_rows(Fp8Params A) {
    if (TILES) {
        const int beyond = (int)blockIdx.x - rows_blocks(A.rows, A.kb);
        if (beyond >= 0) return unit_changes(A, 4 * beyond + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    }
    const int lane = threadIdx.x & 15, sub = threadIdx.x >> 4 & 3;
    const long long at = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * kRowsAhead;
    const long long blocks = (long long)((A.rows + 3) / 4) * A.kb;
    f32x4 x[kRowsAhead][2];
#pragma unroll
    for (int i = 0; i < kRowsAhead; i++) {
        const long long b = min(at + i, blocks - 1);
        const int col = (int)(b % A.kb) * kFp8Block + 8 * lane, row = min((int)(b / A.kb) * 4 + sub, A.rows - 1);
        const float *from = A.x + (size_t)row * A.ld_x + (col < A.w.k ? col : 0);
        x[i][0] = load4(from), x[i][1] = load4(from + 4);
        if (col >= A.w.k) x[i][0] = x[i][1] = f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < kRowsAhead; i++) {
        const u32x4 v = block_values(x[i][0], x[i][1]);
        const int row = (int)((at + i) / A.kb) * 4 + sub, b = (int)((at + i) % A.kb);
        uint8_t *to = A.xc + ((size_t)(row >> 4) * A.kb + b) * 4096 + (lane >> 3) * 2048 + (lane & 1) * 1024;
        const int place = place_of(lane >> 1 & 3) ^ (row >> 2 & 3);
        if (at + i < blocks && row < A.rows) *glb(reinterpret_cast<u32x4 *>(to + (row & 15) * 64 + place * 16)) = v;
    }
}

// A weight in 8 bits, a block of 128 x 128 each: the same scales.  Bound by memory: 12288
// rows of 2048, 126 MB, in 21.7 us (5.8 TB/s); 256 of 256 4.1, latency.
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
// become bfloat16, within 2^-117 and 2^117, and the rest: 1 to 2, but 2^-32 and on,
// or to 2^11, for a scale that is `far` out, at the ends of f32.  A sum then is of the
// result's size: a large x beside a small scale does not leave f32.
struct Scale {
    float power, rest;
    bool none, bad, far;  // 0; Inf or NaN
    __device__ __forceinline__ explicit Scale(float s) {
        const int e = (int)(__float_as_uint(s) >> 23 & 255), c = min(max(e, 10), 244);
        none = s == 0.0f, bad = e == 255, far = !none && !bad && e != c;
        power = none || bad ? 1.0f : power_of(c);
        rest = none || bad ? 1.0f : s * power_of(254 - c);
    }
};

// 16 weight rows by 16 rows of x, 32 of the contraction.  Lane (r = lane % 16, G =
// lane / 16) holds 8 values of row r of either operand and the result's rows 4 G..
// of column r.  Which 8 is free: of 64, half u takes 16 G + 8 u and on, so that a lane
// reads codes 16 bytes at a time.
__device__ __forceinline__ f32x4 mma(bf16x8 w, bf16x8 x, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0);
}

template <int N, class F>
__device__ __forceinline__ void each(F &&f) {
    if constexpr (N > 0) {
        each<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

// Where a lane's four sums of a part of a divided tile lie: by fragments, each as a wave
// stores it.
template <int BN, int BM>
__device__ __forceinline__ f32x4 *part_of(const Fp8Params &A, size_t part, int fragment, int lane) {
    return reinterpret_cast<f32x4 *>(A.part) + (part * (BN / 16 * (BM / 16)) + fragment) * 64 + lane;
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

// 16 bytes a lane from memory to LDS, 1 KB in a row from `to` on.  Written out, as the
// compiler has every read of LDS wait for all such loads before it; whoever uses
// what they bring waits for them himself.
__device__ __forceinline__ void to_lds(const uint8_t *base, unsigned offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to));
}
__device__ __forceinline__ unsigned lds_address(void *p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)p;
}

// BN weight rows by BM rows of x a block, WN by WM waves.  A step is 64 of the
// contraction in two halves of x; both operands come to LDS directly, two steps
// ahead: x by halves in rings of three, codes by blocks of 128 in a ring of two, in
// whole lines of 128 bytes (16 rows of 64 bytes a load reach half the rate from L2: 71
// GB/s a CU with all of them loading, 132).  The one barrier of a step lies between
// its halves: behind it the second half, the next step's codes and its first half are
// read and multiplied in one stretch, so that neither the reads nor the codes'
// conversion wait for a barrier of their own.
//
// Sums are held in units of the current block's `rest` (fp8_unit), one multiplication
// for each 128: a second set of sums for the block would take the registers of the tile.
// The unit stays within 1 and 2, or a sum would leave f32 in it: blocks whose scale is far
// out are zeros in the steps and are added after them, each under its own scale.  The
// factors between units are k_fp8_rows', which has their roundings not add up: found here
// as rest * (1 / rest), a product of them was up to 2.4e-6 off after 48 blocks, always to
// one side, and 1 only by chance between equal scales.
//
// 256 x 256, 8192 rows, 2048 to 12288: a call takes 382 us of which the rows are 27,
// so some 355, 1.16 PFLOP/s, where 8192 cubed in bfloat16 is 1.24 in the library (375
// to 420 in a kernel trace, under which the clock is lower).  Of a step's 2950 cycles
// the products take 2048 (two waves a SIMD); the multiplications, the conversions and
// the loads' addresses, some 300 each, overlap with them in part, and at 1.9 to 2.1
// GHz the card's power bounds both.  Measured on the way: all loads right behind the
// barrier 3400 cycles, a barrier behind each half 4000; a pattern of products and
// other instructions imposed on the compiler's order 3150 to 4200.
//
// Eight waves on 128 x 128 rather than four: 512 rows, 2048 to 4096, 20.6 us against
// 23.5; 2048 rows, 6144 to 2048, 52.8 against 59.9.
template <int BN, int BM, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM, 2) void k_fp8_tile(Fp8Params A) {
    constexpr int W = WN * WM, NF = BN / WN / 16, MF = BM / WM / 16;
    static_assert(BN / WN <= kFp8Block && kFp8Block % (BN / WN) == 0, "one scale a wave");
    constexpr int LA = BN / 8 / W, LB = BM / 16 / W;  // loads of 1 KB a wave, of codes and of half of x
    constexpr int kCodes = BN * 128, kHalf = BM * 64;
    __shared__ __align__(16) uint8_t ring[2 * kCodes + 6 * kHalf];  // codes [2], x [3][2]
    const unsigned ring_at = lds_address(ring);
    const int lane = threadIdx.x & 63, r = lane & 15, G = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN;
    int id = blockIdx.x, first = 0, last = (A.w.k + 63) / 64;
    const int part = id - A.whole;
    const bool divided = A.splits > 1 && part >= 0;
    if (divided) {
        id = A.whole + part / A.splits;
        first = 2 * A.each * (part % A.splits);
        last = min(first + 2 * A.each, last);
    }
    const int n0 = id % A.tiles_n * BN, m0 = id / A.tiles_n * BM;
    // A load of codes brings 8 rows of 128 bytes; their eight pieces lie in LDS at
    // their number exclusive-or half of the row's.
    const uint8_t *codes = A.w.codes + (size_t)n0 * A.w.ld, *xs = A.xc + (size_t)(m0 / 16 + wave * LB) * A.kb * 4096;
    unsigned row_at[LA];
    int piece[LA];
#pragma unroll
    for (int i = 0; i < LA; i++) {
        const int row = (wave * LA + i) * 8 + (lane >> 3);
        row_at[i] = (unsigned)min(row, A.w.n - 1 - n0) * (unsigned)A.w.ld;
        piece[i] = 16 * ((lane & 7) ^ (row >> 1 & 7));
    }
    auto load_half = [&](int slot, int s, int u, int i) {
        to_lds(xs + ((size_t)i * A.kb * 4096 + (size_t)s * 2048 + u * 1024), lane * 16,
               ring_at + 2 * kCodes + (2 * slot + u) * kHalf + (wave * LB + i) * 1024);
    };
    auto load_codes = [&](int s, int i) {  // of the block that begins with step s
        // behind k the block's first codes: x has zeros there
        const unsigned at = piece[i] < A.w.k - s * 64 ? piece[i] : 0;
        to_lds(codes + (size_t)s * 64, row_at[i] + at, ring_at + (s >> 1 & 1) * kCodes + (wave * LA + i) * 1024);
    };
    // where this lane reads: its row of a fragment, its piece
    const int my_code = r * 128 + 16 * (G ^ (r >> 1)), my_x = r * 64 + 16 * (place_of(G) ^ (r >> 2));
    auto codes_at = [&](int s, int i) {
        return *reinterpret_cast<const i32x4 *>(ring + (s >> 1 & 1) * kCodes + (wn * NF + i) * 2048 +
                                                (my_code ^ (s & 1) * 64));
    };
    auto half_at = [&](int slot, int u, int j) {
        return *reinterpret_cast<const bf16x8 *>(ring + 2 * kCodes + (2 * slot + u) * kHalf + (wm * MF + j) * 1024 + my_x);
    };
    const size_t scales_at = (size_t)(min(n0 + wn * NF * 16, A.w.n - 1) / kFp8Block) * A.kb;
    const KCONST float *ws = (const KCONST float *)A.w.scales + scales_at;
    f32x4 acc[NF][MF] = {};
    // 64 blocks' power and factor, a lane each, from block `ahead` on: a scalar load in each
    // block would be waited for there
    i32x2 changes;
    int ahead;
    auto look_ahead = [&](int b) {
        ahead = b;
        changes = *glb(reinterpret_cast<const i32x2 *>(A.changes) + scales_at + min(b + lane, A.kb - 1));
    };
    float rest = ws[(last - 1) >> 1], power = 1.0f, by = 1.0f;
    int met = 0;
    bool none = false;
    i32x4 c[NF];    // this step's codes
    bf16x8 w[NF];   // the half at hand
    auto half = [&](int slot, int u, float by, bool scaled, auto &&between) {
        each<MF>([&](auto j) {
            const bf16x8 x = half_at(slot, u, j);
#pragma unroll
            for (int i = 0; i < NF; i++) {
                if (scaled) acc[i][j] *= by;  // just before its products, behind others'
                acc[i][j] = mma(w[i], x, acc[i][j]);
            }
            between(j);
        });
    };
    auto nothing = [](int) {};
    auto new_block = [&](int s) {  // its scale
        const int l = (s >> 1) - ahead, bits = __builtin_amdgcn_readlane(changes[0], l);
        power = __int_as_float(bits), by = __int_as_float(__builtin_amdgcn_readlane(changes[1], l));
        none = bits & kFp8None, met |= bits;
    };
    // codes under a scale of 0 are zeros, and for now under one far out; every wave that
    // reads these writes them
    auto clear_codes = [&](int s) {
        for (int i = 0; i < NF; i++)
            *reinterpret_cast<i32x4 *>(ring + (s >> 1 & 1) * kCodes + (wn * NF + i) * 2048 + (my_code ^ (s & 1) * 64)) =
                i32x4{0, 0, 0, 0};
    };
    // a step's codes, its first half and the conversion for the second
    auto begin = [&](int slot, int s, auto block) {
#pragma unroll
        for (int i = 0; i < NF; i++) {
            c[i] = codes_at(s, i);
            w[i] = values8(c[i][0], c[i][1], power);
        }
        half(slot, 0, by, block, nothing);
#pragma unroll
        for (int i = 0; i < NF; i++) w[i] = values8(c[i][2], c[i][3], power);
    };
    // From the middle of step s to that of the next one.  At the barrier what is read
    // behind it is here (what the last step asked for may be on its way), and what the
    // loads behind it go over has been read.  They are spread among the products, as
    // both waves of a SIMD come from the barrier together.  far: there are three more
    // steps, and the loads are on no branch.
    auto through = [&](int slot, int s, auto odd, auto far) {
        constexpr int kAway = 2 * LB + (odd ? 0 : LA), kNew = 2 * LB + (odd ? LA : 0), kEach = (kNew + MF - 1) / MF;
        const int next_slot = slot == 2 ? 0 : slot + 1;
        if (odd) new_block(s + 1);
        if (far || s + 2 < last) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kAway) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        auto load = [&](auto l) {  // the new loads in their order
            if constexpr (l < LB) load_half(slot == 0 ? 2 : slot - 1, s + 2, 1, l);
            else if constexpr (odd && l < LB + LA) load_codes(s + 3, l - LB);
            else if constexpr (l < kNew) load_half(slot, s + 3, 0, l - (kNew - LB));
        };
        if (!far) {
            if (s + 2 < last) each<LB>(load);
            if (s + 3 < last)
                each<kNew>([&](auto l) {
                    if constexpr (l >= LB) load(l);
                });
        }
        if (none) clear_codes(s + 1);
        half(slot, 1, 1.0f, false, [&](auto j) {
            if constexpr (far)
                each<kEach>([&](auto e) { load(std::integral_constant<int, j * kEach + e>{}); });
        });
        begin(next_slot, s + 1, odd);
        return next_slot;
    };
    auto more_ahead = [&](int s) {
        if ((s >> 1) + 1 - ahead < 64) return;
        look_ahead((s >> 1) + 1);
        asm volatile("" : "+v"(changes));  // waited for here, not in every block
    };
    const auto yes = std::true_type{};
    const auto no = std::false_type{};
    look_ahead(first >> 1);
    each<LA>([&](auto i) { load_codes(first, i); });
    each<LB>([&](auto i) { load_half(0, first, 0, i), load_half(0, first, 1, i); });
    if (first + 1 < last) each<LB>([&](auto i) { load_half(1, first + 1, 0, i), load_half(1, first + 1, 1, i); });
    if (first + 2 < last) {
        each<LA>([&](auto i) { load_codes(first + 2, i); });
        each<LB>([&](auto i) { load_half(2, first + 2, 0, i); });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    new_block(first);
    if (none) clear_codes(first);
    int slot = 0, s = first;
    begin(slot, first, yes);
    for (; s + 4 < last; s += 2) {
        more_ahead(s);
        slot = through(slot, s, no, yes);
        slot = through(slot, s + 1, yes, yes);
    }
    for (; s + 2 < last; s += 2) {
        more_ahead(s);
        slot = through(slot, s, no, no);
        slot = through(slot, s + 1, yes, no);
    }
    if (s + 1 < last) slot = through(slot, s, no, no);
    half(slot, 1, 1.0f, false, nothing);
    rest = __uint_as_float(met & kFp8Bad ? 0x7fc00000u : fp8_unit(__float_as_uint(rest)));
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) acc[i][j] *= rest;
    // straight from memory to registers, as without tiles
    for (int b = first >> 1; met & kFp8Far && 2 * b < last; b++) {
        const Scale z(ws[b]);
        if (!z.far) continue;
#pragma unroll 1
        for (int q = 0; q < 4; q++) {
            const int at = b * 128 + 64 * (q >> 1) + 16 * G + 8 * (q & 1);
            const uint8_t *wr = A.w.codes + (at < A.w.k ? at : b * 128);
            const uint8_t *xr = A.xc + ((size_t)(m0 / 16 + wm * MF) * A.kb + b) * 4096 + q * 1024 + my_x;
#pragma unroll
            for (int i = 0; i < NF; i++) {
                const int n = min(n0 + (wn * NF + i) * 16 + r, A.w.n - 1);
                const i32x2 v = *glb(reinterpret_cast<const i32x2 *>(wr + (size_t)n * A.w.ld));
                w[i] = values8(v[0], v[1], z.power);
            }
#pragma unroll
            for (int j = 0; j < MF; j++) {
                const bf16x8 x = *glb(reinterpret_cast<const bf16x8 *>(xr + (size_t)j * A.kb * 4096));
#pragma unroll
                for (int i = 0; i < NF; i++) {
                    const f32x4 p = mma(w[i], x, f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(z.rest, p[e], acc[i][j][e]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MF; j++) {
        const int row = m0 + (wm * MF + j) * 16 + r;
#pragma unroll
        for (int i = 0; i < NF; i++) {
            const int n = n0 + (wn * NF + i) * 16 + 4 * G;
            if (row >= A.rows || n >= A.w.n) continue;
            if (divided) *glb(part_of<BN, BM>(A, part, (wave * NF + i) * MF + j, lane)) = acc[i][j];
            else put(A, row, n, acc[i][j]);
        }
    }
}

// The parts' sums of the divided tiles, in their order.  Four columns a thread.
template <int BN, int BM, int WN, int WM>
__global__ __launch_bounds__(256) void k_fp8_join(Fp8Params A) {
    constexpr int F = BN / 16 * (BM / 16), NF = BN / WN / 16, MF = BM / WM / 16;
    const int lane = threadIdx.x & 63, r = lane & 15, G = lane >> 4;
    const int at = blockIdx.x * 4 + (threadIdx.x >> 6), tile = at / F, f = at % F;  // a wave a fragment
    const int wave = f / (NF * MF), i = f / MF % NF, j = f % MF, id = A.whole + tile;
    const int row = id / A.tiles_n * BM + (wave / WN * MF + j) * 16 + r;
    const int n = id % A.tiles_n * BN + (wave % WN * NF + i) * 16 + 4 * G;
    if (row >= A.rows || n >= A.w.n) return;
    f32x4 v = {0, 0, 0, 0};
    for (int k0 = 0; k0 < A.splits; k0 += 8) {
        f32x4 p[8];
#pragma unroll
        for (int k = 0; k < 8; k++)
            p[k] = *glb(part_of<BN, BM>(A, (size_t)tile * A.splits + min(k0 + k, A.splits - 1), f, lane));
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k0 + k < A.splits) v += p[k];
    }
    put(A, row, n, v);
}

// Without tiles: 16 weight rows by RF times 16 of x a block, whose blocks of 128 its W
// waves take in turn, straight from memory to registers.  OWN: the block meanwhile
// brings x to 8 bits itself, into LDS (fp8_own_rows); otherwise it comes from scratch,
// which k_fp8_rows has filled.  Bound by a chain of latencies and by what every block
// reads of the weight and of x from L2 (75 GB/s a CU).  In a kernel trace one row, 2048 to
// 12288, 25 MB, takes 9 to 9.9 us (2.5 to 2.8 TB/s; 8.8 among calls in a graph); 16 rows,
// 6144 to 2048 8.1 us, 2048 to 4096 4.4, 32 of these 5.6, 64 8.1.  With 32 weight rows a
// block, half of x's reads and half of the blocks, these three took 1.3 to 1.4 times as long.
template <int W, bool OWN, int RF>
__global__ __launch_bounds__(64 * W, W == 4 ? 3 : RF > 1 ? 2 : 4) void k_fp8_few(Fp8Params A) {
    constexpr int kAhead = 4 / RF;  // blocks of 128 asked for at once
    extern __shared__ __align__(16) uint8_t lds[];  // sums of the waves, then x as in scratch, `side` rows a piece
    f32x4 *so = reinterpret_cast<f32x4 *>(lds);
    uint8_t *xs = lds + W * RF * 1024;
    const int lane = threadIdx.x & 63, r = lane & 15, G = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x % A.tiles_n * 16, group = blockIdx.x / A.tiles_n;
    const uint8_t *wr = A.w.codes + (size_t)min(n0 + r, A.w.n - 1) * A.w.ld;
    const KCONST float *ws = (const KCONST float *)(A.w.scales + (size_t)(n0 / kFp8Block) * A.kb);
    i32x4 w[kAhead][2];
    bf16x8 xv[OWN ? 1 : kAhead][RF][4];
    float scale[kAhead];
    const int side = OWN && A.rows <= kFewRows ? A.rows : 16, mine = min(r, side - 1);
    const uint8_t *xr = (OWN ? xs : A.xc + (size_t)group * RF * A.kb * 4096) + mine * 64 + 16 * (place_of(G) ^ (mine >> 2));
    auto ask = [&](int b0) {
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            const int b = min(b0 + W * a, A.kb - 1);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int at = b * 128 + 64 * h + 16 * G;  // behind k the block's first codes: x has zeros there
                w[a][h] = *glb(reinterpret_cast<const i32x4 *>(wr + (at < A.w.k ? at : b * 128)));
            }
            scale[a] = ws[b];
            if (!OWN)
#pragma unroll
                for (int f = 0; f < RF; f++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        xv[OWN ? 0 : a][f][q] =
                            *glb(reinterpret_cast<const bf16x8 *>(xr + ((size_t)f * A.kb + b) * 4096 + q * 1024));
        }
    };
    ask(wave);
    const int items = OWN ? min(A.rows - 16 * group, 16) * A.kb : 0;  // 16 lanes a row's block of 128
    for (int i0 = threadIdx.x >> 4; i0 < items; i0 += 16 * W) {
        f32x4 x[4][2];
        const int l = threadIdx.x & 15;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int it = min(i0 + 4 * W * i, items - 1), col = it % A.kb * kFp8Block + 8 * l;
            const float *from = A.x + (size_t)(16 * group + it / A.kb) * A.ld_x + (col < A.w.k ? col : 0);
            x[i][0] = load4(from), x[i][1] = load4(from + 4);
            if (col >= A.w.k) x[i][0] = x[i][1] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int it = i0 + 4 * W * i, row = it / A.kb, piece = it % A.kb * 4 + 2 * (l >> 3) + (l & 1);
            const u32x4 v = block_values(x[i][0], x[i][1]);
            if (it < items)
                *reinterpret_cast<u32x4 *>(xs + (piece * side + row) * 64 + 16 * (place_of(l >> 1 & 3) ^ (row >> 2))) = v;
        }
    }
    if (OWN) __syncthreads();
    f32x4 acc[RF] = {};
    for (int b0 = wave; b0 < A.kb; b0 += kAhead * W) {
        if (b0 != wave) ask(b0);
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            const int b = b0 + W * a;
            if (b >= A.kb) break;
            const Scale s(scale[a]);
            const int mask = s.none ? 0 : -1;  // codes under a scale of 0 are zeros
            const float by = s.bad ? __uint_as_float(0x7fc00000u) : s.rest;
            f32x4 p[RF] = {};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const i32x4 c = w[a][q >> 1];
                const bf16x8 v = values8(c[2 * (q & 1)] & mask, c[2 * (q & 1) + 1] & mask, s.power);
#pragma unroll
                for (int f = 0; f < RF; f++) {
                    const uint8_t *at = xr + ((f * A.kb + b) * 4 + q) * side * 64;
                    p[f] = mma(v, OWN ? *reinterpret_cast<const bf16x8 *>(at) : xv[OWN ? 0 : a][f][q], p[f]);
                }
            }
#pragma unroll
            for (int f = 0; f < RF; f++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[f][i] = fmaf(by, p[f][i], acc[f][i]);
        }
    }
#pragma unroll
    for (int f = 0; f < RF; f++) so[(f * W + wave) * 64 + lane] = acc[f];
    __syncthreads();
    if (wave >= RF) return;  // a wave for 16 rows
    f32x4 sum = so[wave * W * 64 + lane];
#pragma unroll
    for (int k = 1; k < W; k++) sum += so[(wave * W + k) * 64 + lane];
    const int n = n0 + 4 * G, row = 16 * (group * RF + wave) + r;
    if (row < A.rows && n < A.w.n) put(A, row, n, sum);
}

template <int W, bool OWN, int RF>
void few_of(hipStream_t st, const Fp8Params &p, size_t x_bytes) {
    const unsigned blocks = (unsigned)p.tiles_n * (unsigned)((p.rows + 16 * RF - 1) / (16 * RF));
    hipLaunchKernelGGL((k_fp8_few<W, OWN, RF>), dim3(blocks), dim3(64 * W), W * RF * 1024 + x_bytes, st, p);
}

template <int BN, int BM, int WN, int WM>
void tiles_of(hipStream_t st, const Fp8Params &p, const Fp8Plan &plan) {
    hipLaunchKernelGGL((k_fp8_tile<BN, BM, WN, WM>), dim3((unsigned)fp8_launched(plan)), dim3(64 * WN * WM), 0, st, p);
    if (plan.splits == 1) return;
    const unsigned waves = (unsigned)(plan.tiles_n * plan.tiles_m - plan.whole) * (BN / 16 * (BM / 16));
    hipLaunchKernelGGL((k_fp8_join<BN, BM, WN, WM>), dim3(waves / 4), dim3(256), 0, st, p);
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
        p.whole = plan.whole;
        p.splits = plan.splits;
        p.each = plan.each;
        if (fp8_own_rows(p.rows, p.w.n, p.kb)) {
            const size_t x_bytes = (size_t)fp8_own_bytes(p.rows, p.kb);
            if (plan.waves == 4) few_of<4, true, 1>(st, p, x_bytes);
            else few_of<8, true, 1>(st, p, x_bytes);
            continue;
        }
        const unsigned blocks = rows_blocks(p.rows, p.kb);
        if (plan.bn == 16) {
            hipLaunchKernelGGL(k_fp8_rows<false>, dim3(blocks), dim3(256), 0, st, p);
            if (plan.bm == 16) few_of<8, false, 1>(st, p, 0);
            else if (plan.bm == 32) few_of<8, false, 2>(st, p, 0);
            else few_of<8, false, 4>(st, p, 0);
            continue;
        }
        const unsigned scale_rows = fp8_blocks(p.w.n);
        hipLaunchKernelGGL(k_fp8_rows<true>, dim3(blocks + (scale_rows + 3) / 4), dim3(256), 0, st, p);
        if (plan.bm == 256) tiles_of<256, 256, 4, 2>(st, p, plan);
        else if (plan.bm == 128) tiles_of<128, 128, 4, 2>(st, p, plan);
        else tiles_of<64, 64, 2, 2>(st, p, plan);
    }
}

void launch_fp8_quantize(hipStream_t st, const float *src, int ld_src, const qtts_fp8_weight &w) {
    const int kb = fp8_blocks(w.k), nb = (w.n + kFp8Block - 1) / kFp8Block;
    hipLaunchKernelGGL(k_fp8_weight, dim3((unsigned)nb * kb), dim3(256), 0, st, src, ld_src, w, kb);
}

}  // namespace qtts
