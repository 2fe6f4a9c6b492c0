// fp8_plan.h — what decides which memory the products on 8-bit floats touch: the
// checks of a call's arguments and how its work is divided.  Plain C++ without
// device code, so that the CPU tests run the same lines.
#pragma once

#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "../../include/qtts.h"
#include "paged_plan.h"

namespace qtts {

constexpr int kFp8Block = 128;                    // side of a weight's block, length of a row's
constexpr int kFp8MaxSide = 1 << 17;              // of n and k
constexpr int kFp8MaxStride = 1 << 23;            // a tile's rows are reached by 32-bit offsets
constexpr long long kFp8MaxRows = 1LL << 24;
constexpr size_t kFp8ScratchBytes = (size_t)128 << 20;  // a context's: rows, in bfloat16
constexpr size_t kFp8ChangesBytes = (size_t)8 << 20;    // and a weight's scales, as tiles take them
constexpr int kFp8RowStep = 256;                  // rows that a tile takes at most
constexpr int kFp8MaxSplits = 16;                 // parts of a sum
constexpr long long kFp8PartFloats = 4LL << 20;   // all parts' sums
constexpr int kFewRows = 4;                       // that a block may hold by themselves, not 16 at once

static_assert(kFp8ChangesBytes >= (size_t)(kFp8MaxSide / kFp8Block) * (kFp8MaxSide / kFp8Block) * 8, "all blocks");

inline int fp8_blocks(int k) { return (k + kFp8Block - 1) / kFp8Block; }

// Rows that the scratch holds at once, a multiple of kFp8RowStep: a product of
// more goes over them in turn.
inline int fp8_rows_at_once(int k) {
    const size_t each = (size_t)fp8_blocks(k) * kFp8Block * 2;
    return (int)(kFp8ScratchBytes / each / kFp8RowStep) * kFp8RowStep;
}

inline Refusal check_fp8_weight(const qtts_fp8_weight &w) {
    if (w.n < 1 || w.k < 16 || w.k % 16 != 0 || w.n > kFp8MaxSide || w.k > kFp8MaxSide)
        return {QTTS_ESHAPE, "fp8 weight: n and k must be 1..131072, k a multiple of 16"};
    if (w.ld < w.k) return {QTTS_ESHAPE, "fp8 weight: a row stride below the row"};
    if (w.ld > kFp8MaxStride) return {QTTS_ERANGE, "fp8 weight: a row stride above 2^23"};
    if (w.ld % 16 != 0) return {QTTS_EINVAL, "fp8 weight: the row stride must be a multiple of 16"};
    if (!w.codes || !w.scales) return {QTTS_EINVAL, "fp8 weight: null buffer"};
    if (!aligned_to(w.codes, 16) || !aligned_to(w.scales, 4))
        return {QTTS_EINVAL, "fp8 weight: codes must be 16-byte aligned"};
    return kAccepted;
}

inline Refusal check_fp8_gemm(const qtts_fp8_weight &w, const float *x, int32_t ld_x, int32_t rows, const float *add,
                              int32_t ld_add, const float *y, int32_t ld_y) {
    QTTS_REFUSE(check_fp8_weight(w));
    if (rows < 0 || rows > kFp8MaxRows) return {QTTS_ESHAPE, "fp8 product: rows must be 0..2^24"};
    if (rows == 0) return kAccepted;
    QTTS_REFUSE(check_rows(x, ld_x, w.k));
    QTTS_REFUSE(check_rows(y, ld_y, w.n));
    if (x == y) return {QTTS_EINVAL, "fp8 product: y must not be x"};
    if (add) {
        QTTS_REFUSE(check_rows(add, ld_add, w.n));
        if (add == y && ld_add != ld_y) return {QTTS_EINVAL, "fp8 product: in place, add takes y's stride"};
    }
    return kAccepted;
}

inline Refusal check_fp8_quantize(const float *src, int32_t ld_src, const qtts_fp8_weight &w) {
    QTTS_REFUSE(check_fp8_weight(w));
    return check_rows(src, ld_src, w.k);
}

// A product's tiles: bn columns of the output (rows of the weight) by bm rows.  The
// first `whole` have a block each; the blocks of 128 of the contraction of the others
// are divided over `splits` blocks, `each` of them each.
struct Fp8Plan {
    int bn, bm;  // bn == 16: the kernel without tiles in LDS, 16, 32 or 64 rows a block
    int tiles_n, tiles_m, whole, splits, each;
    long long ns;  // what it is taken to cost
    int waves;     // of a block of that kernel
};
inline long long fp8_launched(const Fp8Plan &p) {
    return p.whole + ((long long)p.tiles_n * p.tiles_m - p.whole) * p.splits;
}

// A tile's step of 64, in ns: with a CU to itself and where blocks fill it, as measured
// (4096 deep, 64 to 4096 blocks).
struct Fp8Tile {
    int bn, bm, alone, full;
};
constexpr Fp8Tile kFp8Tiles[] = {{256, 256, 1600, 1850}, {128, 128, 570, 520}, {64, 64, 310, 205}};

// Whether that kernel brings x to 8 bits itself, in each block anew, for a launch less: up
// to four rows while they fit 64 KB of LDS, more while a CU's blocks of 16 rows have no
// more than 128 times 128 values to bring over (us so and with a launch for it: 8 rows of
// 2048 -> 4096 6.7 and 6.8, 8 of 1024 -> 8000 6.2 and 7.0, but 16 of these 8.3 and 6.7, 8
// of 2048 -> 12288 12.4 and 10.1; one of 6144 -> 2048 7.9 and 10.1).
inline bool fp8_own_rows(int rows, int n, int kb) {
    if (rows <= kFewRows) return rows * kb <= 256;
    const long long blocks = (n + 15) / 16 * ((rows + 15) / 16LL);
    return (rows < 16 ? rows : 16) * kb * ((blocks + 255) / 256) <= 128;
}
inline long long fp8_own_bytes(int rows, int kb) { return (rows <= kFewRows ? rows : 16LL) * kb * 256; }

// The unit that a tile's sums are held in under a block's scale: the scale without its
// power of two, 1 to 2 with its sign; 1 where the codes do not hold that power (under
// 2^-117 or over 2^117, 0, Inf, NaN).
QTTS_HD bool fp8_held(unsigned scale) { return (scale >> 23 & 255) - 10 <= 234; }
QTTS_HD unsigned fp8_unit(unsigned scale) { return fp8_held(scale) ? (scale & 0x807fffffu) | 0x3f800000u : 0x3f800000u; }

// A block's power of two, which its codes take, for an instruction that uses only the
// exponent; below it what a tile has to know of the block.
constexpr int kFp8None = 1, kFp8Bad = 2, kFp8Far = 4;  // zeros in the steps; Inf or NaN; added behind them
QTTS_HD unsigned fp8_power(unsigned scale) {
    const unsigned e = scale & 0x7f800000u;
    if (fp8_held(scale)) return e;
    return e == 0x7f800000u ? e | kFp8Bad : e | kFp8None | (scale << 1 ? kFp8Far : 0);
}

// From one unit to another: the quotient, rounded, as bits; what the rounding leaves of
// it, and half of the quotient's last place, both in 2^-48 of it.  Of the reciprocals a
// step or two may be wrong.
struct Fp8Change {
    int quotient, left, half;
};
QTTS_HD Fp8Change fp8_change(float from, float to, float from_inverse, float to_inverse) {
    const float near = from * to_inverse, q = fmaf(fmaf(-near, to, from), to_inverse, near), size = fabsf(q);
    union {
        float f;
        int i;
    } bits{q};
    const float half = (size < 1.0f ? 0x1p23f : 0x1p24f) * fabsf(to * from_inverse);
    return {bits.i, (int)(fmaf(-q, to, from) * from_inverse * 0x1p48f), size == 1.0f ? 1 << 29 : (int)half};
}
// What the roundings of the quotients before have left is carried on; once it is half a
// place, the quotient's neighbour is taken in its place.  The factors' product then is
// never further than 2^-24 from the units' quotient, however often these change, and
// equal units change nothing.
QTTS_HD int fp8_step(const Fp8Change &c, int carried) {  // from the quotient to the factor
    const int all = carried + c.left;
    return all > c.half ? 1 : all < -c.half ? -1 : 0;
}
QTTS_HD int fp8_carry(const Fp8Change &c, int carried) {  // on to the next change
    const int all = carried + c.left, place = 2 * c.half;
    return all - (all > c.half ? place : all < -c.half ? -place : 0);
}
// Whether a quotient can go on by one more place of the same size: away from 1, where
// places change theirs.
QTTS_HD bool fp8_apart(int quotient) { return (unsigned)(quotient & 0x7fffffff) - 0x3f7fffffu > 2; }

// Whether a call uses the scratch.  (One of more rows than that holds does.)
inline bool fp8_scratch(int rows, int n, int k) {
    return rows > fp8_rows_at_once(k) || !fp8_own_rows(rows, n, fp8_blocks(k));
}

inline Fp8Plan fp8_divided(int rows, int n, int k, int bn, int bm, int splits) {
    const int kb = fp8_blocks(k);
    Fp8Plan p{bn, bm, (n + bn - 1) / bn, (rows + bm - 1) / bm, 0, 1, 0, 0, 0};
    p.each = (kb + splits - 1) / splits;
    p.splits = (kb + p.each - 1) / p.each;
    p.each = (kb + p.splits - 1) / p.splits;
    return p;
}

// The tile and division that are taken to cost least: no tile divided, all of them, or
// those past the last whole round of 256.  A block's start and end cost some 3 us;
// the fullest CU works off its blocks; joining costs a launch and the parts' way to memory and back.
// Against all that can be chosen, 1 % more over 26 shapes (17 to 8192 rows), 8 % at
// worst.  us, the chosen one with a star, tiles of 256, 128 and 64 whole and the last
// round divided in 128 and in 64: 512 x 1552 -> 1001 22, 13, 9.9*; 900 x 2048 -> 4096 57,
// 24.3*, 26.1; 1064 rows of it 54, 34, 33, 29*, 30; 2112 rows 58, 57, 51, 44*, 50;
// 4096 rows 63.9*, 66.1, 83.6; 2100 x 6144 -> 2048 132, 85, 82, 62*, 72; 8192 x 2048 ->
// 12288 362*, 410, -.  128 x 6144 -> 2048 in 64: 14 in four parts, 37 in one.
//
// Where the reads that every block repeats cost less, the kernel without tiles, in as
// many rows a block as cost least (kernels' times, both sides of one session): 32 rows
// of 2048 -> 4096 4.9 us (in tiles 8.4), 64 7.0 (9.2); 128 of 2048 -> 2048 6.7 (9.2);
// 333 of 1552 -> 1001 7.8 (10.1); 230 of 3248 -> 150 3.9 (7.7); but 200 of 6144 ->
// 2048 29 (17*).  Over 110 drawn shapes 4 % more than the best of all that can be
// chosen.
inline Fp8Plan fp8_plan(int rows, int n, int k) {
    const int kb = fp8_blocks(k);
    Fp8Plan best{};
    for (int side = 16; side <= 64; side *= 2) {
        Fp8Plan p = fp8_divided(rows, n, k, 16, side, 1);
        p.waves = 8;
        if (fp8_own_rows(rows, n, kb)) {
            // more waves for a long row where they do not stand in another block's way (one
            // row of 6144 -> 2048 7.9 us, 8.5 with four; -> 12288 20.7 and 17.5)
            p.waves = p.tiles_n > 256 || kb <= 16 ? 4 : 8;
            return p;
        }
        // what a block reads of x in bfloat16 and of codes
        const long long reads = 16LL * k * (2 * side / 16 + 1), blocks = (long long)p.tiles_n * p.tiles_m;
        p.ns = 2200 + (blocks + 255) / 256 * (200 + reads * 13 / 1000);
        if (blocks <= (1 << 22) && (best.bn == 0 || p.ns < best.ns)) best = p;
    }
    for (const Fp8Tile &t : kFp8Tiles)
        for (int splits = 1; splits <= kFp8MaxSplits && splits <= kb; splits++) {
            Fp8Plan p = fp8_divided(rows, n, k, t.bn, t.bm, splits);
            if (p.splits != splits) continue;
            const long long tiles = (long long)p.tiles_n * p.tiles_m, rounds = splits > 1 ? tiles / 256 : 0;
            for (long long round : {0LL, rounds}) {
                p.whole = (int)(256 * round);
                const long long rest = tiles - p.whole, pieces = rest * splits, floats = pieces * t.bn * t.bm;
                if (splits > 1 && (rest == 0 || floats > kFp8PartFloats)) continue;
                if (fp8_launched(p) > (1 << 22)) continue;  // a launch counts its threads in 32 bits
                const long long most = (pieces + 255) / 256, step = 2LL * p.each, all = 2LL * kb;
                long long work = most * step * t.full;
                if (round) work = round * all * t.full + (most == 1 ? step * t.alone : work);
                const long long alone = (round ? all : step) * t.alone;
                p.ns = 3000 + (work > alone ? work : alone);
                // (the last tiles' rows may be few)
                const long long low = rest < p.tiles_n ? rest : p.tiles_n, few = (long long)p.tiles_m * t.bm - rows;
                if (splits > 1) p.ns += 3500 + (floats - low * few * splits * t.bn) * 8 / 4000;
                if (best.bn == 0 || p.ns < best.ns) best = p;
            }
        }
    return best;
}

}  // namespace qtts
