// fp8_plan.h — what decides which memory the products on 8-bit floats touch: the
// checks of a call's arguments and how its work is divided.  Plain C++ without
// device code, so that the CPU tests run the same lines.
#pragma once

#include <cstdint>

#include "../../include/qtts.h"
#include "paged_plan.h"

namespace qtts {

constexpr int kFp8Block = 128;                    // side of a weight's block, length of a row's
constexpr int kFp8MaxSide = 1 << 17;              // of n and k
constexpr long long kFp8MaxRows = 1LL << 24;
constexpr size_t kFp8ScratchBytes = (size_t)64 << 20;  // a context's: rows, in bfloat16
constexpr int kFp8RowStep = 256;                  // rows that a tile takes at most
constexpr long long kFp8PartFloats = 4LL << 20;   // split sums
constexpr int kFp8MaxSplits = 64;
constexpr int kFp8Counters = 8192;                // a tile's, zero between launches

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

// A product's tiles: BN columns of the output (rows of the weight) by BM rows,
// blocks of 128 of the contraction divided over `splits` blocks of a tile.
struct Fp8Plan {
    int bn, bm;     // bm <= 16: the kernel for few rows
    int tiles_n, tiles_m, splits;
};

inline Fp8Plan fp8_plan(int rows, int n, int k) {
    const int kb = fp8_blocks(k);
    Fp8Plan p;
    p.bn = rows <= 16 ? 32 : 256;
    p.bm = rows <= 16 ? 16 : 128;
    p.tiles_n = (n + p.bn - 1) / p.bn;
    p.tiles_m = (rows + p.bm - 1) / p.bm;
    p.splits = 1;
    const long long tiles = (long long)p.tiles_n * p.tiles_m;
    const int least = rows <= 16 ? 4 : 2;  // blocks of a split at least
    long long want = 512 / tiles;
    if (want > kb / least) want = kb / least;
    if (want > kFp8MaxSplits) want = kFp8MaxSplits;
    while (want > 1 && (tiles > kFp8Counters || tiles * want * p.bn * p.bm > kFp8PartFloats)) want--;
    if (want > 1) {
        const int each = (int)((kb + want - 1) / want);
        p.splits = (kb + each - 1) / each;
    }
    return p;
}

}  // namespace qtts
