// Argument checks shared by the entry points of the C ABI (lr_abi.hip, cache_abi.hip).
#pragma once
#include <math.h>
#include <stdint.h>

#include "../../include/lr_attn.h"
#include "lr_common.h"

namespace lr {
namespace abi {

constexpr int ERR_ARGS = (int)hipErrorInvalidValue;

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// A bf16 rows tensor: 16-byte aligned base, row stride a multiple of 8 elements and wide enough for its heads.
inline bool rows_ok(const void* p, int64_t rs, int heads) {
    return p && aligned(p, 16) && rs % 8 == 0 && rs >= (int64_t)heads * lr::D;
}

inline bool scale_ok(float s) { return s > 0.0f && isfinite(s); }

// Table checks shared by the rope entry points. rows_needed: table rows that will be read.
inline bool table_ok(int kind, const void* ta, const void* tb, int64_t stride, int rot, int pairing, int split_mod) {
    if (kind == LR_TABLE_NONE) return true;
    if (kind < LR_TABLE_NONE || kind > LR_TABLE_MAT2_F32) return false;
    if (rot <= 0 || rot > lr::D || rot % 2) return false;
    if (pairing != LR_PAIR_INTERLEAVED && pairing != LR_PAIR_SPLIT_HALF) return false;
    if (pairing == LR_PAIR_SPLIT_HALF && rot % split_mod) return false;
    if (!ta || stride < 0) return false;
    const int pairs = rot / 2;
    if (kind == LR_TABLE_COSSIN_F32) return tb && aligned(ta, 4) && aligned(tb, 4) && stride >= pairs;
    if (kind == LR_TABLE_MAT2_BF16) return aligned(ta, 8) && stride % 4 == 0 && stride >= 4 * pairs;
    return aligned(ta, 16) && stride % 4 == 0 && stride >= 4 * pairs;  // LR_TABLE_MAT2_F32
}

// cos / sin tables whose rows are 16-byte aligned are read as 16-byte chunks
inline int tab_vec(int kind, const void* ta, const void* tb, int64_t stride) {
    return kind == LR_TABLE_COSSIN_F32 && aligned(ta, 16) && aligned(tb, 16) && stride % 4 == 0;
}

// byte range [lo, hi) of a rows tensor: rows rows of heads heads, row stride rs elements
struct Span {
    uintptr_t lo, hi;
};
inline Span rows_span(const void* p, int64_t rows, int64_t rs, int heads) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return Span{lo, lo + (uintptr_t)(((rows - 1) * rs + (int64_t)heads * lr::D) * 2)};
}
inline bool overlap(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

}  // namespace abi
}  // namespace lr
