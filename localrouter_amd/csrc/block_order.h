// The order in which an XCD's blocks of rows start (attn_cache_wide.hip). Plain C++: the host's tests run it too.
#pragma once

namespace lr {

// The block, longest first, that workgroup `idx` of an XCD's `local` takes, `per_cu` of them resident on each of its 32 CUs. Of two
// a CU, workgroups 32 apart share one: where all are resident at once, the second 32 go in the opposite order, the shortest beside
// the longest. Elsewhere longest first throughout: of one a CU, the one that ends last would else be given the longest of the rest
// (8 waves, 64 blocks an XCD, with the second 32 reversed / longest first: 4,096 causal tokens x 32 heads over 8 173 / 150 us over
// pages, 157 / 138 over rows, behind 4,096 more 412 / 377 and 384 / 357; 2 x 2,048 behind 2,048 238 / 207).
constexpr int start_order(int idx, int local, int per_cu) {
    return per_cu == 2 && local <= 64 && idx >= 32 ? local + 31 - idx : idx;
}

}  // namespace lr
