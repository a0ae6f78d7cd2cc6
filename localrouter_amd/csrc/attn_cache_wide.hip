// The ranged attention (attn_cache.hip) of calls with many rows of a kv head: chunks, frames and large trees, where the matrix
// products bound it, over rows, pages and pages of 8 bits. The same contract; the loop is that of the key-split kernel
// (attn_keysplit.hip): a half-step of 16 MFMA slots runs the next half-tile's scores, the previous one's products and this one's exponentials. A workgroup is 128 rows
// (tokens x the query heads of one kv head), four waves of 32 rows over a ring of two key tiles and two value tiles; two
// workgroups share a CU, one's start, end and waits under the other's products. Long calls that fill the CUs take 256 rows, eight
// waves and four of each tile. What bounds them is the clock under the power limit: 16,384 tokens x 32 heads over windows of four
// frames of 1,024 run at 1,034 to 1,135 TFLOP/s; under the profiler at 1.79 GHz, MFMA busy 52 % of the call. What differs from the
// key-split kernel:
//
//  * The tiles are a list (the first tokens' tiles, then the rows' own range), and a half-tile that some row of the wave does
//    not see whole takes a masked step: its 32 keys' visibility as one word a row, built from the row's limits (and its tree
//    bits), two instructions a score to apply.
//  * A row's softmax reference is the maximum of the first half-tile in which it sees a key, which a window's list does not
//    put first for every row: until each row of the wave has one, half-tiles take the masked step, which also sets references.
//  * Pages hold at least 16 rows, so the 16 rows of a value load are in one page, and the 32 rows of a key load in at most
//    two: scalar bases from the staged page-table entries.
//  * A row that overflowed its reference, or met an infinity or NaN, is computed again over the keys that it sees.
//  * Pages of 8 bits: the tiles go through registers, loaded a step ahead, and are converted on their way into LDS, once for all the
//    workgroup's rows (in the products' place each wave would convert every fragment): 16 conversions and 4 LDS writes a wave and
//    step beside 32 MFMA, twice as many in workgroups of four waves. 2,048 tokens x 32 heads over 8 behind 6,000 positions 268 us, over
//    bf16 pages 249.
#include "lr_common.h"
#include "block_order.h"
#include "lr_cache_kernels.h"
#include "tile_image.h"

namespace lr {

namespace {

#include "attn_common.inc"

constexpr int RA = 3;             // fragments read ahead
constexpr int FR = 4;             // fragment ring entries
static_assert(IMG_TILE_KEYS == RANGE_WIDE_TILE, "the host's cut");

#include "attn_tiles.inc"
#include "raise_rows.inc"
#include "dma1.inc"
#include "range_attn.inc"

// The sequence of rank `rank` when the batch is ordered longest first (B <= 64), so that the last workgroups to start are
// short ones.
__device__ __forceinline__ int seq_by_length(const RangeAttnArgs& a, int rank) {
    const int lane = threadIdx.x & 63;
    const int len = lane < a.B ? a.lens[lane] : INT32_MIN;
    int before = 0;
    for (int j = 0; j < a.B; ++j) {
        const int other = __builtin_amdgcn_readlane(len, j);
        before += other > len || (other == len && j < lane);
    }
    return __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < a.B && before == rank));
}

// The block of rows of workgroup `id`, its part (0 <= split < nsplit) and its number among the blocks that are cut (-1: whole).
// Hardware workgroup id runs on XCD id % 8; with by_xcd `idx` is its number there, else it is id. Rows, by_xcd: an XCD works on
// whole heads, one after the other (the blocks of a head share its keys in the XCD's L2), the last blocks of a head first:
// without a full window they are the longest; otherwise the heads alternate. Pages: longest sequences first, the blocks of one
// sequence and head next to each other, by_xcd on one XCD (in the order of
// block_order.h). The first `whole` blocks (of an XCD, or of the launch) are not cut.
template <int QW, int SRC>
__device__ __forceinline__ bool block_of(const RangeAttnArgs& a, int id, int& b, int& hk, int& blk, int& split, int& cut) {
    constexpr bool PAGED = paged(SRC);
    const int xcd = a.by_xcd ? id & 7 : 0;
    int idx = a.by_xcd ? id >> 3 : id;
    if (a.by_xcd && a.nsplit == 1) idx = start_order(idx, a.local, 8 / QW);
    split = 0;
    cut = -1;
    if (a.nsplit > 1 && idx >= a.whole) {
        const int at = idx - a.whole, q = div_small(at, a.nsplit, a.rcp_split);
        split = at - q * a.nsplit;
        idx = a.whole + q;
        cut = xcd * (a.local - a.whole) + q;
    }
    b = 0;
    if (PAGED || a.by_xcd) {
        int pair = div_small(idx, a.nblk, a.rcp_nblk);
        blk = a.nblk - 1 - (idx - pair * a.nblk);
        if (PAGED) {
            if (a.by_xcd) pair = pair * 8 + xcd;
            if (pair >= a.B * a.HK) return false;
            b = div_small(pair, a.HK, a.rcp_hk);
            hk = pair - b * a.HK;
            if (a.B > 1 && a.B <= 64) b = seq_by_length(a, b);
        } else {
            hk = pair + xcd * (a.HK / 8);
        }
    } else {
        const int at = div_small(idx, a.HK, a.rcp_hk);
        hk = idx - at * a.HK;
        blk = a.nblk - 1 - at;
    }
    return true;
}

// The keys of a batch in pieces of equal length (a.teams). Sequences of one launch end when the longest does; here the pairs (sequence,
// kv head) of an XCD lie end to end and are cut every Q tiles, so that each place has Q tiles of work whatever the lengths, and the
// row blocks of a pair, next to each other, read the same keys at the same time (apart, each would read them from HBM). Lane j < P:
// the piece that starts with pair j; lane P + t - 1: the one that starts at the cut t Q inside a pair. Pieces go out longest first:
// a place whose piece was short takes the longest of the rest.
struct Pieces {
    int P, tiles, end, Q;   // pairs an XCD; lane j's pair: its tiles, and where it ends
    int j, x0, x1;          // lane's piece: its pair, its tiles (none: x0 == x1)

    template <int KBM>
    __device__ __forceinline__ void init(const RangeAttnArgs& a, int xcd) {
        const int lane = threadIdx.x & 63;
        P = a.B * a.HK >> 3;
        const int pair = min(lane, P - 1) * 8 + xcd;
        const Seq sq = seq_of<PAGES>(a, div_small(pair, a.HK, a.rcp_hk));
        const int rows = max(sq.n, 0) * a.G;
        tiles = lane < P && rows > 0 ? max(1, (sq.end + IMG_TILE_KEYS - 1) / IMG_TILE_KEYS) : 0;
        end = tiles;
        int work = tiles * ((rows + KBM - 1) / KBM);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(end, d, 64), y = __shfl_xor(work, d, 64);
            end += lane >= d ? x : 0;
            work += y;
        }
        const int all = __builtin_amdgcn_readlane(end, 63);
        work = __builtin_amdgcn_readfirstlane(work);
        const int teams = work > 0 ? min(a.teams, max(1, (a.places * all + work / 2) / work)) : 1;
        Q = max(16, (all + teams - 1) / teams);   // (shorter pieces cost more than they spread)
        const int pos = (lane - P + 1) * Q;
        int at = 0;   // pairs that end at or before this lane's cut
        for (int k = 0; k < P; ++k) at += __builtin_amdgcn_readlane(end, k) <= pos;
        j = lane < P ? lane : min(at, P - 1);
        const int e = __shfl(end, j, 64), s = e - __shfl(tiles, j, 64);
        const int first = lane < P ? s : pos, last = min(e, lane < P ? (s / Q + 1) * Q : pos + Q);
        const bool is = lane < P ? tiles > 0 : pos < all && s < pos;
        x0 = is ? first - s : 0;
        x1 = is ? last - s : 0;
    }
    // the piece of rank r: its lane, or -1
    __device__ __forceinline__ int rank(int r) const {
        const int lane = threadIdx.x & 63, len = x1 - x0;
        int before = 0;
        for (int k = 0; k < 64; ++k) {
            const int other = __builtin_amdgcn_readlane(len, k);
            before += other > len || (other == len && k < lane);
        }
        const uint64_t m = __builtin_amdgcn_ballot_w64(before == r && len > 0);
        return m ? __builtin_ctzll(m) : -1;
    }
};

// Blocks of 8-bit pages in equal shares (a.places without a.teams): the blocks of an XCD's pairs, each counted as its sequence's tiles,
// lie end to end and are cut every Q tiles, so that each place has Q tiles of work however many blocks there are. Number x < PLACES: the
// piece that starts at the cut x Q; PLACES + m: the one that starts with block m, unless a cut is there (m < 128: the host checks it).
// Longest first, as Pieces.
struct BlockPieces {
    static constexpr int KBM = 256, PLACES = RANGE_WIDE_PLACES, E = 3;   // pieces a lane
    int P, tiles, blocks, end, last, Q;        // pairs an XCD; lane j's pair: a block's tiles, its blocks, where tiles and blocks end
    int pos[E], len[E];

    __device__ __forceinline__ void init(const RangeAttnArgs& a, int xcd) {
        const int lane = threadIdx.x & 63;
        P = a.B * a.HK >> 3;
        const Seq sq = seq_of<PAGES8>(a, div_small(min(lane, P - 1) * 8 + xcd, a.HK, a.rcp_hk));
        const int rows = lane < P ? max(sq.n, 0) * a.G : 0;
        tiles = max(1, (sq.end + IMG_TILE_KEYS - 1) / IMG_TILE_KEYS);
        blocks = (rows + KBM - 1) / KBM;
        end = tiles * blocks;   // (the host checks that all of them fit)
        last = blocks;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(end, d, 64), y = __shfl_up(last, d, 64);
            end += lane >= d ? x : 0;
            last += lane >= d ? y : 0;
        }
        Q = max(16, (__builtin_amdgcn_readlane(end, 63) + PLACES - 1) / PLACES);   // (shorter pieces cost more than they spread)
    }
    // pair j's block number nth, from the one with the most keys on: where it begins
    __device__ __forceinline__ int begin(int j, int nth) const {
        return __builtin_amdgcn_readlane(end, j) - (__builtin_amdgcn_readlane(blocks, j) - nth) * __builtin_amdgcn_readlane(tiles, j);
    }
    __device__ __forceinline__ void cut() {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int at = i == 0 ? lane * Q : (i - 1) * 64 + lane;
            int j = 0;
            for (int k = 0; k < P; ++k) j += __builtin_amdgcn_readlane(i == 0 ? end : last, k) <= at;
            const bool is = j < P;
            j = min(j, P - 1);
            const int n = __shfl(tiles, j, 64), all = __shfl(blocks, j, 64), e = __shfl(end, j, 64);
            const int nth = i == 0 ? all - (e - at + n - 1) / n : all - (__shfl(last, j, 64) - at), from = e - (all - nth) * n;
            pos[i] = i == 0 ? at : from;
            len[i] = is && (i == 0 || from % Q != 0) ? min(from + n, (pos[i] / Q + 1) * Q) - pos[i] : 0;
        }
    }
    // the piece of rank r: its number and where it starts and ends
    __device__ __forceinline__ bool rank(int r, int& x, int& p0, int& p1) const {
        const int lane = threadIdx.x & 63;
        int key[E], found = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) key[i] = len[i] > 0 ? len[i] << 8 | (255 - i * 64 - lane) : 0;
        for (int bit = 1 << 24; bit; bit >>= 1) {   // the greatest value that more than r of them reach
            int n = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(key[i] >= (found | bit)));
            found |= n > r ? bit : 0;
        }
        if (found == 0) return false;
        x = 255 - (found & 255);
        p0 = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int at = __builtin_amdgcn_readlane(pos[i], x & 63);
            p0 = x >> 6 == i ? at : p0;
        }
        x = x < 64 ? x : PLACES + x - 64;   // (a lane's first entry holds a cut, the others blocks)
        p1 = p0 + (found >> 8);
        return true;
    }
    // the pair and the block in which tile p0 lies
    __device__ __forceinline__ void block(int p0, int& j, int& nth) const {
        j = __popcll(__builtin_amdgcn_ballot_w64(end <= p0));
        const int n = __builtin_amdgcn_readlane(tiles, j);
        nth = __builtin_amdgcn_readlane(blocks, j) - (__builtin_amdgcn_readlane(end, j) - p0 + n - 1) / n;
    }
};

template <int QW, int SRC>
__global__ __launch_bounds__(64 * QW, 8 / QW) __attribute__((amdgpu_waves_per_eu(2, 2))) void range_wide_kernel(RangeAttnArgs a) {
    constexpr int KBM = 32 * QW;                        // rows per block
    constexpr bool PAGED = paged(SRC);
    // steps of refills in flight beside the current one's. (8 waves have the LDS for 2: pages come from HBM, ~2 us away under load: 16
    // trees of up to 64 tokens over up to 30,000 keys 860 -> 841 us. Rows come from the L2s: 16,384 tokens of video 1,171 us with 2,
    // 1,164 with 0.)
    constexpr int E = QW == 8 && SRC == PAGES ? 2 : 0;
    constexpr int LP = 16 / QW;                         // direct loads of a tile per wave
    // loads in flight at a step's end, when the next step's keys and this one's values have landed; with E > 0 a step early, so that
    // the next step's first key fragments are read before the barrier (the trees 811 -> 798 us)
    constexpr int AHEAD = E > 0 ? (E - 1) * 2 * LP : 0;
    constexpr int SLOTS = 2 + E;                        // key tiles and value tiles
    constexpr int RING_LDS = 2 * SLOTS * IMG_TILE_BYTES;
    static_assert(8 / QW * (RING_LDS + 4 * RANGE_WIDE_STAGED + 256) <= 160 * 1024, "8 waves a CU");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[RING_LDS];
    __shared__ int staged[PAGED ? RANGE_WIDE_STAGED : 1];
    constexpr int BT = IMG_TILE_KEYS;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, hf = lane >> 5;

    int b, hk, blk, split, cut, px0 = 0, px1 = 0;   // (px1: of a piece)
    if (SRC == PAGES8 && QW == 8 && a.places && !a.teams) {
        const int xcd = blockIdx.x & 7;
        BlockPieces pc;
        pc.init(a, xcd);
        pc.cut();
        int x, p0, p1, j, nth;
        if (!pc.rank(blockIdx.x >> 3, x, p0, p1)) return;
        pc.block(p0, j, nth);
        const int pair = 8 * j + xcd, from = pc.begin(j, nth);
        px0 = p0 - from;
        px1 = p1 - from;
        b = div_small(pair, a.HK, a.rcp_hk);
        hk = pair - b * a.HK;
        blk = __builtin_amdgcn_readlane(pc.blocks, j) - 1 - nth;
        split = 0;
        cut = px1 - px0 == __builtin_amdgcn_readlane(pc.tiles, j) ? -1 : xcd * (BlockPieces::PLACES + pc.P * a.nblk) + x;
    } else if (PAGED && a.teams) {
        const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3, r = div_small(idx, a.nblk, a.rcp_nblk);
        Pieces pc;
        pc.template init<KBM>(a, xcd);
        const int at = pc.rank(r);
        if (at < 0) return;
        const int j = __builtin_amdgcn_readlane(pc.j, at), pair = 8 * j + xcd;
        px0 = __builtin_amdgcn_readlane(pc.x0, at);
        px1 = __builtin_amdgcn_readlane(pc.x1, at);
        b = div_small(pair, a.HK, a.rcp_hk);
        hk = pair - b * a.HK;
        blk = a.nblk - 1 - (idx - r * a.nblk);
        split = 0;
        const bool all = px1 - px0 == __builtin_amdgcn_readlane(pc.tiles, j);
        cut = all ? -1 : (xcd * (pc.P + a.teams) + at) * a.nblk + blk;
    } else if (!block_of<QW, SRC>(a, blockIdx.x, b, hk, blk, split, cut)) {
        return;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    hk = __builtin_amdgcn_readfirstlane(hk);
    blk = __builtin_amdgcn_readfirstlane(blk);
    const Seq sq = seq_of<SRC>(a, b);
    const int row0 = blk * KBM;
    const int rows = max(sq.n, 0) * a.G;   // (at most 2^30: the host checks)
    if (row0 >= rows) return;
    TileList<BT, SRC> tl;
    tl.init(a, sq, div_small(row0, a.G, a.rcp_g), div_small(min(rows, row0 + KBM) - 1, a.G, a.rcp_g));
    if (PAGED && (SRC == PAGES8 ? px1 : a.teams) > 0) {
        tl.x0 = px0;
        tl.x1 = min(tl.total, px1);
    } else if (PAGED || cut >= 0) tl.part(split, a.per ? a.per : div_small(tl.total + a.nsplit - 1, a.nsplit, a.rcp_split));
    const bool bad = tl.template stage<64 * QW>(a, b, staged);
    const int x0 = __builtin_amdgcn_readfirstlane(tl.x0), x1 = __builtin_amdgcn_readfirstlane(tl.x1);

    // ---- this lane's row
    const int r = row0 + 32 * wv + n, rr = min(r, rows - 1);
    const bool live = r < rows;
    const int i = div_small(rr, a.G, a.rcp_g), head = hk * a.G + rr - i * a.G;
    const Sees me = sees_of<SRC>(a, sq, i);
    const int64_t part = (int64_t)cut * a.nsplit + split;   // its slot among the parts (merge_rows)
    if (x0 >= x1) {   // nothing to see in this part
        if (live) {
            if (cut >= 0) {
                a.part_ml[2 * (part * KBM + 32 * wv + n) + hf] = hf ? 0.0f : -INFINITY;
            } else {
                uint16_t* dst = a.out + (int64_t)(sq.t0 + i) * a.o_rs + head * D + 64 * hf;
#pragma unroll
                for (int e = 0; e < 8; ++e) *reinterpret_cast<u32x4*>(dst + 8 * e) = u32x4{0, 0, 0, 0};
            }
        }
        return;
    }
    // half-tiles (h = 2 x + half) that every row of the wave sees whole need no mask: h < free_s among the first tokens',
    // free_lo <= h < free_hi of the rows' own range
    int free_s = 0, free_lo = 0, free_hi = 0;
    if (!bad) {
        const int hi_all = __builtin_amdgcn_readfirstlane(PAGED && a.tree ? max(0, min(sq.p0, sq.end)) : wave_min_i(me.hi));
        const int lo_all = __builtin_amdgcn_readfirstlane(wave_max_i(me.lo)), skip = 2 * (tl.lt - tl.st);
        free_s = min(2 * tl.st, min(a.sinks, hi_all) / 32);
        free_lo = max(2 * tl.st, (lo_all + 31) / 32 - skip);
        free_hi = hi_all / 32 - skip;
    }
    const int nsteps = x1 - x0;

    // ---- direct loads: a tile is four 1 KB loads of each wave. Load u of a key tile: fragment 4 wv + u (key
    // block wv >> 1, k-step 4 (wv & 1) + u), lane 32 hf + n row img_key_perm(n) of the block. Load u of a value tile: rows
    // 16 wv + 4 u + vt_lane_row(lane) in the row-block layout (attn_tiles.inc). Rows past the last key read that one.
    const int64_t k_rs = PAGED ? a.pg.rs : a.k_rs, v_rs = PAGED ? a.pg.rs : a.v_rs;
    const int64_t hoff = (int64_t)hk * (PAGED ? a.pg.hs : D);
    const uint64_t khead = (uint64_t)(uintptr_t)(a.k + hoff), vhead = (uint64_t)(uintptr_t)(a.v + hoff);
    const uint32_t krowb = (uint32_t)k_rs * 2u, rowb = (uint32_t)v_rs * 2u;   // (below 2^24: the host checks)
    const uint32_t ring = lds_addr(lds), vring = ring + SLOTS * IMG_TILE_BYTES;
    const uint32_t lane16 = (uint32_t)lane * 16u;
    const uint32_t krow = (uint32_t)img_key_perm(n), kcol = (uint32_t)(32 * LP * (wv % (QW / 2)) + 16 * hf);
    const uint32_t vrow = (uint32_t)(vt_lane_row(lane) + 4 * LP * wv % 16), vchunk = (uint32_t)(16 * vt_lane_chunk(lane));
    auto tile_of = [&](int u) __attribute__((always_inline)) { return min(x0 + u, x1 - 1); };
    // the first of the `run` rows of tile x from its row g on (16: a page's least), clamped to the last run that exists
    auto first = [&](int x, int g, int run) __attribute__((always_inline)) { return min(tl.key0(x) + g, (tl.end - 1) & -run); };
    auto page = [&](int x, int g, int run) __attribute__((always_inline)) {
        return PAGED ? tl.entry(x, first(x, g, run) - tl.key0(x)) : 0;
    };
    // its base, given its page, and the last row of it that exists
    auto base_of = [&](int x, int g, int run, int64_t rs, int entry, int& last) __attribute__((always_inline)) {
        const int j = first(x, g, run);
        last = min(run, tl.end - j) - 1;
        if constexpr (PAGED)
            return (uint64_t)(((int64_t)__builtin_amdgcn_readfirstlane(max(entry, 0)) * a.pg.ps +
                               (int64_t)(j & ((1 << tl.shift) - 1)) * rs) * 2);
        return (uint64_t)((int64_t)j * rs * 2);
    };
    // the page-table entries of the next refills, read a half-step ahead (read where they are used, each kept the wave's
    // products waiting for LDS)
    int ev = 0, ek = 0, ek1 = 0;
    const int vg = 16 * (4 * wv / QW), kg = 32 * (2 * wv / QW);
    const bool two_pages = PAGED && tl.shift == 4;   // a key load's 32 rows (whose distance fits 32 bits: the host checks)
    auto v_page = [&](int x) __attribute__((always_inline)) { ev = page(x, vg, 16); };
    auto k_page = [&](int x) __attribute__((always_inline)) {
        ek = page(x, kg, two_pages ? 16 : 32);
        if (two_pages) ek1 = page(x, kg + 16, 16);
    };
    uint32_t ko = 0;
    auto k_src = [&](int x) __attribute__((always_inline)) {
        int last;
        if (two_pages) {
            int last1;
            const uint64_t b0 = base_of(x, kg, 16, k_rs, ek, last), b1 = base_of(x, kg + 16, 16, k_rs, ek1, last1);
            const uint64_t b = b0 < b1 ? b0 : b1;
            const bool up = (krow & 16) != 0;
            ko = __umul24(min(krow & 15, (uint32_t)(up ? last1 : last)), krowb) + kcol + (uint32_t)((up ? b1 : b0) - b);
            return khead + b;
        }
        const uint64_t b = base_of(x, kg, 32, k_rs, ek, last);
        ko = __umul24(min(krow, (uint32_t)last), krowb) + kcol;
        return khead + b;
    };
    int vlast = 15;
    auto v_src = [&](int x) __attribute__((always_inline)) { return vhead + base_of(x, vg, 16, v_rs, ev, vlast); };
    auto load_k1 = [&](uint64_t src, uint32_t dst, int u) __attribute__((always_inline)) {
        const uint32_t to = dst + (uint32_t)(1024 * (LP * wv + u));
        if (u == 0) dma1_at<0>(src, ko, to);
        else if (u == 1) dma1_at<32>(src, ko, to);
        else if (u == 2) dma1_at<64>(src, ko, to);
        else dma1_at<96>(src, ko, to);
    };
    auto load_v1 = [&](uint64_t src, uint32_t dst, int u) __attribute__((always_inline)) {
        dma1_at<0>(src, __umul24(min(vrow + 4 * u, (uint32_t)vlast), rowb) + vchunk, dst + (uint32_t)(1024 * (LP * wv + u)));
    };

    // ---- pages in 8 bits: a step's tiles go through registers, loaded a step before they are converted and written to their
    // slots (the same as above: what reads them does not differ). Of a key tile a wave takes 32 rows (two groups of 16 with a scale and
    // a page each, lane's group n >> 4) and 32 LP dims less, of a value tile 64 / QW rows: LP / 2 loads of 16 dims each a lane, which become
    // two fragments' halves, or two chunks.
    constexpr int L8 = LP / 2;
    u32x4 kr8[L8], vr8[L8];
    uint32_t ksc = 0, vsc = 0;
    const uint32_t rs8 = (uint32_t)a.pg.rs;   // (below 2^23: the host checks)
    const uint8_t *const k8 = reinterpret_cast<const uint8_t*>(a.k) + hoff, *const v8 = reinterpret_cast<const uint8_t*>(a.v) + hoff;
    const int kq = wv % (QW / 2), kg8 = kg + (n & 16);   // (wave's dims 32 LP / 2 kq ..; lane's group of rows)
    const uint32_t k8_at = (uint32_t)((8 * (2 * wv / QW) + L8 * 2 * kq + hf) * IMG_FRAG_BYTES + 16 * n);
    const int vrow8 = 64 / QW * wv % 16 + 4 * hf + ((lane >> 1) & 3), vcol8 = (lane & 1) + 2 * ((lane >> 3) & 3);
    const uint32_t v8_at = (uint32_t)vt_offset(64 / QW * wv + 4 * hf + ((lane >> 1) & 3), 2 * vcol8);
    auto pages8 = [&](int vx, int kx) __attribute__((always_inline)) {   // the entries of the next loads
        ev = tl.entry(vx, first(vx, vg, 16) - tl.key0(vx));
        ek = tl.entry(kx, first(kx, kg8, 16) - tl.key0(kx));
    };
    auto load8_k = [&](int x) __attribute__((always_inline)) {
        const int j = first(x, kg8, 16), r = j & ((1 << tl.shift) - 1);
        const int64_t page = max(ek, 0);
        const uint8_t* src = k8 + page * a.pg.ps + (int64_t)((uint64_t)(uint32_t)r * rs8) +
                             (min(krow & 15, (uint32_t)(tl.end - 1 - j)) * rs8 + (uint32_t)(32 * L8 * kq + 16 * hf));
#pragma unroll
        for (int u = 0; u < L8; ++u) kr8[u] = *reinterpret_cast<const u32x4*>(src + 32 * u);
        ksc = a.k_sc[page * a.sc_ps + (int64_t)((r >> 4) * a.HK + hk)];
    };
    auto load8_v = [&](int x) __attribute__((always_inline)) {
        const int j = first(x, vg, 16), r = j & ((1 << tl.shift) - 1), last = tl.end - 1 - j;
        const int64_t page = __builtin_amdgcn_readfirstlane(max(ev, 0));
        const uint8_t* src = v8 + page * a.pg.ps + (int64_t)((uint64_t)(uint32_t)r * rs8);
#pragma unroll
        for (int u = 0; u < L8; ++u)
            vr8[u] = *reinterpret_cast<const u32x4*>(src + ((uint32_t)min(vrow8 + 8 * u, last) * rs8 + (uint32_t)(16 * vcol8)));
        vsc = a.v_sc[page * a.sc_ps + (int64_t)((r >> 4) * a.HK + hk)];
    };
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    // half h of a load's 16 dims
    auto put8_k = [&](uint32_t to, int u, int h) __attribute__((always_inline)) {
        *(lds_u32x4*)(uintptr_t)(to + k8_at + (uint32_t)(2 * IMG_FRAG_BYTES * u + 512 * h)) =
            __builtin_bit_cast(u32x4, widen(kr8[u][2 * h], kr8[u][2 * h + 1], scale8(ksc)));
    };
    auto put8_v = [&](uint32_t to, int u, int h) __attribute__((always_inline)) {
        *(lds_u32x4*)(uintptr_t)(to + v8_at + (uint32_t)(2048 * u + 16 * h)) =
            __builtin_bit_cast(u32x4, widen(vr8[u][2 * h], vr8[u][2 * h + 1], scale8(vsc)));
    };

    // ---- registers (as the key-split kernel's)
    bf16x8 qa[8];
    f32x16 o[4], s[2], negm;
    u32x4 p[2][2];
    float ls = 0.0f;
    bf16x8 fr[FR];
    const uint32_t vlane = (uint32_t)vt_lane(lane);
    auto vfrag_off = [](int x) __attribute__((always_inline)) { return 4096 * (x >> 2) + 256 * (x & 3); };

    auto slot = [](int x) __attribute__((always_inline)) { return (uint32_t)(x % SLOTS * IMG_TILE_BYTES); };
    // V(0) .. V(E) and K(1) .. K(E + 1)
    auto first_pairs = [&]() __attribute__((always_inline)) {
        if constexpr (SRC == PAGES8) {   // K(0) as well; the loads of step 1's
            pages8(tile_of(0), tile_of(0));
            load8_v(tile_of(0));
            load8_k(tile_of(0));
            pages8(tile_of(1), tile_of(1));
#pragma unroll
            for (int u = 0; u < L8; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    put8_k(ring, u, h);
                    put8_v(vring, u, h);
                }
            load8_k(tile_of(1));
            load8_v(tile_of(1));
            pages8(tile_of(2), tile_of(2));
#pragma unroll
            for (int u = 0; u < L8; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) put8_k(ring + slot(1), u, h);
            load8_k(tile_of(2));
            return;
        }
#pragma unroll
        for (int t = 0; t <= E; ++t) {
            v_page(tile_of(t));
            const uint64_t vs = v_src(tile_of(t));
#pragma unroll
            for (int u = 0; u < LP; ++u) load_v1(vs, vring + slot(t), u);
            k_page(tile_of(t + 1));
            const uint64_t ks = k_src(tile_of(t + 1));
#pragma unroll
            for (int u = 0; u < LP; ++u) load_k1(ks, ring + slot(t + 1), u);
        }
    };
    {
        const uint16_t* src = a.q + (int64_t)(sq.t0 + i) * a.q_rs + head * D + 8 * hf;
        if constexpr (SRC != PAGES8) {
            k_page(tile_of(0));
            const uint64_t kb = k_src(tile_of(0));
#pragma unroll
            for (int u = 0; u < LP; ++u) load_k1(kb, ring, u);
        }
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qa[ks] = *reinterpret_cast<const bf16x8*>(src + 16 * ks);
        if constexpr (E == 0) first_pairs();   // (more of them at once would keep the first product waiting)
    }

    // ---- masked half-tiles: what the row does not see out, and a reference for the rows that have none yet
    float mref = 0.0f;
    const float c = a.c;
    bool set = !live;
    bool unset_any = true;
    auto special = [&](int x, int half) __attribute__((always_inline)) {
        const int h = 2 * x + half;
        return unset_any || !(h < free_s || (h >= free_lo && h < free_hi));
    };
    auto mask_half = [&](f32x16& sb, int x, int half) __attribute__((always_inline)) {
        const uint32_t m = seen_bits<BT, SRC>(a, sq, tl, bad, i, me, x, 32 * half) >> (8 * hf);
#pragma unroll
        for (int q = 0; q < 16; ++q)
            sb[q] = if_seen(sb[q], m, 16 * (q >> 3) + (q & 7));
        if (unset_any) {
            float mx = sb[0];
#pragma unroll
            for (int q = 1; q < 16; ++q) mx = fmaxf(mx, sb[q]);
            mx = wave_pair_max(mx);
            // (the scores of a row without a reference are relative to 0)
            const float dm = !set && mx > -INFINITY ? mx : 0.0f;
            set = set || mx > -INFINITY;
            sb -= dm;
            negm -= dm;
            mref = fmaf(dm, c, mref);
            asm volatile(LR_NOP48 : "+v"(negm));
            // rows that see nothing further on need none
            const int next = tl.key0(x) + 32 * half + 32;
            unset_any = __builtin_amdgcn_ballot_w64(!set && me.hi > next) != 0;
        }
    };

    float e0 = 0.0f, e1 = 0.0f;
    auto stage_e = [&](const f32x16& sb, int w) __attribute__((always_inline)) {
        e0 = __builtin_amdgcn_exp2f(sb[8 * (w >> 2) + 2 * (w & 3)] * c);
        e1 = __builtin_amdgcn_exp2f(sb[8 * (w >> 2) + 2 * (w & 3) + 1] * c);
        asm volatile("" ::"v"(e0), "v"(e1));   // computed in this slot, not sunk towards the next use
    };
    const bf16x2 ones2 = {(bf16)1.0f, (bf16)1.0f};
    auto stage_c = [&](u32x4 (&pb)[2], int w) __attribute__((always_inline)) {
        const uint32_t x = pack_bf16x2(e0, e1);
        pb[w >> 2][w & 3] = x;
        ls = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), ones2, ls, false);
        asm volatile("" ::"v"(x), "v"(ls));
    };
    auto half_step = [&](f32x16& so, const u32x4 (&ppv)[2], const f32x16& si, u32x4 (&po)[2], auto pv_tag,
                         auto&& rd) __attribute__((always_inline)) {
        constexpr bool HAS_PV = decltype(pv_tag)::value;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < 16; ++f) {
            if (f < 8) {
                if (f == 0) qk_init(so, fr[0], qa[0], negm);
                else qk_acc(so, fr[f % FR], qa[f]);
            } else {
                if constexpr (HAS_PV) pv(o[(f - 8) & 3], fr[f % FR], ppv[(f - 8) >> 2]);
            }
            if ((f & 1) == 0) stage_e(si, f >> 1);
            else stage_c(po, f >> 1);
            rd(f + RA);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // a step's refills, one load every other slot of its first half: V(t + E) from slot 1 on, then K(t + E + 1) (past the last
    // tile repeats of it, never read); their addresses in the slots before, under the products
    uint64_t src = 0;
    // (in 8 bits: a piece of V(t), loaded in the step before, every other slot, then its registers' next loads; then K(t + 1).)
    auto refill = [&](int f, int t) __attribute__((always_inline)) {
        if constexpr (SRC == PAGES8) {
            constexpr int PIECES = 2 * L8;
            if (f % 2 == 0 && f / 2 < PIECES) put8_v(vring + slot(t), f / 2 / 2, f / 2 % 2);
            if (f == 2 * PIECES - 1) load8_v(tile_of(t + 1));
            if (f % 2 == 0 && f / 2 >= PIECES && f / 2 < 2 * PIECES) put8_k(ring + slot(t + 1), (f / 2 - PIECES) / 2, f / 2 % 2);
            if (f == 4 * PIECES - 1) load8_k(tile_of(t + 2));
            return;
        }
        if (f == 0) src = v_src(tile_of(t + E));
        if (f == 2 * LP) src = k_src(tile_of(t + E + 1));
        if (f % 2 == 1) {
            if (f / 2 < LP) load_v1(src, vring + slot(t + E), f / 2);
            else if (f / 2 < 2 * LP) load_k1(src, ring + slot(t + E + 1), f / 2 - LP);
        }
    };

    // ---- the queries and K(0) resident; S of the first half-tile, and the rows' references
#pragma unroll
    for (int db = 0; db < 4; ++db) o[db] = f32x16{};
    negm = f32x16{};
    if constexpr (SRC == PAGES8) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    else LR_WAIT_VMCNT(0);
    block_barrier();
    if constexpr (E > 0) first_pairs();
    // the entries of step u + 1's refills (of their loads); what a step's end waits for
    auto next_pages = [&](int u) __attribute__((always_inline)) {
        if constexpr (SRC == PAGES8) {
            pages8(tile_of(u + 2), tile_of(u + 3));
        } else {
            v_page(tile_of(u + 1 + E));
            k_page(tile_of(u + 2 + E));
        }
    };
    auto landed = [&]() __attribute__((always_inline)) {
        if constexpr (SRC == PAGES8) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else LR_WAIT_VMCNT(AHEAD);
    };
    // a wave without rows only loads its share of the tiles (and leaves the clock to the others)
    if (row0 + 32 * wv >= rows) {
        for (int u = 0;; ++u) {
            next_pages(u);
            landed();
            block_barrier();
            if (u + 1 >= nsteps) break;
#pragma unroll
            for (int f = 0; f < 4 * LP; ++f) refill(f, u + 1);
        }
        if constexpr (SRC != PAGES8) LR_WAIT_VMCNT(0);
        return;
    }
    {
        uint32_t kb0 = ring + lane16;
        asm volatile("" : "+v"(kb0));
        fence_q8(qa);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            const bf16x8 kf = frag_at(kb0 + (uint32_t)(ks * IMG_FRAG_BYTES));
            if (ks == 0) qk_zero(s[0], kf, qa[0]);
            else qk_acc(s[0], kf, qa[ks]);
        }
        fence_s(s[0]);
        mask_half(s[0], x0, 0);
    }
    // ---- step 0: S of half-tile 1 (K(0), fragments 8-15), P of half-tile 0
    {
        next_pages(0);
        uint32_t kb = ring + lane16;
        asm volatile("" : "+v"(kb));
        auto rd0 = [&](int f) __attribute__((always_inline)) {
            if (f < 8) fr[f % FR] = frag_at(kb + (8 + f) * IMG_FRAG_BYTES);
        };
#pragma unroll
        for (int f = 0; f < RA; ++f) rd0(f);
        half_step(s[1], p[1], s[0], p[0], BoolTag<false>{}, [&](int f) __attribute__((always_inline)) {
            rd0(f);
        });
        landed();
        block_barrier();
        if constexpr (E > 0) {
            uint32_t kn = ring + slot(1) + lane16;
            asm volatile("" : "+v"(kn));
#pragma unroll
            for (int f = 0; f < RA; ++f) fr[f % FR] = frag_at(kn + f * IMG_FRAG_BYTES);
        }
    }
    // ---- step u: key tile u (both halves), value tile u - 1. Its refills go to the slots of V(u - 2) and K(u - 1), both
    // read before the last barrier, and have landed at the end of step u (of step u + E - 1 with E > 0).
    for (int u = 1; u < nsteps; ++u) {
        if constexpr (SRC == PAGES8) mref = fmaf(raise_rows(c, ls, o, p[0], s[1], negm), c, mref);
        const int x = x0 + u, xp = x - 1;
        uint32_t kb = ring + slot(u) + lane16, vb = vring + slot(u - 1) + vlane, kn = ring + slot(u + 1) + lane16;
        asm volatile("" : "+v"(kb), "+v"(vb), "+v"(kn));
        auto rd_b = [&](int f) __attribute__((always_inline)) {
            if (f < 8) fr[f % FR] = frag_at(kb + f * IMG_FRAG_BYTES);
            else if (f < 16) fr[f % FR] = vfrag_at(vb + vfrag_off(f - 8));
            else fr[f % FR] = frag_at(kb + (f - 8) * IMG_FRAG_BYTES);
        };
        auto rd_a = [&](int f) __attribute__((always_inline)) {
            if (PAGED && f == 8) next_pages(u);
            if (f < 8) fr[f % FR] = frag_at(kb + (8 + f) * IMG_FRAG_BYTES);
            else if (f < 16) fr[f % FR] = vfrag_at(vb + vfrag_off(f));
            else if (E > 0) fr[f % FR] = frag_at(kn + (f - 16) * IMG_FRAG_BYTES);   // (the next step's first)
        };
        if constexpr (E == 0)
#pragma unroll
            for (int f = 0; f < RA; ++f) rd_b(f);
        if (special(xp, 1)) mask_half(s[1], xp, 1);
        half_step(s[0], p[0], s[1], p[1], BoolTag<true>{}, [&](int f) __attribute__((always_inline)) {
            refill(f - RA, u);
            rd_b(f);
        });
        if (special(x, 0)) mask_half(s[0], x, 0);
        half_step(s[1], p[1], s[0], p[0], BoolTag<true>{}, rd_a);
        landed();
        block_barrier();
    }
    // ---- the last half-tile's P and the last value tile's products
    {
        if constexpr (SRC == PAGES8) mref = fmaf(raise_rows(c, ls, o, p[0], s[1], negm), c, mref);
        const int u = nsteps - 1, x = x0 + u;
        if constexpr (E > 0) LR_WAIT_VMCNT(0);   // (no load into LDS outlives the workgroup)
        if (special(x, 1)) mask_half(s[1], x, 1);
        uint32_t vb0 = vring + slot(u) + vlane;
        asm volatile("" : "+v"(vb0));
        bf16x8 vf[4];
#pragma unroll
        for (int y = 0; y < 3; ++y) vf[y] = vfrag_at(vb0 + vfrag_off(y));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < 16; ++y) {
            if (y + 3 < 16) vf[(y + 3) & 3] = vfrag_at(vb0 + vfrag_off(y + 3));
            pv(o[y & 3], vf[y & 3], (y < 8 ? p[0] : p[1])[(y >> 2) & 1]);
            if (y < 8) {
                stage_e(s[1], y);
                stage_c(p[1], y);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // ---- rows out. (A row that saw a key has a sum of at least 1; a sum past 2^100, or not a number, means that its reference
    // was overflowed.)
    const float l = wave_pair_sum(ls);
    float nan = l <= 0x1p100f ? 0.0f : __builtin_nanf("");   // NaN iff the row is not finite
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) nan = fmaf(0.0f, o[db][e], nan);
    uint64_t again = __builtin_amdgcn_ballot_w64(nan != 0.0f && live);
    again = (again | again >> 32) & 0xffffffffu;
    if (cut >= 0) {
        if (live) {
            f32x4* po = reinterpret_cast<f32x4*>(a.part_o) + (part * QW + wv) * 1024 + lane;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int gg = 0; gg < 4; ++gg)
                    po[64 * (4 * db + gg)] = f32x4{o[db][4 * gg], o[db][4 * gg + 1], o[db][4 * gg + 2], o[db][4 * gg + 3]};
            a.part_ml[2 * (part * KBM + 32 * wv + n) + hf] = hf ? l : l > 0.0f ? mref : -INFINITY;
        }
    } else {
        // 8 dims a store: the lower lanes take both halves' words of the even 8-dim groups, the upper lanes of the odd ones
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        uint16_t* dst = a.out + (int64_t)(sq.t0 + i) * a.o_rs + head * D + 8 * hf;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t w[2][2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int at = 4 * (2 * x + e);
                    w[e][0] = pack_bf16x2(o[db][at] * inv, o[db][at + 1] * inv);
                    w[e][1] = pack_bf16x2(o[db][at + 2] * inv, o[db][at + 3] * inv);
                }
                const auto r0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
                const auto r1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
                if (live) *reinterpret_cast<u32x4*>(dst + 32 * db + 16 * x) = u32x4{r0[0], r1[0], r0[1], r1[1]};
            }
    }
    while (again) {
        const int q = __builtin_ctzll(again);
        again &= again - 1;
        const int ri = __builtin_amdgcn_readlane(i, q), rhead = __builtin_amdgcn_readlane(head, q);
        redo_row<BT, SRC>(a, sq, tl, hk, ri, rhead, [&](float o0, float o1, float m, float rl) {
            if (cut >= 0) {
                float* po = a.part_o + (part * QW + wv) * 4096 + 256 * (lane >> 2) + 4 * (q + 32 * (lane >> 1 & 1)) + 2 * (lane & 1);
                *reinterpret_cast<float2*>(po) = float2{o0, o1};
                if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (part * KBM + 32 * wv + q)) = float2{m, rl};
            } else {
                put_row(a.out + (int64_t)(sq.t0 + ri) * a.o_rs + rhead * D, o0, o1, rl);
            }
        });
    }
}

// The parts of 32 rows of a block (wave w of the workgroups that had it), by four waves, wave d the dims 32 d .. 32 d + 31. Part x
// lies as its wave held it (slot(x)): row n's references and sums in order, its dims 8 c + 4 hf .. + 3 of 32 d at [4 d + c][n + 32 hf].
// Four parts are in flight. A part that saw no key (reference -inf) has no weight, and its row may never have been written.
template <int QW, class Slot>
__device__ __forceinline__ void merge_rows(const RangeAttnArgs& a, const Seq& sq, int hk, int blk, int w, int parts, Slot&& slot) {
    const int lane = threadIdx.x & 63, n = lane & 31, hf = lane >> 5, d = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows = max(sq.n, 0) * a.G, r = (blk * QW + w) * 32 + n;
    if ((blk * QW + w) * 32 >= rows) return;
    float M = -INFINITY, L = 0.0f;
    f32x4 sum[4] = {};
    for (int s0 = 0; s0 < parts; s0 += 4) {
        float2 ml[4];
        f32x4 x[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t at = slot(min(s0 + u, parts - 1)) * QW + w;
            ml[u] = reinterpret_cast<const float2*>(a.part_ml)[at * 32 + n];
#pragma unroll
            for (int c = 0; c < 4; ++c) x[u][c] = reinterpret_cast<const f32x4*>(a.part_o)[at * 1024 + 64 * (4 * d + c) + lane];
        }
        float Mn = M;
#pragma unroll
        for (int u = 0; u < 4; ++u) Mn = fmaxf(Mn, ml[u].x);
        const float ref = Mn > -INFINITY ? Mn : 0.0f, alpha = __builtin_amdgcn_exp2f(M - ref);
        M = Mn;
        L *= alpha;
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] *= alpha;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool in = ml[u].x > -INFINITY && s0 + u < parts;
            const float wt = __builtin_amdgcn_exp2f(ml[u].x - ref);
            L = in ? fmaf(wt, ml[u].y, L) : L;
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[c][e] = in ? fmaf(wt, x[u][c][e], sum[c][e]) : sum[c][e];
        }
    }
    if (r >= rows) return;
    const int i = div_small(r, a.G, a.rcp_g), head = hk * a.G + r - i * a.G;
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    uint16_t* dst = a.out + (int64_t)(sq.t0 + i) * a.o_rs + head * D + 32 * d + 4 * hf;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        u32x2 v;
        v[0] = pack_bf16x2(sum[c][0] * inv, sum[c][1] * inv);
        v[1] = pack_bf16x2(sum[c][2] * inv, sum[c][3] * inv);
        *reinterpret_cast<u32x2*>(dst + 8 * c) = v;
    }
}

// The parts of the blocks that were cut: workgroup (cut block, 32 rows).
template <int QW, int SRC>
__global__ __launch_bounds__(256) void range_wide_merge_kernel(RangeAttnArgs a) {
    const int c = blockIdx.x / QW, w = blockIdx.x % QW;
    const int of = a.local - a.whole;   // cut blocks an XCD
    const int xcd = a.by_xcd ? c / of : 0, first = a.whole + (c - xcd * of) * a.nsplit;   // the block's first workgroup
    int b, hk, blk, split, cut;
    if (!block_of<QW, SRC>(a, a.by_xcd ? 8 * first + xcd : first, b, hk, blk, split, cut)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    const Seq sq = seq_of<SRC>(a, b);
    merge_rows<QW>(a, sq, hk, blk, w, a.nsplit, [&](int x) { return (int64_t)cut * a.nsplit + x; });
}

// The same of pieces: workgroup (pair, row block, 32 rows).
template <int QW>
__global__ __launch_bounds__(256) void range_pieces_merge_kernel(RangeAttnArgs a) {
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3, c = at / QW, j = div_small(c, a.nblk, a.rcp_nblk), blk = c - j * a.nblk;
    Pieces pc;
    pc.template init<32 * QW>(a, xcd);
    const int e = __builtin_amdgcn_readlane(pc.end, j), s = e - __builtin_amdgcn_readlane(pc.tiles, j), t0 = s / pc.Q;
    const int parts = 1 + (max(e - 1, 0) / pc.Q - t0);
    if (s == e || parts <= 1) return;   // (the attention wrote its rows)
    const int pair = 8 * j + xcd, b = div_small(pair, a.HK, a.rcp_hk), hk = pair - b * a.HK;
    const Seq sq = seq_of<PAGES>(a, b);
    merge_rows<QW>(a, sq, hk, blk, at % QW, parts, [&](int x) {
        return (int64_t)(xcd * (pc.P + a.teams) + (x == 0 ? j : pc.P + t0 + x - 1)) * a.nblk + blk;
    });
}

// The same of shares: workgroup (pair, block, 32 rows).
template <int QW>
__global__ __launch_bounds__(256) void range_shares_merge_kernel(RangeAttnArgs a) {
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3, c = at / QW, j = div_small(c, a.nblk, a.rcp_nblk), nth = c - j * a.nblk;
    BlockPieces pc;
    pc.init(a, xcd);
    const int blocks = __builtin_amdgcn_readlane(pc.blocks, j);
    if (nth >= blocks) return;
    const int p0 = pc.begin(j, nth), first = p0 / pc.Q, parts = (p0 + __builtin_amdgcn_readlane(pc.tiles, j) - 1) / pc.Q - first + 1;
    if (parts <= 1) return;   // (the attention wrote its rows)
    const int pair = 8 * j + xcd, b = div_small(pair, a.HK, a.rcp_hk), hk = pair - b * a.HK;
    const int x0 = p0 % pc.Q ? BlockPieces::PLACES + __builtin_amdgcn_readlane(pc.last, j) - blocks + nth : first;
    merge_rows<QW>(a, seq_of<PAGES8>(a, b), hk, blocks - 1 - nth, at % QW, parts, [&](int x) {
        return (int64_t)xcd * (BlockPieces::PLACES + pc.P * a.nblk) + (x == 0 ? x0 : first + x);
    });
}

template <int QW, int SRC>
hipError_t launch_waves(const RangeAttnArgs& a, hipStream_t stream) {
    if constexpr (paged(SRC))
        if (a.teams) {
            const int64_t pairs = (int64_t)a.B * a.HK, blocks = (pairs + 8 * a.teams) * a.nblk, merge = pairs * a.nblk * QW;
            hipLaunchKernelGGL((range_wide_kernel<QW, SRC>), dim3((unsigned)blocks), dim3(64 * QW), 0, stream, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(range_pieces_merge_kernel<QW>, dim3((unsigned)merge), dim3(256), 0, stream, a);
            return hipGetLastError();
        }
    if constexpr (SRC == PAGES8 && QW == 8)
        if (a.places) {
            const int64_t pairs = (int64_t)a.B * a.HK, blocks = 8 * BlockPieces::PLACES + pairs * a.nblk;
            hipLaunchKernelGGL((range_wide_kernel<QW, SRC>), dim3((unsigned)blocks), dim3(64 * QW), 0, stream, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(range_shares_merge_kernel<QW>, dim3((unsigned)(pairs * a.nblk * QW)), dim3(256), 0, stream, a);
            return hipGetLastError();
        }
    const int xcds = a.by_xcd ? 8 : 1;
    const int64_t of = a.nsplit > 1 ? a.local - a.whole : 0;   // cut blocks
    const int64_t blocks = xcds * (a.local + of * (a.nsplit - 1)), merge = xcds * of * QW;
    if (blocks > RANGE_MAX_BLOCKS || merge > 2 * RANGE_MAX_BLOCKS) return hipErrorInvalidValue;
    hipLaunchKernelGGL((range_wide_kernel<QW, SRC>), dim3((unsigned)blocks), dim3(64 * QW), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || of == 0) return e;
    hipLaunchKernelGGL((range_wide_merge_kernel<QW, SRC>), dim3((unsigned)merge), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_range_wide8(const RangeAttnArgs& a, int waves, hipStream_t stream) {
    return waves == 8 ? launch_waves<8, PAGES8>(a, stream) : launch_waves<4, PAGES8>(a, stream);
}

hipError_t launch_range_wide(const RangeAttnArgs& a, bool paged, int waves, hipStream_t stream) {
    if (waves == 8) return paged ? launch_waves<8, PAGES>(a, stream) : launch_waves<8, ROWS>(a, stream);
    return paged ? launch_waves<4, PAGES>(a, stream) : launch_waves<4, ROWS>(a, stream);
}

}  // namespace lr
