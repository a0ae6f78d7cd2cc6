// The ranged attention (attn_cache.hip) of calls with many rows of a kv head: chunks, frames and large trees, where the matrix
// products bound it. The same contract; the loop is that of the key-split kernel (attn_keysplit.hip): a half-step of 16 MFMA
// slots runs the next half-tile's scores, the previous one's products and this one's exponentials. A workgroup is 128 rows
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
#include "range_attn.inc"

// One 1 KB direct load, global -> LDS: lane l's 16 bytes come from gaddr + voff + OFF and land at lds + 16 l (the instruction
// offset applies to both addresses).
template <int OFF>
__device__ __forceinline__ void dma1_at(uint64_t gaddr, uint32_t voff, uint32_t lds) {
    LR_ASM_M0_BEGIN
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%3" ::"v"(voff), "s"(gaddr), "s"(lds - OFF),
                 "n"(OFF)
                 : "memory", "m0");
    LR_ASM_M0_END
}

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
template <int QW, bool PAGED>
__device__ __forceinline__ bool block_of(const RangeAttnArgs& a, int id, int& b, int& hk, int& blk, int& split, int& cut) {
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
        const Seq sq = seq_of<true>(a, div_small(pair, a.HK, a.rcp_hk));
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

template <int QW, bool PAGED>
__global__ __launch_bounds__(64 * QW, 8 / QW) __attribute__((amdgpu_waves_per_eu(2, 2))) void range_wide_kernel(RangeAttnArgs a) {
    constexpr int KBM = 32 * QW;                        // rows per block
    // steps of refills in flight beside the current one's. (8 waves have the LDS for 2: pages come from HBM, ~2 us away under load: 16
    // trees of up to 64 tokens over up to 30,000 keys 860 -> 841 us. Rows come from the L2s: 16,384 tokens of video 1,171 us with 2,
    // 1,164 with 0.)
    constexpr int E = QW == 8 && PAGED ? 2 : 0;
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

    int b, hk, blk, split, cut, px0 = 0, px1 = 0;
    if (PAGED && a.teams) {
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
    } else if (!block_of<QW, PAGED>(a, blockIdx.x, b, hk, blk, split, cut)) {
        return;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    hk = __builtin_amdgcn_readfirstlane(hk);
    blk = __builtin_amdgcn_readfirstlane(blk);
    const Seq sq = seq_of<PAGED>(a, b);
    const int row0 = blk * KBM;
    const int rows = max(sq.n, 0) * a.G;   // (at most 2^30: the host checks)
    if (row0 >= rows) return;
    TileList<BT, PAGED> tl;
    tl.init(a, sq, div_small(row0, a.G, a.rcp_g), div_small(min(rows, row0 + KBM) - 1, a.G, a.rcp_g));
    if (PAGED && a.teams) {
        tl.x0 = px0;
        tl.x1 = min(tl.total, px1);
    } else if (PAGED || cut >= 0) tl.part(split, a.per ? a.per : div_small(tl.total + a.nsplit - 1, a.nsplit, a.rcp_split));
    const bool bad = tl.template stage<64 * QW>(a, b, staged);
    const int x0 = __builtin_amdgcn_readfirstlane(tl.x0), x1 = __builtin_amdgcn_readfirstlane(tl.x1);

    // ---- this lane's row
    const int r = row0 + 32 * wv + n, rr = min(r, rows - 1);
    const bool live = r < rows;
    const int i = div_small(rr, a.G, a.rcp_g), head = hk * a.G + rr - i * a.G;
    const Sees me = sees_of<PAGED>(a, sq, i);
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
        k_page(tile_of(0));
        const uint64_t kb = k_src(tile_of(0));
#pragma unroll
        for (int u = 0; u < LP; ++u) load_k1(kb, ring, u);
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
        const uint32_t m = seen_bits<BT, PAGED>(a, sq, tl, bad, i, me, x, 32 * half) >> (8 * hf);
#pragma unroll
        for (int q = 0; q < 16; ++q)
            if (!(m >> (16 * (q >> 3) + (q & 7)) & 1)) sb[q] = -INFINITY;
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
    auto refill = [&](int f, int t) __attribute__((always_inline)) {
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
    LR_WAIT_VMCNT(0);
    block_barrier();
    if constexpr (E > 0) first_pairs();
    // a wave without rows only loads its share of the tiles (and leaves the clock to the others)
    if (row0 + 32 * wv >= rows) {
        for (int u = 0;; ++u) {
            v_page(tile_of(u + 1 + E));
            k_page(tile_of(u + 2 + E));
            LR_WAIT_VMCNT(AHEAD);
            block_barrier();
            if (u + 1 >= nsteps) break;
#pragma unroll
            for (int f = 0; f < 4 * LP; ++f) refill(f, u + 1);
        }
        LR_WAIT_VMCNT(0);
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
        v_page(tile_of(1 + E));   // (of step 1's refills)
        k_page(tile_of(2 + E));
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
        LR_WAIT_VMCNT(AHEAD);
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
        const int x = x0 + u, xp = x - 1;
        uint32_t kb = ring + slot(u) + lane16, vb = vring + slot(u - 1) + vlane, kn = ring + slot(u + 1) + lane16;
        asm volatile("" : "+v"(kb), "+v"(vb), "+v"(kn));
        auto rd_b = [&](int f) __attribute__((always_inline)) {
            if (f < 8) fr[f % FR] = frag_at(kb + f * IMG_FRAG_BYTES);
            else if (f < 16) fr[f % FR] = vfrag_at(vb + vfrag_off(f - 8));
            else fr[f % FR] = frag_at(kb + (f - 8) * IMG_FRAG_BYTES);
        };
        auto rd_a = [&](int f) __attribute__((always_inline)) {
            if (PAGED && f == 8) {
                v_page(tile_of(u + 1 + E));
                k_page(tile_of(u + 2 + E));
            }
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
        LR_WAIT_VMCNT(AHEAD);
        block_barrier();
    }
    // ---- the last half-tile's P and the last value tile's products
    {
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
        redo_row<BT, PAGED>(a, sq, tl, hk, ri, rhead, [&](float o0, float o1, float m, float rl) {
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
template <int QW, bool PAGED>
__global__ __launch_bounds__(256) void range_wide_merge_kernel(RangeAttnArgs a) {
    const int c = blockIdx.x / QW, w = blockIdx.x % QW;
    const int of = a.local - a.whole;   // cut blocks an XCD
    const int xcd = a.by_xcd ? c / of : 0, first = a.whole + (c - xcd * of) * a.nsplit;   // the block's first workgroup
    int b, hk, blk, split, cut;
    if (!block_of<QW, PAGED>(a, a.by_xcd ? 8 * first + xcd : first, b, hk, blk, split, cut)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    const Seq sq = seq_of<PAGED>(a, b);
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
    const Seq sq = seq_of<true>(a, b);
    merge_rows<QW>(a, sq, hk, blk, at % QW, parts, [&](int x) {
        return (int64_t)(xcd * (pc.P + a.teams) + (x == 0 ? j : pc.P + t0 + x - 1)) * a.nblk + blk;
    });
}

template <int QW, bool PAGED>
hipError_t launch_waves(const RangeAttnArgs& a, hipStream_t stream) {
    if constexpr (PAGED)
        if (a.teams) {
            const int64_t pairs = (int64_t)a.B * a.HK, blocks = (pairs + 8 * a.teams) * a.nblk, merge = pairs * a.nblk * QW;
            hipLaunchKernelGGL((range_wide_kernel<QW, PAGED>), dim3((unsigned)blocks), dim3(64 * QW), 0, stream, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(range_pieces_merge_kernel<QW>, dim3((unsigned)merge), dim3(256), 0, stream, a);
            return hipGetLastError();
        }
    const int xcds = a.by_xcd ? 8 : 1;
    const int64_t of = a.nsplit > 1 ? a.local - a.whole : 0;   // cut blocks
    const int64_t blocks = xcds * (a.local + of * (a.nsplit - 1)), merge = xcds * of * QW;
    if (blocks > RANGE_MAX_BLOCKS || merge > 2 * RANGE_MAX_BLOCKS) return hipErrorInvalidValue;
    hipLaunchKernelGGL((range_wide_kernel<QW, PAGED>), dim3((unsigned)blocks), dim3(64 * QW), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || of == 0) return e;
    hipLaunchKernelGGL((range_wide_merge_kernel<QW, PAGED>), dim3((unsigned)merge), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_range_wide(const RangeAttnArgs& a, bool paged, int waves, hipStream_t stream) {
    if (waves == 8) return paged ? launch_waves<8, true>(a, stream) : launch_waves<8, false>(a, stream);
    return paged ? launch_waves<4, true>(a, stream) : launch_waves<4, false>(a, stream);
}

}  // namespace lr
