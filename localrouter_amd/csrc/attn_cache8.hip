// Attention over a cache in pages of 8 bits (gfx950): what attn_cache.hip computes over bf16 pages, with
//
//   k_j = 2^e(j) q8_j,  v_j the same: e4m3 rows, a scale for each 16 rows of a page and head (cache8_rows.hip)
//
// for single tokens and small trees: bound by HBM where there is much to read (half of what bf16 pages take), and by the chain
// from one load and one instruction to the next where there is not.
//
// A workgroup is a block of 16 or 32 rows (tokens x the query heads of one kv head), or the same block of two kv heads, and a part of its
// tiles of 32 keys, which a head's waves (two, four or eight) take in turn. Keys and values go from memory to registers, not through LDS:
// a lane's 32 bytes of a key are four steps of its products' operand (dims 16 g .. + 15 and 64 + 16 g .. + 15 of row n for lane 16 g + n;
// the queries' lanes hold the same dims), and of the values it takes 8 dims of the 8 keys whose probabilities it holds, transposed by byte
// permutations. Conversion to bf16 with the scale is one instruction for two values, and exact: e4m3 has 4 significant bits and bf16's
// exponents. P is rounded to bf16, which the products take, and the sum is that of the rounded P; everything else is fp32. (Error against
// 64 bits, relative L2: 0.0017 to 0.0020; the output's own rounding alone 0.0017.)
//
// Single tokens of 48 sequences of up to 9,000 positions, 32 heads over 8, 648 MB: 135 us, 4.8 TB/s; of one sequence of 2,100 10.0 us. 20
// trees of 9 tokens over up to 12,000, 24 over 8, 363 MB: 96 us, of which the merge is 6.
#include "lr_common.h"
#include "lr_cache_kernels.h"

namespace lr {

namespace {

#include "attn_common.inc"

#include "range_attn.inc"
#include "range_parts.inc"

// Bytes of four words a, b, c, d: word i of the result holds byte i of each.
__device__ __forceinline__ u32x4 transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602);
    const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602);
    return u32x4{__builtin_amdgcn_perm(cd0, ab0, 0x05040100), __builtin_amdgcn_perm(cd0, ab0, 0x07060302),
                 __builtin_amdgcn_perm(cd1, ab1, 0x05040100), __builtin_amdgcn_perm(cd1, ab1, 0x07060302)};
}

// What a wave holds of a tile of 32 keys: two halves of 16, each in one page.
struct Keys8 {
    u32x4 k[2][2];   // key n of the half: dims 16 g .. + 15 and 64 + 16 g .. + 15
    uint32_t s[2];
};
struct Values8 {
    u32x2 v[2][4];   // values 4 g + r of the half: dims 8 n .. + 7
    uint32_t s[2];
};

// HW kv heads a workgroup, KH waves each, that take the tiles of the same keys at the same time: of pages that lie token by token, two
// heads' rows are 256 bytes next to each other (32 sequences of 10,000 to 20,000 keys over 8 heads, 970 MB, one head a workgroup 4.4
// TB/s, two 5.0).
// Lane 16 g + n: row n of each block of 16; of a tile's scores the keys 4 g + r and 16 + 4 g + r (r < 4), in which order its
// products take the keys; of the sums the dims 32 g + 8 r + d, o[d][r].
// SHARES: a batch of one block a sequence and kv head in equal shares. Its pairs (sequence, workgroup's heads) lie end to end, and a
// workgroup takes the Q tiles from w Q on, whatever the lengths: the end of one pair, whole ones, the beginning of another. Parts of a
// pair: slot 2 w + 1 of the workgroup where it begins, slot 2 w of the others.
struct Shares {
    int B, tiles, end, Q;   // lane b: the sequence's tiles, and where its pairs end

    __device__ __forceinline__ void init(const RangeAttnArgs& a) {
        const int lane = threadIdx.x & 63;
        B = a.B;
        const Seq sq = seq_of<PAGES8>(a, min(lane, B - 1));
        int lo, hi;
        TileList<RANGE_TILE, PAGES8>::limits(a, sq, 0, max(sq.n, 1) - 1, lo, hi);
        tiles = lane < B && sq.n > 0 ? max(1, TileList<RANGE_TILE, PAGES8>::count(a, lo, hi)) : 0;
        end = tiles * a.hgroups;   // (the host checks that all of them fit)
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(end, d, 64);
            end += lane >= d ? x : 0;
        }
        const int all = __builtin_amdgcn_readlane(end, 63);
        Q = max(a.per, (all + a.places - 1) / a.places);
    }
    __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(end, 63); }
    // the pair at `pos`: its sequence, heads, tiles and where it begins
    __device__ __forceinline__ void at(int pos, int& b, int& hg, int& n, int& begin) const {
        b = __popcll(__builtin_amdgcn_ballot_w64(end <= pos));
        n = __builtin_amdgcn_readlane(tiles, b);
        const int first = b ? __builtin_amdgcn_readlane(end, b - 1) : 0;
        hg = (int)((uint32_t)(pos - first) / (uint32_t)n);
        begin = first + hg * n;
    }
};

template <int NB, int KH, int HW, bool SHARES>
__global__ __launch_bounds__(KH * HW * 64, NB == 1 && !SHARES ? 3 : 2) void range8_step_kernel(RangeAttnArgs a) {
    constexpr int SRC = PAGES8, BT = RANGE_TILE, BR = 16 * NB, KG = KH * HW;
    constexpr int OWN_F = NB * 8 * 256;   // a wave's sums
    __shared__ __attribute__((aligned(1024))) float mo[KG * OWN_F];
    __shared__ float2 mls[KG * NB * 16];
    __shared__ int staged[RANGE8_STAGED];

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kg = wave % KH, hw = wave / KH;

    // ---- which rows, which keys
    int at = 0, split = 0, blk = 0, hg, b, pos = 0, pos_end = 1, pair_tiles = 0, pair = 0;
    Shares sh;
    if constexpr (SHARES) {
        sh.init(a);
        pos = blockIdx.x * sh.Q;
        pos_end = min(sh.all(), pos + sh.Q);
    } else {
        at = div_small(blockIdx.x, a.nsplit, a.rcp_split);
        split = blockIdx.x - at * a.nsplit;
        blk = div_small(at, a.hgroups, a.rcp_hk);
        hg = at - blk * a.hgroups;
        b = blockIdx.y;
    }
  while (pos < pos_end) {
    int lane = tid & 63;
    if constexpr (SHARES) {
        asm volatile("" : "+v"(lane));   // (what is computed of it stays inside the loop: it would not fit the registers beside it)
        sh.at(pos, b, hg, pair_tiles, pair);
        b = __builtin_amdgcn_readfirstlane(b);
        hg = __builtin_amdgcn_readfirstlane(hg);
    }
    const int n = lane & 15, g = lane >> 4;
    const int hk = hg * HW + hw;
    // without a window a part's entries do not depend on the sequence: they are read beside its numbers
    int early = -1;
    const int per_tile = max(1, BT >> a.pg.shift);
    const bool ahead = !SHARES && !a.window && a.per * per_tile <= KG * 64;
    if (ahead && tid < a.per * per_tile) {
        const int j = BT * (split * a.per + tid / per_tile) + (tid % per_tile << a.pg.shift);
        if (j >> a.pg.shift < a.pg.table_pages) early = a.pg.table[(int64_t)b * a.pg.table_rs + (j >> a.pg.shift)];
    }
    const Seq sq = seq_of<SRC>(a, b);
    const int row0 = blk * BR, rows = max(sq.n, 0) * a.G;   // (at most 2^30: the host checks)
    if (row0 >= rows) return;
    const int i_first = div_small(row0, a.G, a.rcp_g), i_last = div_small(min(rows, row0 + BR) - 1, a.G, a.rcp_g);
    TileList<BT, SRC> tl;
    tl.init(a, sq, i_first, i_last);
    int parts, first_share = 0;
    if constexpr (SHARES) {
        const int x = pos - pair, y = min(pair_tiles, x + pos_end - pos);
        pos += y - x;
        tl.x0 = __builtin_amdgcn_readfirstlane(x);
        tl.x1 = __builtin_amdgcn_readfirstlane(min(tl.total, y));
        first_share = (int)((uint32_t)pair / (uint32_t)sh.Q);
        parts = __builtin_amdgcn_readfirstlane((int)((uint32_t)(pair + pair_tiles - 1) / (uint32_t)sh.Q) - first_share + 1);
        split = (int)blockIdx.x - first_share;
    } else {
        tl.part(split, a.per);
        parts = min(a.nsplit, max(1, (tl.total + a.per - 1) / a.per));   // the sequence may be shorter than the longest
        if (split >= parts) return;
        pos = pos_end;
    }
    const int x0 = tl.x0, x1 = tl.x1;
    auto slot = [&](int i) { return SHARES ? 2 * (first_share + i) + (i == 0) : i; };

    // ---- this lane's rows
    const int64_t hoff = (int64_t)hk * a.pg.hs;
    bool live[NB];
    int ri[NB], head[NB];
    Sees me[NB];
    bf16x8 qf[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int r = row0 + 16 * nb + n, rr = min(r, rows - 1);
        live[nb] = r < rows;
        ri[nb] = div_small(rr, a.G, a.rcp_g);
        head[nb] = hk * a.G + rr - ri[nb] * a.G;
        me[nb] = sees_of<SRC>(a, sq, ri[nb]);
        const uint16_t* src = a.q + (int64_t)(sq.t0 + ri[nb]) * a.q_rs + head[nb] * D + 16 * g;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[nb][ks] = *reinterpret_cast<const bf16x8*>(src + 64 * (ks >> 1) + 8 * (ks & 1));
    }
    int hi_all, lo_all, lo_last;
    seen_by_all<SRC>(a, sq, i_first, i_last, me[0], hi_all, lo_all);
    if (NB > 1) {
        seen_by_all<SRC>(a, sq, i_first, i_last, me[NB - 1], hi_all, lo_last);
        lo_all = max(lo_all, lo_last);
    }
    const bool bad = tl.template stage<KG * 64>(a, b, staged, ahead, early);

    const int mine = x1 > x0 + kg ? (x1 - x0 - kg + KH - 1) / KH : 0;   // tiles of this wave
    auto tile_of = [&](int t) { return x0 + kg + t * KH; };
    const uint8_t *k8 = reinterpret_cast<const uint8_t*>(a.k) + hoff, *v8 = reinterpret_cast<const uint8_t*>(a.v) + hoff;
    const uint32_t rs = (uint32_t)a.pg.rs;   // (below 2^23: the host checks)

    f32x4 o[NB][8];
    float m_used[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        m_used[nb] = -INFINITY;
        l[nb] = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[nb][d] = f32x4{};
    }
    const float c = a.c;
    const bf16x2 ones2 = {(bf16)1.0f, (bf16)1.0f};

    // (rows past the last key read that one)
    auto half_of = [&](int x, int hb, int64_t& base, int64_t& sc, uint32_t& last) __attribute__((always_inline)) {
        const int k0 = tl.key0(x), j = min(k0 + 16 * hb, (tl.end - 1) & ~15);
        const int page = max(__builtin_amdgcn_readfirstlane(tl.entry(x, j - k0)), 0), r = j & ((1 << tl.shift) - 1);
        base = (int64_t)page * a.pg.ps + (int64_t)r * a.pg.rs;
        sc = (int64_t)page * a.sc_ps + (int64_t)(r >> 4) * a.HK + hk;
        last = (uint32_t)min(15, tl.end - 1 - j);
    };
    auto load_k = [&](Keys8& w, int x) __attribute__((always_inline)) {
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
            int64_t base, sc;
            uint32_t last;
            half_of(x, hb, base, sc, last);
            const uint8_t* src = k8 + base + (min((uint32_t)n, last) * rs + 16 * g);
            w.k[hb][0] = *reinterpret_cast<const u32x4*>(src);
            w.k[hb][1] = *reinterpret_cast<const u32x4*>(src + 64);
            w.s[hb] = a.k_sc[sc];
        }
    };
    auto load_v = [&](Values8& w, int x) __attribute__((always_inline)) {
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
            int64_t base, sc;
            uint32_t last;
            half_of(x, hb, base, sc, last);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                w.v[hb][r] = *reinterpret_cast<const u32x2*>(v8 + base + (min((uint32_t)(4 * g + r), last) * rs + 8 * n));
            w.s[hb] = a.v_sc[sc];
        }
    };
    // tile t, whose keys are in w and values in wv; then they take the keys of tile t + 2 and the values of tile t + VA
    constexpr int VA = NB == 1 ? 2 : 1;   // (blocks of 32 rows have no registers for two tiles of values)
    auto step = [&](Keys8& w, Values8& wv, int t) __attribute__((always_inline)) {
        const int x = tile_of(t), key0 = tl.key0(x);
        f32x4 s[NB][2] = {};
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
            const float sc = scale8(w.s[hb]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const bf16x8 kf = widen(w.k[hb][ks >> 1][2 * (ks & 1)], w.k[hb][ks >> 1][2 * (ks & 1) + 1], sc);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) s[nb][hb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[nb][ks], s[nb][hb], 0, 0, 0);
            }
        }
        if (t + 2 < mine) load_k(w, tile_of(t + 2));
        const bool whole = key0 + BT <= hi_all && (key0 >= lo_all || key0 + BT <= a.sinks) && !bad;
        u32x4 pw[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            f32x4 &s0 = s[nb][0], &s1 = s[nb][1];
            if (!whole) {
                const uint32_t m = seen_bits<BT, SRC>(a, sq, tl, bad, ri[nb], me[nb], x, 0) >> (4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s0[e] = if_seen(s0[e], m, e);
                    s1[e] = if_seen(s1[e], m, 16 + e);
                }
            }
            const float mx = c * quad_max(fmaxf(fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s0[2], s0[3])),
                                                fmaxf(fmaxf(s1[0], s1[1]), fmaxf(s1[2], s1[3]))));
            if (__builtin_amdgcn_ballot_w64(mx > m_used[nb] + RESCALE_TAU)) {
                const float mn = fmaxf(m_used[nb], mx);
                const float alpha = mn > -INFINITY ? __builtin_amdgcn_exp2f(m_used[nb] - mn) : 1.0f;
                m_used[nb] = mn;
                l[nb] *= alpha;
#pragma unroll
                for (int d = 0; d < 8; ++d) o[nb][d] *= alpha;
            }
            // (no key seen so far: the reference is -inf and every score -inf; any finite reference gives P = 0)
            const float nm = m_used[nb] > -INFINITY ? -m_used[nb] : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t p2 = pack_bf16x2(__builtin_amdgcn_exp2f(fmaf(s[nb][e >> 1][2 * (e & 1)], c, nm)),
                                                __builtin_amdgcn_exp2f(fmaf(s[nb][e >> 1][2 * (e & 1) + 1], c, nm)));
                pw[nb][e] = p2;
                l[nb] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p2), ones2, l[nb], false);
            }
        }
        const float sv0 = scale8(wv.s[0]), sv1 = scale8(wv.s[1]);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const u32x4 lo = transpose4(wv.v[0][0][y], wv.v[0][1][y], wv.v[0][2][y], wv.v[0][3][y]);
            const u32x4 hi = transpose4(wv.v[1][0][y], wv.v[1][1][y], wv.v[1][2][y], wv.v[1][3][y]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bf16x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo[e], sv0, false);
                const bf16x2 a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo[e], sv0, true);
                const bf16x2 b0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi[e], sv1, false);
                const bf16x2 b1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi[e], sv1, true);
                const bf16x8 vf = __builtin_shufflevector(__builtin_shufflevector(a0, a1, 0, 1, 2, 3),
                                                          __builtin_shufflevector(b0, b1, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    o[nb][4 * y + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8, pw[nb]), o[nb][4 * y + e], 0, 0, 0);
            }
        }
        if (t + VA < mine) load_v(wv, tile_of(t + VA));
    };
    Keys8 ka, kb;
    Values8 va, vb;
    if (mine > 0) {
        load_k(ka, tile_of(0));
        load_v(va, tile_of(0));
    }
    if (mine > 1) {
        load_k(kb, tile_of(1));
        if (VA == 2) load_v(vb, tile_of(1));
    }
    for (int t = 0; t < mine; t += 2) {
        step(ka, va, t);
        if (t + 1 < mine) step(kb, VA == 2 ? vb : va, t + 1);
    }

    // ---- merge a head's waves: wave u takes the dims 32 g + 4 x .. + 3, x = u, u + KH, .., from all of them; rows out: O / l, or
    // this part of them
    static_assert(NB <= 2 && 8 % KH == 0, "waves");
    constexpr int OWN = 8 / KH;
    const bool whole_block = parts == 1;
    const PartRows<BR * HW> to(a, SHARES ? 0 : (((int64_t)b * a.nblk + blk) * a.hgroups + hg) * a.nsplit, SHARES ? 2 * a.places : a.nsplit);
    const int mine_slot = slot(split);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        l[nb] = quad_sum(l[nb]);
        if (live[nb]) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {   // dims 32 g + 4 u + e: o[4 (u & 1) + e][u >> 1]
                const f32x4 y = f32x4{o[nb][4 * (u & 1)][u >> 1], o[nb][4 * (u & 1) + 1][u >> 1], o[nb][4 * (u & 1) + 2][u >> 1],
                                      o[nb][4 * (u & 1) + 3][u >> 1]};
                *reinterpret_cast<f32x4*>(mo + wave * OWN_F + (nb * 8 + u) * 256 + 4 * lane) = y;
            }
            if (g == 0) mls[(wave * NB + nb) * 16 + n] = float2{m_used[nb], l[nb]};
        }
    }
    __syncthreads();
    uint32_t broken = 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        bool mine_broken = false;
        if (live[nb]) {
            float mm = -INFINITY, w[KH], sum = 0.0f;
            float2 ml[KH];
#pragma unroll
            for (int u = 0; u < KH; ++u) {
                ml[u] = mls[((hw * KH + u) * NB + nb) * 16 + n];
                mm = fmaxf(mm, ml[u].x);
            }
            const float ref = mm > -INFINITY ? mm : 0.0f;
#pragma unroll
            for (int u = 0; u < KH; ++u) {
                w[u] = __builtin_amdgcn_exp2f(ml[u].x - ref);
                sum = fmaf(w[u], ml[u].y, sum);
            }
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            float chk = sum;
#pragma unroll
            for (int x = 0; x < OWN; ++x) {
                f32x4 own{};
#pragma unroll
                for (int u = 0; u < KH; ++u) {
                    const f32x4 y = *reinterpret_cast<const f32x4*>(mo + (hw * KH + u) * OWN_F + (nb * 8 + kg + KH * x) * 256 + 4 * lane);
#pragma unroll
                    for (int e = 0; e < 4; ++e) own[e] = fmaf(w[u], y[e], own[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) chk = fmaf(0.0f, own[e], chk);
                const int dim = 32 * g + 4 * (kg + KH * x);
                if (whole_block) {
                    u32x2 v;
                    v[0] = pack_bf16x2(own[0] * inv, own[1] * inv);
                    v[1] = pack_bf16x2(own[2] * inv, own[3] * inv);
                    *reinterpret_cast<u32x2*>(a.out + (int64_t)(sq.t0 + ri[nb]) * a.o_rs + head[nb] * D + dim) = v;
                } else {
                    to.put4(mine_slot, hw * BR + 16 * nb + n, dim, own);
                }
            }
            if (!whole_block && g == 0 && kg == 0) to.put_ml(mine_slot, hw * BR + 16 * nb + n, mm, sum);
            mine_broken = !(fabsf(chk) < INFINITY);
        }
        const uint64_t bits = __builtin_amdgcn_ballot_w64(mine_broken);
        const uint32_t half = (uint32_t)(bits | bits >> 32);
        broken |= ((half | half >> 16) & 0xffff) << (16 * nb);
    }
    // ---- rows with an infinity or NaN in some wave's dims again, whole, over the seen keys only
    if (!whole_block) LR_WAIT_VMCNT(0);   // (this wave's part is in memory)
    int* again = reinterpret_cast<int*>(mo);
    again_rows<HW, KH>(again, hw, kg, broken, [&](int q) __attribute__((always_inline)) {
        int i = __builtin_amdgcn_readlane(ri[0], q & 15), h = __builtin_amdgcn_readlane(head[0], q & 15);
        if (NB > 1 && q >= 16) {
            i = __builtin_amdgcn_readlane(ri[NB - 1], q & 15);
            h = __builtin_amdgcn_readlane(head[NB - 1], q & 15);
        }
        redo_row<BT, SRC>(a, sq, tl, hk, i, h, [&](float o0, float o1, float m, float rl) {
            if (whole_block) put_row(a.out + (int64_t)(sq.t0 + i) * a.o_rs + h * D, o0, o1, rl);
            else to.put_row2(mine_slot, hw * BR + q, o0, o1, m, rl);
        });
    });
    if (!whole_block && a.merge_here) to.template merge_last<KG, BR>(a, sq, hg * HW, row0, rows, split, parts, again, slot);
    if constexpr (SHARES) __syncthreads();   // (the sums' and the entries' place)
  }
}

// The parts of the blocks that more than one workgroup had, a wave a row.
template <int NB, int HW, bool SHARES>
__global__ __launch_bounds__(256) void range8_merge_kernel(RangeAttnArgs a) {
    constexpr int BR = 16 * NB, ALL = BR * HW;
    const int at = blockIdx.x / (ALL / 4), q = blockIdx.x % (ALL / 4) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int blk = div_small(at, a.hgroups, a.rcp_hk), hg = at - blk * a.hgroups, b = blockIdx.y;
    const Seq sq = seq_of<PAGES8>(a, b);
    const int rows = max(sq.n, 0) * a.G, row0 = blk * BR, r = row0 + q % BR, hk = hg * HW + q / BR;
    if (r >= rows) return;
    TileList<RANGE_TILE, PAGES8> tl;
    tl.init(a, sq, div_small(row0, a.G, a.rcp_g), div_small(min(rows, row0 + BR) - 1, a.G, a.rcp_g));
    int parts = min(a.nsplit, (tl.total + a.per - 1) / a.per), first_share = 0;
    if constexpr (SHARES) {
        Shares sh;
        sh.init(a);
        const int n = __builtin_amdgcn_readlane(sh.tiles, b), begin = __builtin_amdgcn_readlane(sh.end, b) - (a.hgroups - hg) * n;
        first_share = (int)((uint32_t)begin / (uint32_t)sh.Q);
        parts = (int)((uint32_t)(begin + n - 1) / (uint32_t)sh.Q) - first_share + 1;
    }
    if (parts <= 1) return;   // (the attention wrote its rows)
    auto slot = [&](int x) { return SHARES ? 2 * (first_share + x) + (x == 0) : x; };
    const int i = div_small(r, a.G, a.rcp_g), head = hk * a.G + r - i * a.G;
    const int64_t first = SHARES ? q : (((int64_t)b * a.nblk + blk) * a.hgroups + hg) * a.nsplit * ALL + q;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first;
    const float2* po = reinterpret_cast<const float2*>(a.part_o) + first * (D / 2) + lane;
    merge_parts(parts, a.out + (int64_t)(sq.t0 + i) * a.o_rs + head * D, [&](int s) { return ml[slot(s) * ALL]; },
                [&](int s) { return po[(int64_t)slot(s) * ALL * (D / 2)]; });
}

template <int NB, int KH, int HW, bool SHARES>
hipError_t launch_blocks8(const RangeAttnArgs& a, hipStream_t stream) {
    constexpr int BR = 16 * NB, ALL = BR * HW;
    const int64_t nblk = ((int64_t)a.max_rows * a.G + BR - 1) / BR, merge = nblk * a.hgroups * (ALL / 4);
    const int64_t blocks = SHARES ? a.places : nblk * a.hgroups * a.nsplit, parts = SHARES ? 2 * (int64_t)a.places : a.nsplit;
    // (a block's bytes of parts are counted in 32 bits)
    if (blocks > RANGE_MAX_BLOCKS || merge > 2 * RANGE_MAX_BLOCKS || parts * ALL * D * 4 > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((range8_step_kernel<NB, KH, HW, SHARES>), dim3((unsigned)blocks, SHARES ? 1 : (unsigned)a.B), dim3(64 * KH * HW), 0,
                       stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (!SHARES && a.nsplit == 1) || a.merge_here) return e;
    hipLaunchKernelGGL((range8_merge_kernel<NB, HW, SHARES>), dim3((unsigned)merge, (unsigned)a.B), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_range8(const RangeAttnArgs& a, int br, int kh, int hw, hipStream_t stream) {
    if (a.places) {   // shares
        if (br == 16) return hw == 2 ? launch_blocks8<1, 4, 2, true>(a, stream) : launch_blocks8<1, 4, 1, true>(a, stream);
        return hw == 2 ? launch_blocks8<2, 4, 2, true>(a, stream) : launch_blocks8<2, 4, 1, true>(a, stream);
    }
    if (br == 16) {
        if (hw == 2) return launch_blocks8<1, 2, 2, false>(a, stream);
        return kh == 8 ? launch_blocks8<1, 8, 1, false>(a, stream) : launch_blocks8<1, 4, 1, false>(a, stream);
    }
    return kh == 8 ? launch_blocks8<2, 8, 1, false>(a, stream) : launch_blocks8<2, 4, 1, false>(a, stream);
}

}  // namespace lr
