// Causal attention over prompts packed end to end (gfx950), where there is enough of it for matrix products to bound it: sequence b is
// the rows starts[b] .. starts[b + 1] of q, k, v and out; its token i sees its tokens j <= i, with a window those of i - j < window
// and j < sinks.
//
//   out_i = sum_{j seen by i} 2^(c <q_i, k_j> - m_i) v_j / sum_{j seen by i} 2^(c <q_i, k_j> - m_i),  c = scale log2(e)
//
// P is rounded to bf16, which the products take, and the row's sum is that of the rounded P, so that the weights add up to 1; sums and
// references are fp32. (Error against 64 bits, relative L2: 0.0017 to 0.0021; the output's own rounding alone 0.0016.)
//
// The inner loop is that of attn_cache_wide.hip: a half-step of 16 MFMA slots runs the next half-tile's scores, the previous one's
// products and this one's exponentials, over a ring of two key tiles and two value tiles that direct loads fill. What differs is what
// a batch of prompts needs: its blocks of rows are short (a prompt of 600 tokens has blocks of one to ten key tiles), so that starting
// and ending one costs as much as its products. Here a workgroup stays and takes one block after the other, and the ring runs on
// across them: the next block's first tiles and queries are on their way while the last tile's products are computed and the rows
// written.
//
// Blocks of up to 64 sequences are ordered by the number that they have in their sequence, the last first (without a window that is by
// their tiles, most first), and dealt to the workgroups in turn, each second round in the opposite order, so that all have about as
// much; those of more sequences go out in the sequences' order. A head's blocks go to the workgroups of one XCD (of a number of kv heads
// that 8 divides), whose L2 then holds its keys and values.
//
// What bounds it: of long prompts the clock under the power limit (4 of up to 7,000 tokens, 32 heads over 4, 500 to 530 us, 1,020 TFLOP/s; under the
// profiler 1.78 GHz, MFMA busy 50 %). Of short ones what a block takes beside its tiles, ~800 vector instructions a wave (its masks and
// references, zeros, queries and rows out): 1.75 us a tile and ~5 a block (19 of up to 1,100, 32 over 8: 119 us, 640 TFLOP/s; with a
// workgroup for each block 135). Of captions the two rounds of loads from HBM (40 of up to 257, 16 over 16, 93 MB: 33 us).
#include "lr_common.h"
#include "lr_cache_kernels.h"
#include "tile_image.h"

namespace lr {

namespace {

#include "attn_common.inc"

constexpr int RA = 3;             // fragments read ahead
constexpr int FR = 4;             // fragment ring entries

#include "attn_tiles.inc"
#include "raise_rows.inc"
#include "dma1.inc"
#include "range_attn.inc"

// What every lane has the same of, known as such.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(const void* p) {
    const uint64_t x = (uint64_t)(uintptr_t)p;
    return (uint64_t)(uint32_t)uniform((int)(uint32_t)x) | (uint64_t)(uint32_t)uniform((int)(uint32_t)(x >> 32)) << 32;
}

// A block of rows of one sequence and kv head.
struct Block {
    Seq sq;
    int hk, row0, rows;
    TileList<IMG_TILE_KEYS, PACKED> tl;
};

template <int QW>
__global__ __launch_bounds__(64 * QW, 8 / QW) __attribute__((amdgpu_waves_per_eu(2, 2))) void packed_kernel(RangeAttnArgs a) {
    constexpr int SRC = PACKED, KBM = 32 * QW, LP = 16 / QW, BT = IMG_TILE_KEYS;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * IMG_TILE_BYTES];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, hf = lane >> 5;

    // ---- which blocks: those of ranks w, 2 W - 1 - w, 2 W + w, .. (an XCD's with each other: workgroup w runs on XCD w % 8)
    const int W = gridDim.x, ids = a.nsplit * a.HK;   // (nsplit: the most blocks of a kv head)
    int above = a.nblk;
    PackedBlocks<KBM> pb;
    pb.init(a);
    auto next_block = [&](int& round, Block& to) __attribute__((always_inline)) {
        for (;; ++round) {
            const int w = blockIdx.x, at = (round & 1) && (W & 7) == 0 ? W - 8 - (w & ~7) + (w & 7) : w;
            if ((int64_t)round * W >= ids) return false;
            const int id = round * W + at;
            if (id >= ids) continue;
            const int u = div_small(id, a.HK, a.rcp_hk);
            int blk;
            if (!pb.at(a, u, above, to.sq, blk)) continue;
            blk = uniform(blk);
            if (a.B <= 64) above = blk + 1;   // (ranks go on with blocks of no higher number)
            to.hk = id - u * a.HK;
            to.row0 = blk * KBM;
            to.rows = to.sq.n * a.G;
            if (to.row0 >= to.rows) continue;
            to.tl.init(a, to.sq, div_small(to.row0, a.G, a.rcp_g), div_small(min(to.rows, to.row0 + KBM) - 1, a.G, a.rcp_g));
            return true;
        }
    };
    Block cur, nxt;
    int round = 0;
    if (!next_block(round, cur)) return;

    // ---- direct loads, as attn_cache_wide.hip's over rows: of a key tile the 32 rows of block 2 wv / QW, LP fragments of them; of a
    // value tile the rows 16 (4 wv / QW) .. in the row-block layout. Rows past the last key read that one.
    const uint32_t krowb = (uint32_t)a.k_rs * 2u, rowb = (uint32_t)a.v_rs * 2u;   // (below 2^24: the host checks)
    const uint32_t ring = lds_addr(lds), vring = ring + 2 * IMG_TILE_BYTES;
    const uint32_t lane16 = (uint32_t)lane * 16u;
    const uint32_t krow = (uint32_t)img_key_perm(n), kcol = (uint32_t)(32 * LP * (wv % (QW / 2)) + 16 * hf);
    const uint32_t vrow = (uint32_t)(vt_lane_row(lane) + 4 * LP * wv % 16), vchunk = (uint32_t)(16 * vt_lane_chunk(lane));
    const int vg = 16 * (4 * wv / QW), kg = 32 * (2 * wv / QW);
    uint32_t ko = 0;
    int vlast = 15;
    auto k_src = [&](const Block& b, int x) __attribute__((always_inline)) {
        const int j = min(b.tl.key0(x) + kg, (b.tl.end - 1) & -32);
        ko = __umul24(min(krow, (uint32_t)(min(32, b.tl.end - j) - 1)), krowb) + kcol;
        return uniform(a.k + (int64_t)(b.tl.row0 + j) * a.k_rs + b.hk * D);
    };
    auto v_src = [&](const Block& b, int x) __attribute__((always_inline)) {
        const int j = min(b.tl.key0(x) + vg, (b.tl.end - 1) & -16);
        vlast = min(16, b.tl.end - j) - 1;
        return uniform(a.v + (int64_t)(b.tl.row0 + j) * a.v_rs + b.hk * D);
    };
    auto load_k1 = [&](uint64_t src, uint32_t dst, int u) __attribute__((always_inline)) {
        const uint32_t to = (uint32_t)uniform((int)(dst + (uint32_t)(1024 * (LP * wv + u))));
        if (u == 0) dma1_at<0>(src, ko, to);
        else if (u == 1) dma1_at<32>(src, ko, to);
        else if (u == 2) dma1_at<64>(src, ko, to);
        else dma1_at<96>(src, ko, to);
    };
    auto load_v1 = [&](uint64_t src, uint32_t dst, int u) __attribute__((always_inline)) {
        dma1_at<0>(src, __umul24(min(vrow + 4 * u, (uint32_t)vlast), rowb) + vchunk,
                   (uint32_t)uniform((int)(dst + (uint32_t)(1024 * (LP * wv + u)))));
    };
    auto load_k = [&](const Block& b, int x, uint32_t dst) __attribute__((always_inline)) {
        const uint64_t src = k_src(b, x);
#pragma unroll
        for (int u = 0; u < LP; ++u) load_k1(src, dst, u);
    };
    auto load_v = [&](const Block& b, int x, uint32_t dst) __attribute__((always_inline)) {
        const uint64_t src = v_src(b, x);
#pragma unroll
        for (int u = 0; u < LP; ++u) load_v1(src, dst, u);
    };
    auto slot = [](int x) __attribute__((always_inline)) { return (uint32_t)((x & 1) * IMG_TILE_BYTES); };

    // ---- registers (as the key-split kernel's)
    bf16x8 qa[8];
    f32x16 o[4], s[2], negm;
    u32x4 p[2][2];
    float ls = 0.0f;
    bf16x8 fr[FR];
    const uint32_t vlane = (uint32_t)vt_lane(lane);
    auto vfrag_off = [](int x) __attribute__((always_inline)) { return 4096 * (x >> 2) + 256 * (x & 3); };
    auto load_q = [&](const Block& b) __attribute__((always_inline)) {
        const int rr = min(b.row0 + 32 * wv + n, b.rows - 1), i = div_small(rr, a.G, a.rcp_g), head = b.hk * a.G + rr - i * a.G;
        const uint16_t* src = a.q + (int64_t)(b.sq.t0 + i) * a.q_rs + head * D + 8 * hf;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qa[ks] = *reinterpret_cast<const bf16x8*>(src + 16 * ks);
    };
    const float c = a.c;
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

    // tile u of the block lies in the slots of ring place `at` + u
    int at = 0;
    load_k(cur, 0, ring + slot(0));
    load_q(cur);
    load_v(cur, 0, vring + slot(0));
    if (cur.tl.total > 1) load_k(cur, 1, ring + slot(1));
    LR_WAIT_VMCNT(0);
    block_barrier();

    for (;;) {
        ++round;
        const bool more = next_block(round, nxt);
        const int nsteps = cur.tl.total, wr0 = cur.row0 + 32 * wv;
        const bool idle = wr0 >= cur.rows;   // (a wave without rows only loads)
        const int rr = min(wr0 + n, cur.rows - 1), i = div_small(rr, a.G, a.rcp_g), head = cur.hk * a.G + rr - i * a.G;
        const bool live = wr0 + n < cur.rows;
        const Sees me = sees_of<SRC>(a, cur.sq, i);
        // half-tiles (h = 2 x + half) that every row of the wave sees whole need no mask: h < free_s among the first tokens',
        // free_lo <= h < free_hi of the rows' own range
        const int hi_all = sees_of<SRC>(a, cur.sq, div_small(min(wr0, cur.rows - 1), a.G, a.rcp_g)).hi;
        const int lo_all = sees_of<SRC>(a, cur.sq, div_small(min(wr0 + 31, cur.rows - 1), a.G, a.rcp_g)).lo;
        const int skip = 2 * (cur.tl.lt - cur.tl.st);
        const int free_s = min(2 * cur.tl.st, min(a.sinks, hi_all) / 32);
        const int free_lo = max(2 * cur.tl.st, (lo_all + 31) / 32 - skip), free_hi = hi_all / 32 - skip;

        // a step's refills, one load every other slot of its first half: V(t), then K(t + 1), of the last tile the next block's first
        // (or once more its own, never read)
        uint64_t src = 0;
        auto refill = [&](int f, int t) __attribute__((always_inline)) {
            if (f == 0) src = v_src(cur, t);
            if (f == 2 * LP) {
                if (t + 1 < nsteps) src = k_src(cur, t + 1);
                else if (more) src = k_src(nxt, 0);
                else src = k_src(cur, t);
            }
            if (f % 2 == 1) {
                if (f / 2 < LP) load_v1(src, vring + slot(at + t), f / 2);
                else if (f / 2 < 2 * LP) load_k1(src, ring + slot(at + t + 1), f / 2 - LP);
            }
        };
        // behind the last step: the next block's first values and second keys
        auto lead = [&]() __attribute__((always_inline)) {
            if (!more) return;
            load_v(nxt, 0, vring + slot(at + nsteps));
            if (nxt.tl.total > 1) load_k(nxt, 1, ring + slot(at + nsteps + 1));
        };

        if (idle) {
            if (nsteps == 1 && more) load_k(nxt, 0, ring + slot(at + 1));
            for (int u = 0;; ++u) {
                LR_WAIT_VMCNT(0);
                block_barrier();
                if (u + 1 >= nsteps) break;
#pragma unroll
                for (int f = 0; f < 4 * LP; ++f) refill(f, u + 1);
            }
            lead();
            if (!more) return;
            load_q(nxt);
        } else {
            // ---- masked half-tiles: what the row does not see out, and a reference for the rows that have none yet
            bool set = !live;
            bool unset_any = true;
            auto special = [&](int x, int half) __attribute__((always_inline)) {
                const int h = 2 * x + half;
                return unset_any || !(h < free_s || (h >= free_lo && h < free_hi));
            };
            auto mask_half = [&](f32x16& sb, int x, int half) __attribute__((always_inline)) {
                const uint32_t m = seen_bits<BT, SRC>(a, cur.sq, cur.tl, false, i, me, x, 32 * half) >> (8 * hf);
#pragma unroll
                for (int q = 0; q < 16; ++q) sb[q] = if_seen(sb[q], m, 16 * (q >> 3) + (q & 7));
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
                    asm volatile(LR_NOP48 : "+v"(negm));
                    // rows that see nothing further on need none
                    const int next = cur.tl.key0(x) + 32 * half + 32;
                    unset_any = __builtin_amdgcn_ballot_w64(!set && me.hi > next) != 0;
                }
            };
            ls = 0.0f;
#pragma unroll
            for (int db = 0; db < 4; ++db) o[db] = f32x16{};
            negm = f32x16{};
            if (nsteps == 1 && more) load_k(nxt, 0, ring + slot(at + 1));
            {
                uint32_t kb0 = ring + slot(at) + lane16;
                asm volatile("" : "+v"(kb0));
                fence_q8(qa);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const bf16x8 kf = frag_at(kb0 + (uint32_t)(ks * IMG_FRAG_BYTES));
                    if (ks == 0) qk_zero(s[0], kf, qa[0]);
                    else qk_acc(s[0], kf, qa[ks]);
                }
                fence_s(s[0]);
                mask_half(s[0], 0, 0);
            }
            // ---- step 0: S of half-tile 1 (K(0), fragments 8-15), P of half-tile 0
            {
                uint32_t kb = ring + slot(at) + lane16;
                asm volatile("" : "+v"(kb));
                auto rd0 = [&](int f) __attribute__((always_inline)) {
                    if (f < 8) fr[f % FR] = frag_at(kb + (8 + f) * IMG_FRAG_BYTES);
                };
#pragma unroll
                for (int f = 0; f < RA; ++f) rd0(f);
                half_step(s[1], p[1], s[0], p[0], BoolTag<false>{}, [&](int f) __attribute__((always_inline)) { rd0(f); });
                LR_WAIT_VMCNT(0);
                block_barrier();
            }
            // ---- step u: key tile u (both halves), value tile u - 1. Its refills go to the slots of V(u - 2) and K(u - 1), both
            // read before the last barrier, and have landed at the end of step u.
            for (int u = 1; u < nsteps; ++u) {
                raise_rows(c, ls, o, p[0], s[1], negm);
                uint32_t kb = ring + slot(at + u) + lane16, vb = vring + slot(at + u - 1) + vlane;
                asm volatile("" : "+v"(kb), "+v"(vb));
                auto rd_b = [&](int f) __attribute__((always_inline)) {
                    if (f < 8) fr[f % FR] = frag_at(kb + f * IMG_FRAG_BYTES);
                    else if (f < 16) fr[f % FR] = vfrag_at(vb + vfrag_off(f - 8));
                    else fr[f % FR] = frag_at(kb + (f - 8) * IMG_FRAG_BYTES);
                };
                auto rd_a = [&](int f) __attribute__((always_inline)) {
                    if (f < 8) fr[f % FR] = frag_at(kb + (8 + f) * IMG_FRAG_BYTES);
                    else if (f < 16) fr[f % FR] = vfrag_at(vb + vfrag_off(f));
                };
#pragma unroll
                for (int f = 0; f < RA; ++f) rd_b(f);
                if (special(u - 1, 1)) mask_half(s[1], u - 1, 1);
                half_step(s[0], p[0], s[1], p[1], BoolTag<true>{}, [&](int f) __attribute__((always_inline)) {
                    refill(f - RA, u);
                    rd_b(f);
                });
                if (special(u, 0)) mask_half(s[0], u, 0);
                half_step(s[1], p[1], s[0], p[0], BoolTag<true>{}, rd_a);
                LR_WAIT_VMCNT(0);
                block_barrier();
            }
            // ---- the last half-tile's P and the last value tile's products; the next block's loads beside them
            lead();
            if (more) load_q(nxt);
            {
                raise_rows(c, ls, o, p[0], s[1], negm);
                const int u = nsteps - 1;
                if (special(u, 1)) mask_half(s[1], u, 1);
                uint32_t vb0 = vring + slot(at + u) + vlane;
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
            // 8 dims a store: the lower lanes take both halves' words of the even 8-dim groups, the upper lanes of the odd ones
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            uint16_t* dst = a.out + (int64_t)(cur.sq.t0 + i) * a.o_rs + head * D + 8 * hf;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t w[2][2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int from = 4 * (2 * x + e);
                        w[e][0] = pack_bf16x2(o[db][from] * inv, o[db][from + 1] * inv);
                        w[e][1] = pack_bf16x2(o[db][from + 2] * inv, o[db][from + 3] * inv);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        nan = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w[e >> 1][e & 1]), bf16x2{}, nan, false);
                    const auto r0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
                    const auto r1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
                    if (live) *reinterpret_cast<u32x4*>(dst + 32 * db + 16 * x) = u32x4{r0[0], r1[0], r0[1], r1[1]};
                }
            uint64_t again = __builtin_amdgcn_ballot_w64(nan != 0.0f && live);
            again = (again | again >> 32) & 0xffffffffu;
            while (again) {
                const int q = __builtin_ctzll(again);
                again &= again - 1;
                const int ri = __builtin_amdgcn_readlane(i, q), rhead = __builtin_amdgcn_readlane(head, q);
                redo_row<BT, SRC>(a, cur.sq, cur.tl, cur.hk, ri, rhead, [&](float o0, float o1, float, float rl) {
                    put_row(a.out + (int64_t)(cur.sq.t0 + ri) * a.o_rs + rhead * D, o0, o1, rl);
                });
            }
            if (!more) return;
        }
        at += nsteps;
        cur = nxt;
    }
}

}  // namespace

hipError_t launch_packed_wide(const RangeAttnArgs& a, int waves, hipStream_t stream) {
    RangeAttnArgs b = a;
    b.nsplit = (int)((int64_t)a.T * a.G / (32 * waves)) + a.B;
    const int64_t blocks = (int64_t)b.nsplit * a.HK;
    if (blocks > 1 << 30) return hipErrorInvalidValue;   // (ranks are counted in 32 bits)
    const unsigned grid = (unsigned)(blocks < 2048 / waves ? blocks : 2048 / waves);
    if (waves == 8) hipLaunchKernelGGL(packed_kernel<8>, dim3(grid), dim3(512), 0, stream, b);
    else hipLaunchKernelGGL(packed_kernel<4>, dim3(grid), dim3(256), 0, stream, b);
    return hipGetLastError();
}

}  // namespace lr
