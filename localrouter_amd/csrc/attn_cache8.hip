// Attention over a cache in pages of 8 bits (gfx950): what attn_cache.hip computes over bf16 pages, with
//
//   k_j = 2^e(j) q8_j,  v_j the same: e4m3 rows, a scale for each 16 rows of a page and head (cache8_rows.hip)
//
// for single tokens and small trees: bound by HBM where there is much to read (half of what bf16 pages take), and by the chain
// from one load and one instruction to the next where there is not.
//
// A workgroup is a block of 16 or 32 rows (tokens x the query heads of one kv head) and a part of its tiles of 32 keys, which its
// eight waves take in turn. Keys and values go from memory to registers, not through LDS: a lane's 32 bytes of a key are four steps
// of its products' operand (dims 32 g .. 32 g + 31 of row n for lane 16 g + n; the queries' lanes hold the same dims), and of the
// values it takes 8 dims of the 8 keys whose probabilities it holds, transposed by byte permutations. Conversion to bf16 with the
// scale is one instruction for two values, and exact: e4m3 has 4 significant bits and bf16's exponents.
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

// Lane 16 g + n: row n of each block of 16; of a tile's scores the keys 4 g + r and 16 + 4 g + r (r < 4), in which order its
// products take the keys; of the sums the dims 32 g + 8 r + d, o[d][r].
template <int NB, int KG>
__global__ __launch_bounds__(KG * 64, KG / 4) void range8_step_kernel(RangeAttnArgs a) {
    constexpr int SRC = PAGES8, BT = RANGE_TILE, BR = 16 * NB;
    constexpr int OWN_F = NB * 8 * 256;   // a wave's sums
    __shared__ __attribute__((aligned(1024))) float mo[KG * OWN_F];
    __shared__ float2 mls[KG * NB * 16];
    __shared__ int staged[RANGE_STAGED];

    const int tid = threadIdx.x, lane = tid & 63, kg = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;

    // ---- which rows, which keys
    const int at = div_small(blockIdx.x, a.nsplit, a.rcp_split), split = blockIdx.x - at * a.nsplit;
    const int blk = div_small(at, a.HK, a.rcp_hk), hk = at - blk * a.HK, b = blockIdx.y;
    // without a window a part's entries do not depend on the sequence: they are read beside its numbers
    int early = -1;
    const int per_tile = max(1, BT >> a.pg.shift);
    const bool ahead = !a.window && a.per * per_tile <= KG * 64;
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
    tl.part(split, a.per);
    const int parts = min(a.nsplit, max(1, (tl.total + a.per - 1) / a.per));   // the sequence may be shorter than the longest
    if (split >= parts) return;
    const int x0 = tl.x0, x1 = tl.x1;

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
        const uint16_t* src = a.q + (int64_t)(sq.t0 + ri[nb]) * a.q_rs + head[nb] * D + 32 * g;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[nb][ks] = *reinterpret_cast<const bf16x8*>(src + 8 * ks);
    }
    int hi_all, lo_all, lo_last;
    seen_by_all<SRC>(a, sq, i_first, i_last, me[0], hi_all, lo_all);
    if (NB > 1) {
        seen_by_all<SRC>(a, sq, i_first, i_last, me[NB - 1], hi_all, lo_last);
        lo_all = max(lo_all, lo_last);
    }
    const bool bad = tl.template stage<KG * 64>(a, b, staged, ahead, early);

    const int mine = x1 > x0 + kg ? (x1 - x0 - kg + KG - 1) / KG : 0;   // tiles of this wave
    auto tile_of = [&](int t) { return x0 + kg + t * KG; };
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

    // ---- a tile's two halves of 16 keys: each in one page. Rows past the last key read that one.
    u32x4 kw[2][2];
    u32x2 vw[2][4];
    uint32_t kb[2], vb[2];
    auto half_of = [&](int x, int hb, int64_t& base, int64_t& sc, uint32_t& last) __attribute__((always_inline)) {
        const int k0 = tl.key0(x), j = min(k0 + 16 * hb, (tl.end - 1) & ~15);
        const int page = max(__builtin_amdgcn_readfirstlane(tl.entry(x, j - k0)), 0), r = j & ((1 << tl.shift) - 1);
        base = (int64_t)page * a.pg.ps + (int64_t)r * a.pg.rs;
        sc = (int64_t)page * a.sc_ps + (int64_t)(r >> 4) * a.HK + hk;
        last = (uint32_t)min(15, tl.end - 1 - j);
    };
    auto load_k = [&](int x) __attribute__((always_inline)) {
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
            int64_t base, sc;
            uint32_t last;
            half_of(x, hb, base, sc, last);
            const uint8_t* src = k8 + base + (min((uint32_t)n, last) * rs + 32 * g);
            kw[hb][0] = *reinterpret_cast<const u32x4*>(src);
            kw[hb][1] = *reinterpret_cast<const u32x4*>(src + 16);
            kb[hb] = a.k_sc[sc];
        }
    };
    auto load_v = [&](int x) __attribute__((always_inline)) {
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
            int64_t base, sc;
            uint32_t last;
            half_of(x, hb, base, sc, last);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                vw[hb][r] = *reinterpret_cast<const u32x2*>(v8 + base + (min((uint32_t)(4 * g + r), last) * rs + 8 * n));
            vb[hb] = a.v_sc[sc];
        }
    };
    if (mine > 0) {
        load_k(tile_of(0));
        load_v(tile_of(0));
    }
    for (int t = 0; t < mine; ++t) {
        const int x = tile_of(t), key0 = tl.key0(x);
        f32x4 s[NB][2] = {};
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
            const float sc = scale8(kb[hb]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const bf16x8 kf = widen(kw[hb][ks >> 1][2 * (ks & 1)], kw[hb][ks >> 1][2 * (ks & 1) + 1], sc);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) s[nb][hb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[nb][ks], s[nb][hb], 0, 0, 0);
            }
        }
        if (t + 1 < mine) load_k(tile_of(t + 1));
        const bool whole = key0 + BT <= hi_all && (key0 >= lo_all || key0 + BT <= a.sinks) && !bad;
        u32x4 pw[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            f32x4 &s0 = s[nb][0], &s1 = s[nb][1];
            if (!whole) {
                const uint32_t m = seen_bits<BT, SRC>(a, sq, tl, bad, ri[nb], me[nb], x, 0) >> (4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (!(m >> e & 1)) s0[e] = -INFINITY;
                    if (!(m >> (16 + e) & 1)) s1[e] = -INFINITY;
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
        const float sv0 = scale8(vb[0]), sv1 = scale8(vb[1]);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const u32x4 lo = transpose4(vw[0][0][w], vw[0][1][w], vw[0][2][w], vw[0][3][w]);
            const u32x4 hi = transpose4(vw[1][0][w], vw[1][1][w], vw[1][2][w], vw[1][3][w]);
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
                    o[nb][4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8, pw[nb]), o[nb][4 * w + e], 0, 0, 0);
            }
        }
        if (t + 1 < mine) load_v(tile_of(t + 1));
    }

    // ---- merge the waves: wave u takes the dims 32 g + 4 u .. + 3 from all of them; rows out: O / l, or this part of them
    static_assert(NB <= 2 && KG == 8, "waves");
    const bool whole_block = parts == 1;
    const PartRows<BR> to(a, ((int64_t)b * a.nblk + blk) * a.HK + hk);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        l[nb] = quad_sum(l[nb]);
        if (live[nb]) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {   // dims 32 g + 4 u + e: o[4 (u & 1) + e][u >> 1]
                const f32x4 y = f32x4{o[nb][4 * (u & 1)][u >> 1], o[nb][4 * (u & 1) + 1][u >> 1], o[nb][4 * (u & 1) + 2][u >> 1],
                                      o[nb][4 * (u & 1) + 3][u >> 1]};
                *reinterpret_cast<f32x4*>(mo + kg * OWN_F + (nb * 8 + u) * 256 + 4 * lane) = y;
            }
            if (g == 0) mls[(kg * NB + nb) * 16 + n] = float2{m_used[nb], l[nb]};
        }
    }
    __syncthreads();
    uint32_t broken = 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        bool mine_broken = false;
        if (live[nb]) {
            float mm = -INFINITY, w[KG], sum = 0.0f;
            float2 ml[KG];
#pragma unroll
            for (int u = 0; u < KG; ++u) {
                ml[u] = mls[(u * NB + nb) * 16 + n];
                mm = fmaxf(mm, ml[u].x);
            }
            const float ref = mm > -INFINITY ? mm : 0.0f;
#pragma unroll
            for (int u = 0; u < KG; ++u) {
                w[u] = __builtin_amdgcn_exp2f(ml[u].x - ref);
                sum = fmaf(w[u], ml[u].y, sum);
            }
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            float chk = sum;
            f32x4 own{};
#pragma unroll
            for (int u = 0; u < KG; ++u) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(mo + u * OWN_F + (nb * 8 + kg) * 256 + 4 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) own[e] = fmaf(w[u], y[e], own[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) chk = fmaf(0.0f, own[e], chk);
            const int dim = 32 * g + 4 * kg;
            if (whole_block) {
                u32x2 v;
                v[0] = pack_bf16x2(own[0] * inv, own[1] * inv);
                v[1] = pack_bf16x2(own[2] * inv, own[3] * inv);
                *reinterpret_cast<u32x2*>(a.out + (int64_t)(sq.t0 + ri[nb]) * a.o_rs + head[nb] * D + dim) = v;
            } else {
                to.put4(split, 16 * nb + n, dim, own);
                if (g == 0 && kg == 0) to.put_ml(split, 16 * nb + n, mm, sum);
            }
            mine_broken = !(fabsf(chk) < INFINITY);
        }
        const uint64_t bits = __builtin_amdgcn_ballot_w64(mine_broken);
        const uint32_t half = (uint32_t)(bits | bits >> 32);
        broken |= ((half | half >> 16) & 0xffff) << (16 * nb);
    }
    // ---- rows with an infinity or NaN in some wave's dims again, whole, over the seen keys only
    if (!whole_block) LR_WAIT_VMCNT(0);   // (this wave's part is in memory)
    int* again = reinterpret_cast<int*>(mo);
    again_rows<1, KG>(again, 0, kg, broken, [&](int q) __attribute__((always_inline)) {
        int i = __builtin_amdgcn_readlane(ri[0], q & 15), h = __builtin_amdgcn_readlane(head[0], q & 15);
        if (NB > 1 && q >= 16) {
            i = __builtin_amdgcn_readlane(ri[NB - 1], q & 15);
            h = __builtin_amdgcn_readlane(head[NB - 1], q & 15);
        }
        redo_row<BT, SRC>(a, sq, tl, hk, i, h, [&](float o0, float o1, float m, float rl) {
            if (whole_block) put_row(a.out + (int64_t)(sq.t0 + i) * a.o_rs + h * D, o0, o1, rl);
            else to.put_row2(split, q, o0, o1, m, rl);
        });
    });
    if constexpr (NB == 1)
        if (!whole_block && a.merge_here) to.template merge_last<KG>(a, sq, hk, row0, rows, split, parts, again);
}

template <int BR>
hipError_t launch_blocks8(const RangeAttnArgs& a, void (*kernel)(RangeAttnArgs), hipStream_t stream) {
    const int64_t blocks = ((int64_t)a.max_rows * a.G + BR - 1) / BR * a.HK * a.nsplit, merge = blocks / a.nsplit * (BR / 4);
    // (a block's bytes of parts are counted in 32 bits)
    if (blocks > RANGE_MAX_BLOCKS || merge > 2 * RANGE_MAX_BLOCKS || (int64_t)a.nsplit * BR * D * 4 > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)a.B), dim3(512), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1 || a.merge_here) return e;
    hipLaunchKernelGGL((range_merge_kernel<BR, PAGES8>), dim3((unsigned)merge, (unsigned)a.B), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_range8(const RangeAttnArgs& a, int br, hipStream_t stream) {
    return br == 16 ? launch_blocks8<16>(a, range8_step_kernel<1, 8>, stream) : launch_blocks8<32>(a, range8_step_kernel<2, 8>, stream);
}

}  // namespace lr
