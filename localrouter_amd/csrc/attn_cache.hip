// Attention of tokens that each see their own range of a sequence's keys (gfx950): windows with first tokens over rows, and
// single tokens, chunks and drafted trees over a cache in pages.
//
//   out_i = sum_{j seen by i} 2^(c <q_i, k_j> - m_i) v_j / sum_{j seen by i} 2^(c <q_i, k_j> - m_i),  c = scale log2(e)
//
// for any reference m_i (it cancels). A token at position p sees j < hi with j >= lo or j < sinks:
//   rows   hi = (p / frame + 1) * frame (at most nkeys), lo = (p / frame - window + 1) * frame
//   pages  hi = p + 1, lo = p - window + 1 (0 without a window); under a tree hi = L, the keys from the first drafted one
//          on are seen where the token's mask has their bit, and p is the context's length plus the bits set less one
// A token that sees nothing gets zeros, and a key that it does not see has no part in it whatever it holds.
//
// The rows of one kv head (tokens x the G query heads that share it) form blocks of 32 RB rows; a workgroup of RB x KG waves
// takes one block and one range of key tiles, its KG groups of RB waves alternate over the tiles. Products, score layout and
// fragments are those of the pipelined kernel (attn_fwd.hip): S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_bf16,
// P in registers, K and V tiles row-major in LDS by direct loads.
#include "lr_common.h"
#include "lr_cache_kernels.h"

namespace lr {

namespace {

#include "attn_common.inc"

#include "range_attn.inc"

template <int RB, int KG, int NS, bool PAGED>
__global__ __launch_bounds__(RB * KG * 64, RB * KG / 4) void range_attn_kernel(RangeAttnArgs a) {
    constexpr int BT = RANGE_TILE, TILE = BT * D, NW = RB * KG;
    constexpr int LOADS = 8 / RB;   // direct loads (4 rows each) per wave per K or V tile
    typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;
    constexpr int RING = KG * NS * TILE * 2 * 2, MERGE = (KG - 1) * RB * (64 * 64 + 2 * 64) * 4;
    __shared__ __attribute__((aligned(1024))) char ring[RING > MERGE ? RING : MERGE];
    __shared__ int staged[PAGED ? RANGE_STAGED : 1];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, hf = lane >> 5;
    const int rb = wave % RB, kg = wave / RB;

    // ---- which rows, which keys
    const int idx = blockIdx.x;
    const int at = div_small(idx, a.nsplit, a.rcp_split), split = idx - at * a.nsplit;
    const int blk = div_small(at, a.HK, a.rcp_hk), hk = at - blk * a.HK;
    const int b = blockIdx.y;
    const Seq sq = seq_of<PAGED>(a, b);
    const int row0 = blk * 32 * RB;
    const int rows = max(sq.n, 0) * a.G;   // (at most 2^30: the host checks)
    if (row0 >= rows) return;
    TileList<BT, PAGED> tl;
    tl.init(a, sq, div_small(row0, a.G, a.rcp_g), div_small(min(rows, row0 + 32 * RB) - 1, a.G, a.rcp_g));
    tl.part(split, a.per);
    const int x0 = tl.x0, x1 = tl.x1;

    // ---- this lane's row
    const int wr0 = row0 + 32 * rb, r = wr0 + n;
    const bool live = r < rows;
    const int rr = min(r, rows - 1), i = div_small(rr, a.G, a.rcp_g), head = hk * a.G + rr - i * a.G;
    const Sees me = sees_of<PAGED>(a, sq, i);
    // tiles that every row of the wave sees whole need no mask
    const int hi_all = PAGED && a.tree ? max(0, min(sq.p0, sq.end)) : wave_min_i(me.hi);
    const int lo_all = wave_max_i(me.lo);

    const int64_t k_rs = PAGED ? a.pg.rs : a.k_rs, v_rs = PAGED ? a.pg.rs : a.v_rs;
    const int64_t hoff = (int64_t)hk * (PAGED ? a.pg.hs : D);
    const bool bad = tl.template stage<NW * 64>(a, b, staged);

    // ---- direct loads of a tile: instruction u fills rows 4u .. 4u + 3, swizzled as attn_fwd.hip's
    const int lrow = lane >> 4, lchunk = lane & 15;
    const uint32_t kr_lds = lds_addr(ring) + kg * NS * TILE * 4, vr_lds = kr_lds + NS * TILE * 2;
    auto load_tile = [&](int x, int slot) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int inst = rb + RB * u, row = 4 * inst + lrow;
            const int64_t o = tl.offset(a, x, row, k_rs);
            dma16(a.k + hoff + o + 8 * (lchunk ^ (row & 15)), kr_lds + 2 * (slot * TILE + 512 * inst));
            const int64_t ov = PAGED ? o : tl.offset(a, x, row, v_rs);
            dma16(a.v + hoff + ov + 8 * (lchunk ^ (lrow << 2)), vr_lds + 2 * (slot * TILE + 512 * inst));
        }
    };

    const int mine = x1 > x0 + kg ? (x1 - x0 - kg + KG - 1) / KG : 0;   // tiles of this group
    const int steps = x1 > x0 ? (x1 - x0 + KG - 1) / KG : 0;             // of group 0: every group's barriers
    auto tile_of = [&](int t) { return x0 + kg + t * KG; };

    bf16x8 qf[8];
    {
        const uint16_t* src = a.q + (int64_t)(sq.t0 + i) * a.q_rs + head * D + 8 * hf;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            u32x4 w = *reinterpret_cast<const u32x4*>(src + 16 * ks);
            if (!live) w = u32x4{0, 0, 0, 0};
            qf[ks] = __builtin_bit_cast(bf16x8, w);
        }
    }
    LR_WAIT_VMCNT(0);
    constexpr int AHEAD = RB == 1 ? NS : NS - 1;   // tiles in flight before the first step
    for (int t = 0; t < AHEAD && t < mine; ++t) load_tile(tile_of(t), t);

    const int pr = key_perm(n);
    const int kswz = pr & 15;
    const int g = lane >> 4, sl = lane & 15;
    int vtr[4];
#pragma unroll
    for (int db = 0; db < 4; ++db) {
        const int chunk = 4 * (db ^ (sl >> 2)) + 2 * (g & 1) + ((sl & 3) >> 1);
        vtr[db] = (8 * (g >> 1) + (sl >> 2)) * D + 8 * chunk + 4 * (sl & 1);
    }

    f32x16 o[4];
#pragma unroll
    for (int db = 0; db < 4; ++db) o[db] = f32x16{};
    float m_used = -INFINITY, l_sum = 0.0f;
    const float c = a.c;
    const bf16x2 ones2 = {(bf16)1.0f, (bf16)1.0f};
    const bool any = wr0 < rows;

    for (int t = 0; t < steps; ++t) {
        const bool have = t < mine;
        // tile t must have landed; of the later ones at most `later` may be in flight
        if (t + AHEAD - 1 < mine && AHEAD > 1) LR_WAIT_VMCNT((AHEAD - 1) * 2 * LOADS);
        else LR_WAIT_VMCNT(0);
        if constexpr (RB > 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this wave's reads of tile t - 1, whose slot is refilled
            block_barrier();
            if (t + NS - 1 < mine) load_tile(tile_of(t + NS - 1), (t + NS - 1) % NS);
        }
        if (have && any) {
            const int x = tile_of(t), key0 = tl.key0(x);
            const uint16_t* kt = reinterpret_cast<const uint16_t*>(ring) + kg * NS * TILE * 2 + (t % NS) * TILE;
            const uint16_t* vt = kt + NS * TILE;
            f32x16 s{};
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kt + pr * D + 8 * ((2 * ks + hf) ^ kswz));
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], s, 0, 0, 0);
            }
            const bool whole = key0 + BT <= hi_all && (key0 >= lo_all || key0 + BT <= a.sinks) && !bad;
            if (!whole) {
                const uint32_t m = seen_bits<BT, PAGED>(a, sq, tl, bad, i, me, x, 0) >> (8 * hf);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(m >> (16 * (e >> 3) + (e & 7)) & 1)) s[e] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
            mx = wave_pair_max(mx) * c;
            if (__builtin_amdgcn_ballot_w64(mx > m_used + RESCALE_TAU)) {
                const float mn = fmaxf(m_used, mx);
                const float alpha = mn > -INFINITY ? __builtin_amdgcn_exp2f(m_used - mn) : 1.0f;
                m_used = mn;
                l_sum *= alpha;
#pragma unroll
                for (int db = 0; db < 4; ++db) o[db] *= alpha;
            }
            // (no key seen so far: the reference is -inf and every score -inf; any finite reference gives P = 0)
            const float nm = m_used > -INFINITY ? -m_used : 0.0f;
            uint32_t pw[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pw[e] = pack_bf16x2(__builtin_amdgcn_exp2f(fmaf(s[2 * e], c, nm)),
                                    __builtin_amdgcn_exp2f(fmaf(s[2 * e + 1], c, nm)));
                l_sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pw[e]), ones2, l_sum, false);
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const bf16x8 pb = __builtin_bit_cast(bf16x8, u32x4{pw[4 * kk], pw[4 * kk + 1], pw[4 * kk + 2], pw[4 * kk + 3]});
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    const uint16_t* p0 = vt + vtr[db] + (16 * kk) * D;
                    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p0);
                    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p0 + 4 * D));
                    const bf16x8 vf = __builtin_shufflevector(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi),
                                                              0, 1, 2, 3, 4, 5, 6, 7);
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pb, o[db], 0, 0, 0);
                }
            }
        }
        if constexpr (RB == 1) {
            // this wave's own slot is free again once its reads have returned
            if (t + NS < mine) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                load_tile(tile_of(t + NS), t % NS);
            }
        }
    }

    // ---- merge the key groups in group 0
    float l = wave_pair_sum(l_sum);
    if constexpr (KG > 1) {
        __syncthreads();
        float* mo = reinterpret_cast<float*>(ring);
        float* mml = mo + (KG - 1) * RB * 64 * 64;
        if (kg > 0) {
            const int at = (kg - 1) * RB + rb;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    *reinterpret_cast<f32x4*>(mo + (at * 16 + 4 * db + q4) * 256 + 4 * lane) =
                        f32x4{o[db][4 * q4], o[db][4 * q4 + 1], o[db][4 * q4 + 2], o[db][4 * q4 + 3]};
            mml[at * 128 + lane] = m_used;
            mml[at * 128 + 64 + lane] = l;
        }
        __syncthreads();
        if (kg > 0) return;
        float ms[KG], mm = m_used;
#pragma unroll
        for (int u = 1; u < KG; ++u) {
            ms[u] = mml[((u - 1) * RB + rb) * 128 + lane];
            mm = fmaxf(mm, ms[u]);
        }
        const float ref = mm > -INFINITY ? mm : 0.0f;
        const float w0 = __builtin_amdgcn_exp2f(m_used - ref);
        l *= w0;
#pragma unroll
        for (int db = 0; db < 4; ++db) o[db] *= w0;
#pragma unroll
        for (int u = 1; u < KG; ++u) {
            const int at = (u - 1) * RB + rb;
            const float w = __builtin_amdgcn_exp2f(ms[u] - ref);
            l = fmaf(w, mml[at * 128 + 64 + lane], l);
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(mo + (at * 16 + 4 * db + q4) * 256 + 4 * lane);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[db][4 * q4 + e] = fmaf(w, x[e], o[db][4 * q4 + e]);
                }
        }
        m_used = mm;
    }
    if (!any) return;

    // ---- rows out: O / l, or this range's part
    float chk = l;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) chk = fmaf(0.0f, o[db][e], chk);
    const bool broken = live && !(fabsf(chk) < INFINITY);
    if (live) {
        if (a.nsplit > 1) {
            const int64_t slot = ((int64_t)(sq.t0 + i) * a.H + head) * a.nsplit + split;
            float* po = a.part_o + slot * D + 4 * hf;
            if (m_used > -INFINITY) {
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4)
                        *reinterpret_cast<f32x4*>(po + 32 * db + 8 * q4) =
                            f32x4{o[db][4 * q4], o[db][4 * q4 + 1], o[db][4 * q4 + 2], o[db][4 * q4 + 3]};
            }
            if (hf == 0) {
                a.part_ml[2 * slot] = m_used;
                a.part_ml[2 * slot + 1] = l;
            }
        } else {
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            uint16_t* dst = a.out + (int64_t)(sq.t0 + i) * a.o_rs + head * D + 4 * hf;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    u32x2 w;
                    w[0] = pack_bf16x2(o[db][4 * q4] * inv, o[db][4 * q4 + 1] * inv);
                    w[1] = pack_bf16x2(o[db][4 * q4 + 2] * inv, o[db][4 * q4 + 3] * inv);
                    *reinterpret_cast<u32x2*>(dst + 32 * db + 8 * q4) = w;
                }
        }
    }

    // rows with an infinity or NaN again, over the seen keys only
    uint64_t again = __builtin_amdgcn_ballot_w64(broken);
    again = (again | again >> 32) & 0xffffffffu;
    while (again) {
        const int src = __builtin_ctzll(again);
        again &= again - 1;
        const int ri = __shfl(i, src, 64), rhead = __shfl(head, src, 64);
        redo_row<BT, PAGED>(a, sq, tl, hk, ri, rhead,
                            a.nsplit > 1 ? ((int64_t)(sq.t0 + ri) * a.H + rhead) * a.nsplit + split : -1);
    }
}

// One wave per (token, head) merges its parts.
template <bool PAGED>
__global__ __launch_bounds__(256) void range_merge_kernel(RangeAttnArgs a) {
    const int at = blockIdx.x * 4 + (threadIdx.x >> 6);
    const Seq sq = seq_of<PAGED>(a, blockIdx.y);
    if (at >= (int64_t)max(sq.n, 0) * a.H) return;
    const int i = at / a.H, head = at - i * a.H;
    const int64_t tok = sq.t0 + i;
    merge_parts(a, (tok * a.H + head) * a.nsplit, a.nsplit, a.out + tok * a.o_rs + head * D);
}

template <int RB, int KG, int NS>
hipError_t launch_blocks(const RangeAttnArgs& a, bool paged, hipStream_t stream) {
    const int64_t rows = (int64_t)(paged ? a.max_rows : a.W) * a.G;
    const int64_t blocks = (rows + 32 * RB - 1) / (32 * RB) * a.HK * a.nsplit;
    if (blocks > 0x7fffffff || rows > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks, (unsigned)(paged ? a.B : 1));
    if (paged) hipLaunchKernelGGL((range_attn_kernel<RB, KG, NS, true>), grid, dim3(RB * KG * 64), 0, stream, a);
    else hipLaunchKernelGGL((range_attn_kernel<RB, KG, NS, false>), grid, dim3(RB * KG * 64), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_range_attn(const RangeAttnArgs& a, bool paged, int wide, hipStream_t stream) {
    if (wide) return launch_range_wide(a, paged, wide, stream);
    const int64_t rows = (int64_t)(paged ? a.max_rows : a.W) * a.G;
    hipError_t e;
    if (rows <= 32) e = launch_blocks<1, 4, 2>(a, paged, stream);
    else if (rows <= 64) e = launch_blocks<2, 2, 4>(a, paged, stream);
    else e = launch_blocks<4, 2, 4>(a, paged, stream);
    if (e != hipSuccess || a.nsplit <= 1) return e;
    const int64_t blocks = ((int64_t)(paged ? a.max_rows : a.W) * a.H + 3) / 4;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks, (unsigned)(paged ? a.B : 1));
    if (paged) hipLaunchKernelGGL(range_merge_kernel<true>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(range_merge_kernel<false>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace lr
