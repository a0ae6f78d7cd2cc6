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

constexpr uint64_t PART_DONE = 0x7ff4a3c57fb5d96e;

template <int RB, int KG, int NS, bool PAGED>
__global__ __launch_bounds__(RB * KG * 64, RB * KG / 4) void range_attn_kernel(RangeAttnArgs a) {
    constexpr int BT = RANGE_TILE, TILE = BT * D, NW = RB * KG;
    constexpr int LOADS = 8 / RB;   // direct loads (4 rows each) per wave per K or V tile
    typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;
    constexpr int RING = KG * NS * TILE * 2 * 2, MERGE = KG * RB * (64 * 64 + 2 * 64) * 4;
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
    const int parts = min(a.nsplit, max(1, (tl.total + a.per - 1) / a.per));   // the sequence may be shorter than the longest
    if (split >= parts) return;
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
    // (the queries first: under pages they arrive while the table's entries are waited for)
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
    const bool bad = tl.template stage<NW * 64>(a, b, staged);

    // ---- direct loads of a tile: instruction u fills rows 4u .. 4u + 3, swizzled as attn_fwd.hip's
    const int lrow = lane >> 4, lchunk = lane & 15;
    const uint32_t kr_lds = lds_addr(ring) + kg * NS * TILE * 4, vr_lds = kr_lds + NS * TILE * 2;
    const bool runs = !PAGED || tl.shift >= 5;   // a whole tile's rows are one run
    auto load_tile = [&](int x, int slot) {
        const int key0 = tl.key0(x);
        const uint16_t *kp = a.k + hoff, *vp = a.v + hoff;
        if (runs && key0 + BT <= sq.end) {
            const int64_t row = (PAGED ? key0 & ((1 << tl.shift) - 1) : key0) + 4 * rb + lrow;
            const int64_t pg = PAGED ? (int64_t)max(tl.entry(x, 0), 0) * a.pg.ps : 0;
            kp += pg + row * k_rs;
            vp += pg + row * v_rs + 8 * (lchunk ^ (lrow << 2));
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const int inst = rb + RB * u;
                dma16(kp + 8 * (lchunk ^ ((4 * inst + lrow) & 15)), kr_lds + 2 * (slot * TILE + 512 * inst));
                dma16(vp, vr_lds + 2 * (slot * TILE + 512 * inst));
                kp += 4 * RB * k_rs;
                vp += 4 * RB * v_rs;
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int inst = rb + RB * u, row = 4 * inst + lrow;
            const int64_t o = tl.offset(a, x, row, k_rs), ov = PAGED ? o : tl.offset(a, x, row, v_rs);
            dma16(kp + o + 8 * (lchunk ^ (row & 15)), kr_lds + 2 * (slot * TILE + 512 * inst));
            dma16(vp + ov + 8 * (lchunk ^ (lrow << 2)), vr_lds + 2 * (slot * TILE + 512 * inst));
        }
    };

    const int mine = x1 > x0 + kg ? (x1 - x0 - kg + KG - 1) / KG : 0;   // tiles of this group
    const int steps = x1 > x0 ? (x1 - x0 + KG - 1) / KG : 0;             // of group 0: every group's barriers
    auto tile_of = [&](int t) { return x0 + kg + t * KG; };

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

    // ---- merge the key groups: group u takes the 32-dim blocks u, u + KG, ... of its rows from all of them
    static_assert(KG > 1 && 4 % KG == 0, "groups");
    constexpr int OWN = 4 / KG;   // blocks a group
    float l = wave_pair_sum(l_sum);
    float own[OWN][16];
    {
        __syncthreads();
        float* mo = reinterpret_cast<float*>(ring);
        float* mml = mo + KG * RB * 64 * 64;
#pragma unroll
        for (int db = 0; db < 4; ++db)
            if (db % KG != kg)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    *reinterpret_cast<f32x4*>(mo + ((kg * RB + rb) * 16 + 4 * db + q4) * 256 + 4 * lane) =
                        f32x4{o[db][4 * q4], o[db][4 * q4 + 1], o[db][4 * q4 + 2], o[db][4 * q4 + 3]};
        *reinterpret_cast<float2*>(mml + (kg * RB + rb) * 128 + 2 * lane) = float2{m_used, l};
        __syncthreads();
        float mm = -INFINITY, w[KG];
        float2 ml[KG];
#pragma unroll
        for (int u = 0; u < KG; ++u) {
            ml[u] = *reinterpret_cast<const float2*>(mml + (u * RB + rb) * 128 + 2 * lane);
            mm = fmaxf(mm, ml[u].x);
        }
        const float ref = mm > -INFINITY ? mm : 0.0f;
        l = 0.0f;
#pragma unroll
        for (int u = 0; u < KG; ++u) {
            w[u] = __builtin_amdgcn_exp2f(ml[u].x - ref);
            l = fmaf(w[u], ml[u].y, l);
        }
        m_used = mm;
        // (in the groups' order, whichever group it is)
#pragma unroll
        for (int x = 0; x < OWN; ++x)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                f32x4 sum{};
#pragma unroll
                for (int u = 0; u < KG; ++u) {
                    f32x4 y;
                    if (u == kg) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            y[e] = 0.0f;
#pragma unroll
                            for (int g2 = 0; g2 < KG; ++g2) y[e] = g2 == kg ? o[g2 + KG * x][4 * q4 + e] : y[e];
                        }
                    } else {
                        y = *reinterpret_cast<const f32x4*>(mo + ((u * RB + rb) * 16 + 4 * (kg + KG * x) + q4) * 256 + 4 * lane);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = fmaf(w[u], y[e], sum[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) own[x][4 * q4 + e] = sum[e];
            }
    }

    // ---- rows out: O / l, or this part of them
    constexpr int BR = 32 * RB;
    const bool whole_block = parts == 1;
    const int64_t block = ((int64_t)b * a.nblk + blk) * a.HK + hk;
    // (sc1: coherent at device scope, not kept in this XCD's L2; the last workgroup of the block may run on another)
    const __amdgpu_buffer_rsrc_t rs_o = __builtin_amdgcn_make_buffer_rsrc(a.part_o + block * a.nsplit * BR * D, 0, a.nsplit * BR * D * 4, 0x00020000);
    const __amdgpu_buffer_rsrc_t rs_ml = __builtin_amdgcn_make_buffer_rsrc(a.part_ml + block * a.nsplit * BR * 2, 0, a.nsplit * BR * 8, 0x00020000);
    auto put_part = [&](int q, float m, float ps) {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(ps)}, rs_ml, (split * BR + q) * 8, 0, 16);
    };
    uint64_t bits = 0;
    // (dims of block x of this group's, quarter q4: 32 (kg + KG x) + 8 q4 + 4 hf .. + 3)
    if (any) {
        float chk = l;
#pragma unroll
        for (int x = 0; x < OWN; ++x)
#pragma unroll
            for (int e = 0; e < 16; ++e) chk = fmaf(0.0f, own[x][e], chk);
        const bool broken = live && !(fabsf(chk) < INFINITY);
        if (live && whole_block) {
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            uint16_t* dst = a.out + (int64_t)(sq.t0 + i) * a.o_rs + head * D + 32 * kg + 4 * hf;
#pragma unroll
            for (int x = 0; x < OWN; ++x)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    u32x2 w;
                    w[0] = pack_bf16x2(own[x][4 * q4] * inv, own[x][4 * q4 + 1] * inv);
                    w[1] = pack_bf16x2(own[x][4 * q4 + 2] * inv, own[x][4 * q4 + 3] * inv);
                    *reinterpret_cast<u32x2*>(dst + 32 * KG * x + 8 * q4) = w;
                }
        } else if (live) {
            const int q = 32 * rb + n;
#pragma unroll
            for (int x = 0; x < OWN; ++x)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const f32x4 y = f32x4{own[x][4 * q4], own[x][4 * q4 + 1], own[x][4 * q4 + 2], own[x][4 * q4 + 3]};
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), rs_o,
                                                           ((split * BR + q) * D + 32 * (kg + KG * x) + 8 * q4 + 4 * hf) * 4, 0, 16);
                }
            if (hf == 0 && kg == 0) put_part(q, m_used, l);
        }
        bits = __builtin_amdgcn_ballot_w64(broken);
    }
    // rows with an infinity or NaN in some group's dims again, whole, over the seen keys only
    int* again = reinterpret_cast<int*>(ring);
    __syncthreads();   // (the merge's reads)
    if (__syncthreads_or(bits != 0)) {
        if (tid < RB) again[tid] = 0;
        LR_WAIT_VMCNT(0);   // (the rows that are overwritten below)
        __syncthreads();
        if (lane == 0) atomicOr(again + rb, (int)(uint32_t)(bits | bits >> 32));
        __syncthreads();
        uint32_t left = (uint32_t)again[rb];
        for (int nth = 0; left; left &= left - 1, ++nth) {
            if (nth % KG != kg) continue;
            const int q = __builtin_amdgcn_readfirstlane(__builtin_ctz(left));
            const int ri = __builtin_amdgcn_readlane(i, q), rhead = __builtin_amdgcn_readlane(head, q);
            redo_row<BT, PAGED>(a, sq, tl, hk, ri, rhead, [&](float o0, float o1, float m, float rl) {
                if (whole_block) {
                    put_row(a.out + (int64_t)(sq.t0 + ri) * a.o_rs + rhead * D, o0, o1, rl);
                } else {
                    __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(o0), __float_as_uint(o1)}, rs_o,
                                                          ((split * BR + 32 * rb + q) * D + 2 * lane) * 4, 0, 16);
                    if (lane == 0) put_part(32 * rb + q, m, rl);
                }
            });
        }
    }
    if (whole_block || !a.merge_here) return;

    // ---- the last of the block's parts to end merges them, in their order. A part whose rows are in memory sets its flag, then
    // reads all of them: the last to set its own sees every one (two that do write the same rows). Flags need no clearing before
    // the call: only PART_DONE counts (as a float or a pair of them a NaN that no arithmetic makes), and who merges clears them.
    LR_WAIT_VMCNT(0);
    __syncthreads();   // every wave's rows are in memory
    if (wave == 0) {   // (alone: a flag set after the merge would outlive the call)
        uint64_t* flags = a.flags + block * a.nsplit;
        if (lane == 0) __hip_atomic_store(flags + split, PART_DONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        LR_WAIT_VMCNT(0);
        bool done = true;
        for (int s0 = 0; s0 < parts; s0 += 64)
            done = done && __hip_atomic_load(flags + min(s0 + lane, parts - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == PART_DONE;
        const bool last = __builtin_amdgcn_ballot_w64(done) == ~0ull;
        if (lane == 0) again[0] = last;
        if (last)
            for (int s0 = lane; s0 < parts; s0 += 64)
                __hip_atomic_store(flags + s0, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!__builtin_amdgcn_readfirstlane(again[0])) return;
    // 16 lanes a row (dims 8 c .. 8 c + 7), four rows a wave, eight parts in flight
    const int mc = lane & 15;
    for (int q0 = 4 * wave; q0 < min(BR, rows - row0); q0 += 4 * NW) {
        const int q = min(q0 + (lane >> 4), rows - row0 - 1);   // (past the last row: that one again, the same)
        float M = -INFINITY, L = 0.0f, sum[8] = {};
        for (int s0 = 0; s0 < parts; s0 += 8) {
            u32x2 ml[8];
            u32x4 x[8][2];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int at = min(s0 + u, parts - 1) * BR + q;
                ml[u] = __builtin_amdgcn_raw_buffer_load_b64(rs_ml, at * 8, 0, 16);
                x[u][0] = __builtin_amdgcn_raw_buffer_load_b128(rs_o, at * D * 4 + 32 * mc, 0, 16);
                x[u][1] = __builtin_amdgcn_raw_buffer_load_b128(rs_o, at * D * 4 + 32 * mc + 16, 0, 16);
            }
            float Mn = M;
#pragma unroll
            for (int u = 0; u < 8; ++u) Mn = fmaxf(Mn, __uint_as_float(ml[u][0]));
            const float ref = Mn > -INFINITY ? Mn : 0.0f, alpha = __builtin_amdgcn_exp2f(M - ref);
            M = Mn;
            L *= alpha;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] *= alpha;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                // a part that saw no key has no weight, whatever is in its row
                const float m = __uint_as_float(ml[u][0]);
                const bool in = m > -INFINITY && s0 + u < parts;
                const float w = __builtin_amdgcn_exp2f(m - ref);
                L = in ? fmaf(w, __uint_as_float(ml[u][1]), L) : L;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] = in ? fmaf(w, __uint_as_float(x[u][e >> 2][e & 3]), sum[e]) : sum[e];
            }
        }
        const int ri = div_small(row0 + q, a.G, a.rcp_g), rhead = hk * a.G + row0 + q - ri * a.G;
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(sum[2 * e] * inv, sum[2 * e + 1] * inv);
        *reinterpret_cast<u32x4*>(a.out + (int64_t)(sq.t0 + ri) * a.o_rs + rhead * D + 8 * mc) = w;
    }
}

// The parts of the blocks that more than one workgroup had, a wave a row: where they are many, one workgroup a block would take
// long (64 parts of 32 rows: ~60 us).
template <int BR, bool PAGED>
__global__ __launch_bounds__(256) void range_merge_kernel(RangeAttnArgs a) {
    const int at = blockIdx.x / (BR / 4), q = blockIdx.x % (BR / 4) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int blk = div_small(at, a.HK, a.rcp_hk), hk = at - blk * a.HK, b = blockIdx.y;
    const Seq sq = seq_of<PAGED>(a, b);
    const int rows = max(sq.n, 0) * a.G, row0 = blk * BR;
    if (row0 + q >= rows) return;
    TileList<RANGE_TILE, PAGED> tl;
    tl.init(a, sq, div_small(row0, a.G, a.rcp_g), div_small(min(rows, row0 + BR) - 1, a.G, a.rcp_g));
    const int parts = min(a.nsplit, (tl.total + a.per - 1) / a.per);
    if (parts <= 1) return;   // (the attention wrote its rows)
    const int i = div_small(row0 + q, a.G, a.rcp_g), head = hk * a.G + row0 + q - i * a.G;
    const int64_t first = (((int64_t)b * a.nblk + blk) * a.HK + hk) * a.nsplit * BR + q;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first;
    const float2* po = reinterpret_cast<const float2*>(a.part_o) + first * (D / 2) + lane;
    merge_parts(parts, a.out + (int64_t)(sq.t0 + i) * a.o_rs + head * D, [&](int s) { return ml[s * BR]; },
                [&](int s) { return po[(int64_t)s * BR * (D / 2)]; });
}

template <int RB, int KG, int NS>
hipError_t launch_blocks(const RangeAttnArgs& a, bool paged, hipStream_t stream) {
    const int64_t rows = (int64_t)(paged ? a.max_rows : a.W) * a.G;
    const int64_t blocks = (rows + 32 * RB - 1) / (32 * RB) * a.HK * a.nsplit;
    // (a grid's work-items and a block's bytes of parts are counted in 32 bits)
    if (blocks > 1 << 22 || blocks / a.nsplit * 8 * RB > 1 << 23 || (int64_t)a.nsplit * 32 * RB * D * 4 > INT32_MAX)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks, (unsigned)(paged ? a.B : 1));
    if (paged) hipLaunchKernelGGL((range_attn_kernel<RB, KG, NS, true>), grid, dim3(RB * KG * 64), 0, stream, a);
    else hipLaunchKernelGGL((range_attn_kernel<RB, KG, NS, false>), grid, dim3(RB * KG * 64), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1 || a.merge_here) return e;
    const dim3 merge((unsigned)(blocks / a.nsplit * (8 * RB)), grid.y);
    if (paged) hipLaunchKernelGGL((range_merge_kernel<32 * RB, true>), merge, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((range_merge_kernel<32 * RB, false>), merge, dim3(256), 0, stream, a);
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
    return e;
}

}  // namespace lr
