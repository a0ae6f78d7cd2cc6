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

// What a token of a sequence sees.
struct Sees {
    int lo, hi;   // keys lo <= j < hi, and j < min(sinks, lo)
};

// One sequence of a call as a workgroup needs it.
struct Seq {
    int t0, n;        // first token, tokens
    int p0;           // position of the first token (the first drafted key under a tree)
    int end;          // keys that exist
};

template <bool PAGED>
__device__ __forceinline__ Seq seq_of(const RangeAttnArgs& a, int b) {
    Seq s;
    if constexpr (PAGED) {
        const int s0 = a.starts[b], s1 = a.starts[b + 1], len = a.lens[b];
        s.t0 = max(0, s0);
        s.n = min(min(s1, a.T) - s.t0, a.max_rows);
        // a first token that the call does not have, or more keys than an int's tokens: nothing is done for it
        if (s0 < 0 || len < 0) s.n = 0;
        s.p0 = len - (s1 - s0);
        const int64_t cap = (int64_t)a.pg.table_pages << a.pg.shift;
        s.end = (int)min((int64_t)min(len, a.max_keys), cap);
    } else {
        s.t0 = 0;
        s.n = a.W;
        s.p0 = a.p0;
        s.end = a.nkeys;
    }
    return s;
}

template <bool PAGED>
__device__ __forceinline__ Sees sees_of(const RangeAttnArgs& a, const Seq& s, int i) {
    Sees r;
    if constexpr (PAGED) {
        int p = s.p0 + i;
        r.hi = min(s.end, p + 1);
        if (a.tree) {
            int bits = 0;
            for (int w = 0; w < a.words; ++w) bits += __popcll(a.tree[(int64_t)(s.t0 + i) * a.words + w]);
            p = s.p0 + bits - 1;
            r.hi = s.end;
        }
        r.lo = a.window ? max(0, p - a.window + 1) : 0;
    } else {
        const int f = (s.p0 + i) / a.frame;
        r.hi = (int)min((int64_t)s.end, ((int64_t)f + 1) * a.frame);
        r.lo = (int)max((int64_t)0, ((int64_t)f - a.window + 1) * a.frame);
    }
    r.hi = max(r.hi, 0);
    r.lo = min(r.lo, r.hi);
    return r;
}

__device__ __forceinline__ int wave_max_i(int x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x = max(x, __shfl_xor(x, d, 64));
    return x;
}
__device__ __forceinline__ int wave_min_i(int x) { return -wave_max_i(-x); }

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
    int idx = blockIdx.x;
    const int split = idx % a.nsplit;
    idx /= a.nsplit;
    const int hk = idx % a.HK;
    const int b = blockIdx.y;
    const int blk = idx / a.HK;
    const Seq sq = seq_of<PAGED>(a, b);
    const int row0 = blk * 32 * RB;
    const int64_t rows = (int64_t)max(sq.n, 0) * a.G;
    if (row0 >= rows) return;
    const int i_first = row0 / a.G, i_last = (int)min((int64_t)sq.n - 1, ((int64_t)row0 + 32 * RB - 1) / a.G);
    int lo_min, hi_max;
    if (PAGED && a.tree) {
        lo_min = a.window ? max(0, min(sq.p0 - a.window, sq.end)) : 0;
        hi_max = max(sq.end, 0);
    } else {
        lo_min = sees_of<PAGED>(a, sq, i_first).lo;
        hi_max = sees_of<PAGED>(a, sq, i_last).hi;
    }
    const int st = (min(a.sinks, lo_min) + BT - 1) / BT;            // tiles of first tokens
    const int lt = max(st, lo_min / BT), ht = (hi_max + BT - 1) / BT;
    const int total = st + max(0, ht - lt);
    const int x0 = split * a.tiles_per_split, x1 = min(total, x0 + a.tiles_per_split);
    auto key0_of = [&](int x) { return BT * (x < st ? x : lt + x - st); };

    // ---- this lane's row
    const int wr0 = row0 + 32 * rb, r = wr0 + n;
    const bool live = r < rows;
    const int i = min(r, (int)rows - 1) / a.G, head = hk * a.G + min(r, (int)rows - 1) % a.G;
    const Sees me = sees_of<PAGED>(a, sq, i);
    // tiles that every row of the wave sees whole need no mask
    const int hi_all = PAGED && a.tree ? max(0, min(sq.p0, sq.end)) : wave_min_i(me.hi);
    const int lo_all = wave_max_i(me.lo);

    const int64_t k_rs = PAGED ? a.pg.rs : a.k_rs, v_rs = PAGED ? a.pg.rs : a.v_rs;
    const int64_t hoff = (int64_t)hk * (PAGED ? a.pg.hs : D);
    const int shift = PAGED ? a.pg.shift : 0;
    const int per_tile = PAGED ? max(1, BT >> shift) : 1;
    bool bad = false;
    if constexpr (PAGED) {
        const int cnt = max(0, x1 - x0) * per_tile;
        for (int e = tid; e < cnt; e += NW * 64) {
            const int j = key0_of(x0 + e / per_tile) + (e % per_tile << shift);
            int page = -1;
            if (j < sq.end) {
                page = a.pg.table[(int64_t)b * a.pg.table_rs + (j >> shift)];
                if (page < 0 || page >= a.pg.n_pages) page = -1;
                bad |= page < 0;
            }
            staged[e] = page;
        }
        bad = __syncthreads_or(bad);
    }
    // row `row` of tile x: its key clamped to the last that exists, and its offset in elements from the head's first
    auto entry = [&](int x, int row) { return PAGED ? staged[(x - x0) * per_tile + (per_tile > 1 ? row >> shift : 0)] : 0; };
    auto offset = [&](int x, int row, int64_t rs) -> int64_t {
        const int key0 = key0_of(x);
        const int j = min(key0 + row, sq.end - 1);
        if constexpr (PAGED)
            return (int64_t)max(entry(x, j - key0), 0) * a.pg.ps + (int64_t)(j & ((1 << shift) - 1)) * rs;
        else
            return (int64_t)j * rs;
    };

    // ---- direct loads of a tile: instruction u fills rows 4u .. 4u + 3, swizzled as attn_fwd.hip's
    const int lrow = lane >> 4, lchunk = lane & 15;
    const uint32_t kr_lds = lds_addr(ring) + kg * NS * TILE * 4, vr_lds = kr_lds + NS * TILE * 2;
    auto load_tile = [&](int x, int slot) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int inst = rb + RB * u, row = 4 * inst + lrow;
            const int64_t o = offset(x, row, k_rs);
            dma16(a.k + hoff + o + 8 * (lchunk ^ (row & 15)), kr_lds + 2 * (slot * TILE + 512 * inst));
            const int64_t ov = PAGED ? o : offset(x, row, v_rs);
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

    // whether this lane's row sees key j = key0 + row of tile x
    auto sees = [&](int x, int key0, int row) {
        const int j = key0 + row;
        bool ok = j < me.hi && (j >= me.lo || j < a.sinks);
        if constexpr (PAGED) {
            if (a.tree && j >= sq.p0) {
                const int d = j - sq.p0;
                ok = j < sq.end && (d >> 6) < a.words && (a.tree[(int64_t)(sq.t0 + i) * a.words + (d >> 6)] >> (d & 63) & 1);
            }
            if (bad && ok) ok = entry(x, row) >= 0;
        }
        return ok;
    };

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
            const int x = tile_of(t), key0 = key0_of(x);
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
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = 16 * (e >> 3) + 8 * hf + (e & 7);
                    if (!sees(x, key0, row)) s[e] = -INFINITY;
                }
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

    // ---- rows with an infinity or NaN: zero times it may have come from a key that the row does not see (0 * NaN in the
    // products). Those rows again, key by key over the seen ones only: lane = key for the scores, lane = two dims for the sum.
    uint64_t again = __builtin_amdgcn_ballot_w64(broken);
    again = (again | again >> 32) & 0xffffffffu;
    while (again) {
        const int src = __builtin_ctzll(again);
        again &= again - 1;
        const int ri = __shfl(i, src, 64), rhead = __shfl(head, src, 64);
        const uint16_t* qrow = a.q + (int64_t)(sq.t0 + ri) * a.q_rs + rhead * D;
        float m = -INFINITY, ls = 0.0f, o0 = 0.0f, o1 = 0.0f;
        const Sees rs_ = sees_of<PAGED>(a, sq, ri);
        for (int x = x0; x < x1; ++x) {
            const int key0 = key0_of(x), j = key0 + n;
            bool ok = j < rs_.hi && (j >= rs_.lo || j < a.sinks);
            if constexpr (PAGED) {
                if (a.tree && j >= sq.p0) {
                    const int d = j - sq.p0;
                    ok = j < sq.end && (d >> 6) < a.words &&
                         (a.tree[(int64_t)(sq.t0 + ri) * a.words + (d >> 6)] >> (d & 63) & 1);
                }
                if (ok) ok = entry(x, n) >= 0;
            }
            ok = ok && hf == 0;
            float s = -INFINITY;
            if (ok) {
                const uint16_t* kr = a.k + hoff + offset(x, n, k_rs);
                s = 0.0f;
                for (int d = 0; d < D; d += 8) {
                    const u32x4 kw = *reinterpret_cast<const u32x4*>(kr + d), qw = *reinterpret_cast<const u32x4*>(qrow + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s = fmaf(lo_bf16(kw[e]), lo_bf16(qw[e]), s);
                        s = fmaf(hi_bf16(kw[e]), hi_bf16(qw[e]), s);
                    }
                }
                s *= c;
            }
            float mx = s;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
            const float mn = fmaxf(m, mx), ref = mn > -INFINITY ? mn : 0.0f;
            const float alpha = m > -INFINITY ? __builtin_amdgcn_exp2f(m - ref) : 1.0f;
            m = mn;
            const float p = ok ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
            ls = ls * alpha + p;   // (per lane: summed at the end)
            o0 *= alpha;
            o1 *= alpha;
            uint64_t seen = __builtin_amdgcn_ballot_w64(ok);
            while (seen) {
                const int kk = __builtin_ctzll(seen);
                seen &= seen - 1;
                const float pk = __shfl(p, kk, 64);
                const uint32_t vw = *reinterpret_cast<const uint32_t*>(a.v + hoff + offset(x, kk, v_rs) + 2 * lane);
                o0 = fmaf(pk, lo_bf16(vw), o0);
                o1 = fmaf(pk, hi_bf16(vw), o1);
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) ls += __shfl_xor(ls, d, 64);
        if (a.nsplit > 1) {
            const int64_t slot = ((int64_t)(sq.t0 + ri) * a.H + rhead) * a.nsplit + split;
            *reinterpret_cast<float2*>(a.part_o + slot * D + 2 * lane) = float2{o0, o1};
            if (lane == 0) {
                // (a range whose sum is NaN counts whatever its reference)
                a.part_ml[2 * slot] = m > -INFINITY || ls == 0.0f ? m : 0.0f;
                a.part_ml[2 * slot + 1] = ls;
            }
        } else {
            const float inv = ls != 0.0f ? 1.0f / ls : 0.0f;
            *reinterpret_cast<uint32_t*>(a.out + (int64_t)(sq.t0 + ri) * a.o_rs + rhead * D + 2 * lane) =
                pack_bf16x2(o0 * inv, o1 * inv);
        }
    }
}

// One wave per (token, head): the ranges' parts merged, two dims a lane. A range that saw no key (reference -inf) has left its
// row unwritten.
template <bool PAGED>
__global__ __launch_bounds__(256) void range_merge_kernel(RangeAttnArgs a) {
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const Seq sq = seq_of<PAGED>(a, blockIdx.y);
    if (at >= (int64_t)max(sq.n, 0) * a.H) return;
    const int head = (int)(at % a.H);
    const int64_t tok = sq.t0 + at / a.H, r = tok * a.H + head;
    const float* ml = a.part_ml + r * a.nsplit * 2;
    const float* po = a.part_o + r * a.nsplit * D + 2 * lane;
    float M = -INFINITY;
    for (int s = lane; s < a.nsplit; s += 64) M = fmaxf(M, ml[2 * s]);
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
    float L = 0.0f, o0 = 0.0f, o1 = 0.0f;
    if (M > -INFINITY) {
        for (int s = 0; s < a.nsplit; ++s) {
            const float m = ml[2 * s];
            if (!(m > -INFINITY)) continue;
            const float w = __builtin_amdgcn_exp2f(m - M);
            const float2 v = *reinterpret_cast<const float2*>(po + (int64_t)s * D);
            L = fmaf(w, ml[2 * s + 1], L);
            o0 = fmaf(w, v.x, o0);
            o1 = fmaf(w, v.y, o1);
        }
    }
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    *reinterpret_cast<uint32_t*>(a.out + tok * a.o_rs + head * D + 2 * lane) = pack_bf16x2(o0 * inv, o1 * inv);
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

hipError_t launch_range_attn(const RangeAttnArgs& a, bool paged, hipStream_t stream) {
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
