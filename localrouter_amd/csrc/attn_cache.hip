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
// The rows of one kv head (tokens x the G query heads that share it) form blocks of rows; a workgroup takes one block and one part
// of its key tiles, its waves (or groups of waves) alternate over the tiles. S^T = K Q^T and O^T += V^T P^T with P in registers, K
// and V tiles row-major in LDS by direct loads. Two kernels here, for the calls that the one of attn_cache_wide.hip does not take:
//   range_step_kernel   blocks of 16 or 32 rows: single tokens, small trees; bound by the chain from one load and one instruction
//                       to the next. 8 kv heads, one token of 4 query heads each: 500 keys 7.4 us, 1,900 8.7, 16,000 19; from a
//                       few dozen MB on by HBM (64 sequences of 7,000 keys, 2.7 GB, 477 us = 5.7 TB/s).
//   range_attn_kernel   blocks of 64 or 128 rows: larger batches of trees, pages of fewer than 16 rows, rows far apart.
#include "lr_common.h"
#include "lr_cache_kernels.h"

namespace lr {

namespace {

#include "attn_common.inc"

#include "range_attn.inc"

constexpr uint64_t PART_DONE = 0x7ff4a3c57fb5d96e;

// The parts of one block of BR rows. (sc1, 16: coherent at device scope, not kept in this XCD's L2; the last workgroup of the block
// may run on another.)
template <int BR>
struct PartRows {
    __amdgpu_buffer_rsrc_t rs_o, rs_ml;
    uint64_t* flags;

    __device__ __forceinline__ PartRows(const RangeAttnArgs& a, int64_t block) {
        rs_o = __builtin_amdgcn_make_buffer_rsrc(a.part_o + block * a.nsplit * BR * D, 0, a.nsplit * BR * D * 4, 0x00020000);
        rs_ml = __builtin_amdgcn_make_buffer_rsrc(a.part_ml + block * a.nsplit * BR * 2, 0, a.nsplit * BR * 8, 0x00020000);
        flags = a.flags + block * a.nsplit;
    }
    __device__ __forceinline__ void put_ml(int split, int q, float m, float l) const {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, rs_ml, (split * BR + q) * 8, 0, 16);
    }
    __device__ __forceinline__ void put4(int split, int q, int dim, f32x4 y) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), rs_o, ((split * BR + q) * D + dim) * 4, 0, 16);
    }
    __device__ __forceinline__ void put_row2(int split, int q, float o0, float o1, float m, float l) const {
        const int lane = threadIdx.x & 63;
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(o0), __float_as_uint(o1)}, rs_o,
                                              ((split * BR + q) * D + 2 * lane) * 4, 0, 16);
        if (lane == 0) put_ml(split, q, m, l);
    }

    // The last of the block's parts to end merges them, in their order (every wave's rows are in memory). A part whose rows are
    // in memory sets its flag, then reads all of them: the last to set its own sees every one (two that do write the same
    // rows). Flags need no clearing before the call: only PART_DONE counts (as a float or a pair of them a NaN that no arithmetic
    // makes), and who merges clears them.
    template <int NW>
    __device__ __forceinline__ void merge_last(const RangeAttnArgs& a, const Seq& sq, int hk, int row0, int rows, int split,
                                               int parts, int* shared) const {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (wave == 0) {   // (alone: a flag set after the merge would outlive the call)
            if (lane == 0) __hip_atomic_store(flags + split, PART_DONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            LR_WAIT_VMCNT(0);
            bool done = true;
            for (int s0 = 0; s0 < parts; s0 += 64)
                done = done && __hip_atomic_load(flags + min(s0 + lane, parts - 1), __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT) == PART_DONE;
            const bool last = __builtin_amdgcn_ballot_w64(done) == ~0ull;
            if (lane == 0) shared[0] = last;
            if (last)
                for (int s0 = lane; s0 < parts; s0 += 64)
                    __hip_atomic_store(flags + s0, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!__builtin_amdgcn_readfirstlane(shared[0])) return;
        // 32 lanes a row (dims 4 c .. 4 c + 3), two rows a wave, eight parts in flight
        static_assert(BR == 2 * NW, "one pass");
        const int mc = lane & 31;
        if (2 * wave < rows - row0) {
            const int q = min(2 * wave + (lane >> 5), rows - row0 - 1);   // (past the last row: that one again, the same)
            float M = -INFINITY, L = 0.0f;
            f32x4 sum{};
            for (int s0 = 0; s0 < parts; s0 += 8) {
                u32x2 ml[8];
                u32x4 x[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int at = min(s0 + u, parts - 1) * BR + q;
                    ml[u] = __builtin_amdgcn_raw_buffer_load_b64(rs_ml, at * 8, 0, 16);
                    x[u] = __builtin_amdgcn_raw_buffer_load_b128(rs_o, at * D * 4 + 16 * mc, 0, 16);
                }
                float Mn = M;
#pragma unroll
                for (int u = 0; u < 8; ++u) Mn = fmaxf(Mn, __uint_as_float(ml[u][0]));
                const float ref = Mn > -INFINITY ? Mn : 0.0f, alpha = __builtin_amdgcn_exp2f(M - ref);
                M = Mn;
                L *= alpha;
                sum *= alpha;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    // a part that saw no key has no weight, whatever is in its row
                    const float m = __uint_as_float(ml[u][0]);
                    const bool in = m > -INFINITY && s0 + u < parts;
                    const float w = __builtin_amdgcn_exp2f(m - ref);
                    L = in ? fmaf(w, __uint_as_float(ml[u][1]), L) : L;
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = in ? fmaf(w, __uint_as_float(x[u][e]), sum[e]) : sum[e];
                }
            }
            const int ri = div_small(row0 + q, a.G, a.rcp_g), rhead = hk * a.G + row0 + q - ri * a.G;
            const float inv = L != 0.0f ? 1.0f / L : 0.0f;
            u32x2 w;
            w[0] = pack_bf16x2(sum[0] * inv, sum[1] * inv);
            w[1] = pack_bf16x2(sum[2] * inv, sum[3] * inv);
            *reinterpret_cast<u32x2*>(a.out + (int64_t)(sq.t0 + ri) * a.o_rs + rhead * D + 4 * mc) = w;
        }
    }
};

// The direct loads of a tile by wave rb of RB: instruction u fills rows 4 u .. 4 u + 3, 16-byte chunks swizzled as attn_fwd.hip's.
template <int RB, bool PAGED>
__device__ __forceinline__ void load_tile_rows(const RangeAttnArgs& a, const Seq& sq, const TileList<RANGE_TILE, PAGED>& tl,
                                               int64_t hoff, int x, uint32_t k_lds, uint32_t v_lds, int rb) {
    constexpr int BT = RANGE_TILE, LOADS = 8 / RB;
    const int lane = threadIdx.x & 63, lrow = lane >> 4, lchunk = lane & 15, key0 = tl.key0(x);
    const int64_t k_rs = PAGED ? a.pg.rs : a.k_rs, v_rs = PAGED ? a.pg.rs : a.v_rs;
    const uint16_t *kp = a.k + hoff, *vp = a.v + hoff;
    if ((!PAGED || tl.shift >= 5) && key0 + BT <= sq.end) {   // the tile's rows are one run
        const int64_t row = (PAGED ? key0 & ((1 << tl.shift) - 1) : key0) + 4 * rb + lrow;
        const int64_t pg = PAGED ? (int64_t)max(tl.entry(x, 0), 0) * a.pg.ps : 0;
        kp += pg + row * k_rs;
        vp += pg + row * v_rs + 8 * (lchunk ^ (lrow << 2));
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int inst = rb + RB * u;
            dma16(kp + 8 * (lchunk ^ ((4 * inst + lrow) & 15)), k_lds + 1024 * inst);
            dma16(vp, v_lds + 1024 * inst);
            kp += 4 * RB * k_rs;
            vp += 4 * RB * v_rs;
        }
        return;
    }
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        const int inst = rb + RB * u, row = 4 * inst + lrow;
        const int64_t o = tl.offset(a, x, row, k_rs), ov = PAGED ? o : tl.offset(a, x, row, v_rs);
        dma16(kp + o + 8 * (lchunk ^ (row & 15)), k_lds + 1024 * inst);
        dma16(vp + ov + 8 * (lchunk ^ (lrow << 2)), v_lds + 1024 * inst);
    }
}

// A lane's value over the four lanes of its row (16 apart).
__device__ __forceinline__ float quad_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return wave_pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return wave_pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// The rows of which a group of waves (RB of them) has bits set, again, by its KG waves in turn; f(q): row q of the group. Where every
// wave's rows were in memory before, they are afterwards.
template <int RB, int KG, class F>
__device__ __forceinline__ void again_rows(int* shared, int rb, int kg, uint32_t bits, F&& f) {
    if (!__syncthreads_or(bits != 0)) return;
    LR_WAIT_VMCNT(0);   // (the rows that are overwritten below)
    if (threadIdx.x < RB) shared[threadIdx.x] = 0;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) atomicOr(shared + rb, (int)bits);
    __syncthreads();
    uint32_t left = (uint32_t)shared[rb];
    for (int nth = 0; left; left &= left - 1, ++nth)
        if (nth % KG == kg) f(__builtin_amdgcn_readfirstlane(__builtin_ctz(left)));
    LR_WAIT_VMCNT(0);
    __syncthreads();
}

// Blocks of 64 and 128 rows: KG groups of RB waves (32 rows each) alternate over the tiles, a ring of NS of them a group, on
// v_mfma_f32_32x32x16_bf16 (the pipelined kernel's fragments, attn_fwd.hip). Bound by HBM where it is taken (32 sequences of 16,000
// keys over 8 kv heads, 64 rows each, 2.1 GB, 384 us = 5.5 TB/s): one read of the keys for all rows is what counts.
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
    int hi_all, lo_all;
    seen_by_all<PAGED>(a, sq, div_small(min(wr0, rows - 1), a.G, a.rcp_g), div_small(min(wr0 + 31, rows - 1), a.G, a.rcp_g), me,
                       hi_all, lo_all);

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

    const uint32_t kr_lds = lds_addr(ring) + kg * NS * TILE * 4, vr_lds = kr_lds + NS * TILE * 2;
    auto load_tile = [&](int x, int slot) {
        load_tile_rows<RB, PAGED>(a, sq, tl, hoff, x, kr_lds + 2 * slot * TILE, vr_lds + 2 * slot * TILE, rb);
    };

    const int mine = x1 > x0 + kg ? (x1 - x0 - kg + KG - 1) / KG : 0;   // tiles of this group
    const int steps = x1 > x0 ? (x1 - x0 + KG - 1) / KG : 0;             // of group 0: every group's barriers
    auto tile_of = [&](int t) { return x0 + kg + t * KG; };

    constexpr int AHEAD = NS - 1;   // tiles in flight before the first step
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
        if (t + AHEAD - 1 < mine) LR_WAIT_VMCNT((AHEAD - 1) * 2 * LOADS);
        else LR_WAIT_VMCNT(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this wave's reads of tile t - 1, whose slot is refilled
        block_barrier();
        if (t + NS - 1 < mine) load_tile(tile_of(t + NS - 1), (t + NS - 1) % NS);
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
    const PartRows<BR> to(a, block);
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
                    to.put4(split, q, 32 * (kg + KG * x) + 8 * q4 + 4 * hf, y);
                }
            if (hf == 0 && kg == 0) to.put_ml(split, q, m_used, l);
        }
        bits = __builtin_amdgcn_ballot_w64(broken);
    }
    // ---- rows with an infinity or NaN in some group's dims again, whole, over the seen keys only
    int* again = reinterpret_cast<int*>(ring);
    again_rows<RB, KG>(again, rb, kg, (uint32_t)(bits | bits >> 32), [&](int q) __attribute__((always_inline)) {
        const int ri = __builtin_amdgcn_readlane(i, q), rhead = __builtin_amdgcn_readlane(head, q);
        redo_row<BT, PAGED>(a, sq, tl, hk, ri, rhead, [&](float o0, float o1, float m, float rl) {
            if (whole_block) put_row(a.out + (int64_t)(sq.t0 + ri) * a.o_rs + rhead * D, o0, o1, rl);
            else to.put_row2(split, 32 * rb + q, o0, o1, m, rl);
        });
    });
}

// Calls of few rows of a kv head a sequence (single tokens, small trees): NB blocks of 16 rows, on v_mfma_f32_16x16x32_bf16. What
// they cost is the time from one instruction's result to the next: half the scores and sums a lane of a block of 32, a chain of
// 4 products for a block of 16 keys in place of 8, eight waves of one tile each in place of four of two.
// Lane 16 g + n: row n of each block; of a tile's scores the keys 4 g + r and 16 + 4 g + r (r < 4), in which order its products
// take the keys; of the sums the dims 16 db + 4 g + r.
template <int NB, int KG, bool PAGED>
__global__ __launch_bounds__(KG * 64, KG / 4) void range_step_kernel(RangeAttnArgs a) {
    constexpr int BT = RANGE_TILE, TILE = BT * D, BR = 16 * NB;
    typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;
    constexpr int OWN_LDS = TILE * 2 * 2;   // bytes of LDS a wave: its tiles, then its sums
    static_assert(OWN_LDS >= NB * 8 * 1024, "a wave's sums in the place of its tiles");
    __shared__ __attribute__((aligned(1024))) char ring[KG * OWN_LDS];
    __shared__ float2 mls[KG * NB * 16];
    __shared__ int staged[PAGED ? RANGE_STAGED : 1];

    const int tid = threadIdx.x, lane = tid & 63, kg = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;

    // ---- which rows, which keys
    const int at = div_small(blockIdx.x, a.nsplit, a.rcp_split), split = blockIdx.x - at * a.nsplit;
    const int blk = div_small(at, a.HK, a.rcp_hk), hk = at - blk * a.HK, b = blockIdx.y;
    // without a window a part's entries do not depend on the sequence: they are read beside its numbers
    int early = -1;
    const int per_tile = PAGED ? max(1, BT >> a.pg.shift) : 1;
    const bool ahead = PAGED && !a.window && a.per * per_tile <= KG * 64;
    if (ahead && tid < a.per * per_tile) {
        const int j = BT * (split * a.per + tid / per_tile) + (tid % per_tile << a.pg.shift);
        if (j >> a.pg.shift < a.pg.table_pages) early = a.pg.table[(int64_t)b * a.pg.table_rs + (j >> a.pg.shift)];
    }
    const Seq sq = seq_of<PAGED>(a, b);
    const int row0 = blk * BR, rows = max(sq.n, 0) * a.G;   // (at most 2^30: the host checks)
    if (row0 >= rows) return;
    const int i_first = div_small(row0, a.G, a.rcp_g), i_last = div_small(min(rows, row0 + BR) - 1, a.G, a.rcp_g);
    TileList<BT, PAGED> tl;
    tl.init(a, sq, i_first, i_last);
    tl.part(split, a.per);
    const int parts = min(a.nsplit, max(1, (tl.total + a.per - 1) / a.per));   // the sequence may be shorter than the longest
    if (split >= parts) return;
    const int x0 = tl.x0, x1 = tl.x1;

    // ---- this lane's rows
    const int64_t hoff = (int64_t)hk * (PAGED ? a.pg.hs : D);
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
        me[nb] = sees_of<PAGED>(a, sq, ri[nb]);
        const uint16_t* src = a.q + (int64_t)(sq.t0 + ri[nb]) * a.q_rs + head[nb] * D + 8 * g;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[nb][ks] = *reinterpret_cast<const bf16x8*>(src + 32 * ks);
    }
    int hi_all, lo_all, lo_last;
    seen_by_all<PAGED>(a, sq, i_first, i_last, me[0], hi_all, lo_all);
    if (NB > 1) {
        seen_by_all<PAGED>(a, sq, i_first, i_last, me[NB - 1], hi_all, lo_last);
        lo_all = max(lo_all, lo_last);
    }
    const bool bad = tl.template stage<KG * 64>(a, b, staged, ahead, early);

    const uint32_t kr_lds = lds_addr(ring) + kg * OWN_LDS, vr_lds = kr_lds + TILE * 2;
    const int mine = x1 > x0 + kg ? (x1 - x0 - kg + KG - 1) / KG : 0;   // tiles of this wave
    auto tile_of = [&](int t) { return x0 + kg + t * KG; };
    int vtr[8];   // (dims 16 db .. of rows 4 g + (n >> 2), and 16 rows on)
#pragma unroll
    for (int db = 0; db < 8; ++db)
        vtr[db] = (4 * g + (n >> 2)) * D + 8 * ((2 * db + ((n & 3) >> 1)) ^ (n >> 2 << 2)) + 4 * (n & 1);

    f32x4 o[NB][8];
    float m_used[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        m_used[nb] = -INFINITY;
        l[nb] = 0.0f;
#pragma unroll
        for (int db = 0; db < 8; ++db) o[nb][db] = f32x4{};
    }
    const float c = a.c;
    const bf16x2 ones2 = {(bf16)1.0f, (bf16)1.0f};

    const uint16_t *kt = reinterpret_cast<const uint16_t*>(ring) + kg * TILE * 2, *vt = kt + TILE;
    // (one place that loads, its first pass before any tile: instructions not met yet cost as much as memory)
    for (int t = -1; t < mine; ++t) {
        u32x4 pw[NB];
        bf16x8 vf[8];
        if (t >= 0) {
            LR_WAIT_VMCNT(0);   // tile t has landed
            const int x = tile_of(t), key0 = tl.key0(x);
            f32x4 s[NB][2] = {};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kt + (16 * kb + n) * D + 8 * ((4 * ks + g) ^ n));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[nb][ks], s[nb][kb], 0, 0, 0);
                }
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vt + vtr[db]));
                const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vt + vtr[db] + 16 * D));
                vf[db] = __builtin_shufflevector(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
            }
            const bool whole = key0 + BT <= hi_all && (key0 >= lo_all || key0 + BT <= a.sinks) && !bad;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                f32x4 &s0 = s[nb][0], &s1 = s[nb][1];
                if (!whole) {
                    const uint32_t m = seen_bits<BT, PAGED>(a, sq, tl, bad, ri[nb], me[nb], x, 0) >> (4 * g);
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
                    for (int db = 0; db < 8; ++db) o[nb][db] *= alpha;
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
        }
        if (t + 1 < mine) {   // the tile's place is free again once this wave's reads have returned
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load_tile_rows<1, PAGED>(a, sq, tl, hoff, tile_of(t + 1), kr_lds, vr_lds, 0);
        }
        if (t < 0) continue;
#pragma unroll
        for (int db = 0; db < 8; ++db)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                o[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[db], __builtin_bit_cast(bf16x8, pw[nb]), o[nb][db], 0, 0, 0);
    }

    // ---- merge the waves: wave u takes the 16-dim blocks u, u + KG, ... from all of them (its own too: without a branch a
    // block); rows out: O / l, or this part of them
    static_assert(NB <= 2 && KG > 1 && 8 % KG == 0, "waves");
    constexpr int OWN = 8 / KG;
    const bool whole_block = parts == 1;
    const PartRows<BR> to(a, ((int64_t)b * a.nblk + blk) * a.HK + hk);
    float* mo = reinterpret_cast<float*>(ring);
    constexpr int OWN_F = OWN_LDS / 4;
    asm volatile("" ::: "memory");   // (the wave's own tiles are read)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        l[nb] = quad_sum(l[nb]);
        if (live[nb]) {
#pragma unroll
            for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4*>(mo + kg * OWN_F + (nb * 8 + db) * 256 + 4 * lane) = o[nb][db];
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
            uint16_t* dst = a.out + (int64_t)(sq.t0 + ri[nb]) * a.o_rs + head[nb] * D + 4 * g;
#pragma unroll
            for (int x = 0; x < OWN; ++x) {
                f32x4 own{};
#pragma unroll
                for (int u = 0; u < KG; ++u) {
                    const f32x4 y = *reinterpret_cast<const f32x4*>(mo + u * OWN_F + (nb * 8 + kg + KG * x) * 256 + 4 * lane);
#pragma unroll
                    for (int e = 0; e < 4; ++e) own[e] = fmaf(w[u], y[e], own[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) chk = fmaf(0.0f, own[e], chk);
                const int dim = 16 * (kg + KG * x);
                if (whole_block) {
                    u32x2 v;
                    v[0] = pack_bf16x2(own[0] * inv, own[1] * inv);
                    v[1] = pack_bf16x2(own[2] * inv, own[3] * inv);
                    *reinterpret_cast<u32x2*>(dst + dim) = v;
                } else {
                    to.put4(split, 16 * nb + n, dim + 4 * g, own);
                }
            }
            if (!whole_block && g == 0 && kg == 0) to.put_ml(split, 16 * nb + n, mm, sum);
            mine_broken = !(fabsf(chk) < INFINITY);
        }
        const uint64_t bits = __builtin_amdgcn_ballot_w64(mine_broken);
        const uint32_t half = (uint32_t)(bits | bits >> 32);
        broken |= ((half | half >> 16) & 0xffff) << (16 * nb);
    }
    // ---- rows with an infinity or NaN in some wave's dims again, whole, over the seen keys only
    if (!whole_block) LR_WAIT_VMCNT(0);   // (this wave's part is in memory)
    int* again = reinterpret_cast<int*>(ring);
    again_rows<1, KG>(again, 0, kg, broken, [&](int q) __attribute__((always_inline)) {
        int i = __builtin_amdgcn_readlane(ri[0], q & 15), h = __builtin_amdgcn_readlane(head[0], q & 15);
        if (NB > 1 && q >= 16) {
            i = __builtin_amdgcn_readlane(ri[NB - 1], q & 15);
            h = __builtin_amdgcn_readlane(head[NB - 1], q & 15);
        }
        redo_row<BT, PAGED>(a, sq, tl, hk, i, h, [&](float o0, float o1, float m, float rl) {
            if (whole_block) put_row(a.out + (int64_t)(sq.t0 + i) * a.o_rs + h * D, o0, o1, rl);
            else to.put_row2(split, q, o0, o1, m, rl);
        });
    });
    if constexpr (NB == 1)
        if (!whole_block && a.merge_here) to.template merge_last<KG>(a, sq, hk, row0, rows, split, parts, again);
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

template <int BR>
hipError_t launch_blocks(const RangeAttnArgs& a, bool paged, int threads, void (*rows_kernel)(RangeAttnArgs),
                         void (*paged_kernel)(RangeAttnArgs), hipStream_t stream) {
    const int64_t rows = (int64_t)(paged ? a.max_rows : a.W) * a.G;
    const int64_t blocks = (rows + BR - 1) / BR * a.HK * a.nsplit, merge = blocks / a.nsplit * (BR / 4);
    // (a block's bytes of parts are counted in 32 bits)
    if (blocks > RANGE_MAX_BLOCKS || merge > 2 * RANGE_MAX_BLOCKS || (int64_t)a.nsplit * BR * D * 4 > INT32_MAX) return hipErrorInvalidValue;
    const unsigned seqs = paged ? (unsigned)a.B : 1;
    hipLaunchKernelGGL(paged ? paged_kernel : rows_kernel, dim3((unsigned)blocks, seqs), dim3(threads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1 || a.merge_here) return e;
    if (paged) hipLaunchKernelGGL((range_merge_kernel<BR, true>), dim3((unsigned)merge, seqs), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((range_merge_kernel<BR, false>), dim3((unsigned)merge), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_range_attn(const RangeAttnArgs& a, bool paged, int br, hipStream_t stream) {
    if (br == 16) return launch_blocks<16>(a, paged, 512, range_step_kernel<1, 8, false>, range_step_kernel<1, 8, true>, stream);
    if (br == 32) return launch_blocks<32>(a, paged, 512, range_step_kernel<2, 8, false>, range_step_kernel<2, 8, true>, stream);
    if (br == 64) return launch_blocks<64>(a, paged, 256, range_attn_kernel<2, 2, 4, false>, range_attn_kernel<2, 2, 4, true>, stream);
    return launch_blocks<128>(a, paged, 512, range_attn_kernel<4, 2, 4, false>, range_attn_kernel<4, 2, 4, true>, stream);
}

}  // namespace lr
