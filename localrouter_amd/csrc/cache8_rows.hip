// The append into a cache in pages of 8 bits (gfx950): head norms and rotation of new tokens, queries to bf16 rows, keys and values
// to e4m3 with one scale 2^e for each GROUP8 = 16 rows of a page and head.
//
//   e = the least integer with max|y| <= 448 2^e over the new rows of the group, in [-100, 119]; of a group that holds earlier
//       positions of the sequence no less than before, and where it is more their rows are rounded again, to q 2^(e_old - e)
//   q = rne(clamp(y 2^-e, +-448)); an infinity or NaN is held as NaN and has no part in e
//
// Scales that are powers of two: e4m3 has the same relative precision at any of them, a group that grows rounds its earlier rows
// only where they reach the format's subnormals, and the conversions of the attention take them as they are. One rounding: y in
// fp32 to 8 bits.
//
// Every (sequence, group of 16 positions, head) of keys and of values is one wave, which has the group's rows in registers while
// it finds their maximum: four rows a round, 16 lanes of 8 dims. A sequence of n tokens touches at most (n - 2) / 16 + 2 groups;
// sequence b's are numbered from starts[b] / 16 + 2 b on, which leaves room for as many whatever the lengths, so a wave finds its
// group from starts alone, and the launch is sized by T and B.
//
// What bounds it: HBM with prompts (11 of up to 1,500 tokens, 32 heads over 8, 265 MB: 58 us, 4.6 TB/s), else the launch and the chain of
// loads (the token's sequence among starts, its length, page entry and table row): 24 single tokens 4.6 us, 7 chunks of up to 37 4.7.
#include "lr_common.h"
#include "lr_cache_kernels.h"

namespace lr {

namespace {

#include "append_rows.inc"
#include "div_small.inc"

// The maximum over the wave, in every lane.
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp_f32<DPP_XOR1>(x));
    x = fmaxf(x, dpp_f32<DPP_XOR2>(x));
    x = fmaxf(x, dpp_f32<DPP_HALF_MIRROR>(x));
    x = fmaxf(x, dpp_f32<DPP_MIRROR>(x));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ float exp2_int(int e) {   // 2^e, 0 below 2^-126
    return e < -126 ? 0.0f : __uint_as_float((uint32_t)(e + 127) << 23);
}

// The least e with a <= 448 2^e (448 = 1.75 2^8), in [-100, 119], of a finite a >= 0.
__device__ __forceinline__ int exponent8(float a) {
    const uint32_t x = __float_as_uint(a);
    return min(119, max(-100, (int)(x >> 23) - 127 - 8 + ((x & 0x7fffff) > 0x600000 ? 1 : 0)));
}

// Eight values times s, at most 448, as bytes.
__device__ __forceinline__ u32x2 pack8(const float (&y)[8], float s) {
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int x = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i] * s, y[4 * i + 1] * s, 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2] * s, y[4 * i + 3] * s, x, true);
    }
    return w;
}

// What is left of a value where some of a group are too large or not finite: clamped, NaN.
__device__ __forceinline__ float in_range(float y) {
    const float x = __builtin_amdgcn_fmed3f(y, -0x1.cp127f, 0x1.cp127f);   // (448 * 2^119)
    return fabsf(y) < INFINITY ? x : __builtin_nanf("");
}

// A sequence's tokens and positions.
struct Span8 {
    int b, s0, s1, len;
};

// The sequence of the token t of the lane's 16 (b -1: none). Of at most 64 sequences all are read at once, one a lane.
__device__ __forceinline__ Span8 span_of_token(const CacheAppendArgs& a, int t) {
    Span8 r;
    if (a.B <= 64) {
        const int lane = threadIdx.x & 63, mine = min(lane, a.B - 1);
        const int st = a.starts[mine], next = a.starts[mine + 1], ln = a.lens[mine];
        int b = 0;
#pragma unroll
        for (int g = 0; g < 4; ++g) {   // (the last that begins at or before the group's token)
            const uint64_t m = __builtin_amdgcn_ballot_w64(lane < a.B && st <= __builtin_amdgcn_readlane(t, 16 * g));
            const int last = m ? 63 - __builtin_clzll(m) : 0;
            b = (lane >> 4) == g ? last : b;
        }
        r.s0 = __shfl(st, b, 64);
        r.s1 = __shfl(next, b, 64);
        r.len = __shfl(ln, b, 64);
        r.b = r.s0 <= t && t < r.s1 ? b : -1;
        return r;
    }
    r.b = seq_of_token(a.starts, a.B, t);
    r.s0 = a.starts[max(r.b, 0)];
    r.s1 = a.starts[max(r.b, 0) + 1];
    r.len = a.lens[max(r.b, 0)];
    return r;
}

// Lane c's norm weights (ones without).
__device__ __forceinline__ void weights(const float* w, int c, float (&wv)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) wv[j] = 1.0f;
    if (w) {
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(w + 8 * c), w1 = *reinterpret_cast<const f32x4*>(w + 8 * c + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { wv[j] = w0[j]; wv[4 + j] = w1[j]; }
    }
}

// Queries: one 16-lane group a token and HPG heads, as cache_append_kernel.
template <int KIND, int PAIRING>
__device__ __forceinline__ void query_rows(const CacheAppendArgs& a, int64_t gid) {
    const int c = threadIdx.x & 15, hq = (a.H + HPG - 1) / HPG;
    const int64_t total = (int64_t)a.T * hq, gg = min(gid, total - 1);
    const int t = total < ((int64_t)1 << 32) ? (int)((uint32_t)gg / (uint32_t)hq) : (int)(gg / hq);
    const int h0 = HPG * (int)(gg - (int64_t)t * hq);
    const uint16_t* src = a.q + (int64_t)t * a.q_rs + 8 * c;
    u32x4 xin[HPG];
#pragma unroll
    for (int i = 0; i < HPG; ++i) xin[i] = *reinterpret_cast<const u32x4*>(src + min(h0 + i, a.H - 1) * D);
    float wv[8];
    weights(a.qw, c, wv);
    const Span8 sp = span_of_token(a, t);
    const int slot = sp.len - (sp.s1 - sp.s0) + (t - sp.s0);
    const int pos = a.pos ? a.pos[t] : slot;
    bool live = gid < total && sp.b >= 0 && (KIND == TABLE_NONE || (pos >= 0 && pos < a.tab_rows));
    Rot2 rt[8];
    table_rot<KIND, PAIRING>(a.ta, a.tb, (int64_t)(live ? pos : 0) * a.tab_stride, c, a.rot, a.tab_vec, rt);
    live = live && page_offset(a.pg, sp.b, slot) >= 0;
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = lo_bf16(xin[i][j]);
            x[2 * j + 1] = hi_bf16(xin[i][j]);
        }
        norm_turn<KIND, PAIRING>(x, wv, rt, a.eps, a.rot);
        if (live && h0 + i < a.H) {
            u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
            *reinterpret_cast<u32x4*>(a.q_out + (int64_t)t * a.qo_rs + (h0 + i) * D + 8 * c) = o;
        }
    }
}

// The last sequence whose groups' numbers begin at or before u (read at once, one a lane, of at most 64; else 64 probes a round).
__device__ __forceinline__ Span8 span_of_group(const CacheAppendArgs& a, int u) {
    const int lane = threadIdx.x & 63;
    Span8 r;
    if (a.B <= 64) {
        const int mine = min(lane, a.B - 1);
        const int st = a.starts[mine], next = a.starts[mine + 1], ln = a.lens[mine];
        const uint64_t m = __builtin_amdgcn_ballot_w64(lane < a.B && (st >> 4) + 2 * lane <= u);
        r.b = m ? 63 - __builtin_clzll(m) : 0;
        r.s0 = __builtin_amdgcn_readlane(st, r.b);
        r.s1 = __builtin_amdgcn_readlane(next, r.b);
        r.len = __builtin_amdgcn_readlane(ln, r.b);
        return r;
    }
    int lo = 0, width = a.B;
    while (width > 1) {
        const int step = (width + 63) >> 6, at = lane * step, i = lo + at;
        const bool le = at < width && i < a.B && (a.starts[min(i, a.B - 1)] >> 4) + 2 * i <= u;
        const int cnt = __popcll(__builtin_amdgcn_ballot_w64(le));   // (unsigned as it comes; 0 of starts that begin later)
        lo += max(cnt - 1, 0) * step;
        width = step;
    }
    r.b = __builtin_amdgcn_readfirstlane(lo);
    r.s0 = a.starts[r.b];
    r.s1 = a.starts[r.b + 1];
    r.len = a.lens[r.b];
    return r;
}

// Keys (part < HK) or values of one head of group u. MANY: every round of rows whether there are new ones or not, all loads before any
// is used, without branches between them; and whole rows rotated by cos / sin in a path of their own.
template <int KIND, int PAIRING, bool MANY>
__device__ __forceinline__ void group_rows(const CacheAppend8Args& g, int u, int part) {
    const CacheAppendArgs& a = g.at;
    const int lane = threadIdx.x & 63, c = lane & 15, sub = lane >> 4;
    const bool is_k = part < a.HK;
    const int h = is_k ? part : part - a.HK;
    float wv[8];
    weights(is_k ? a.kw : nullptr, c, wv);
    const Span8 sp = span_of_group(a, u);
    if (sp.s0 < 0 || sp.s1 <= sp.s0 || sp.len < 0) return;
    const int first = sp.len - (sp.s1 - sp.s0), n = min(sp.s1, a.T) - sp.s0;   // the call's first position, its tokens
    const int grp = (first >> 4) + u - ((sp.s0 >> 4) + 2 * sp.b);
    if (grp < (first >> 4) || grp < 0) return;
    const int base = 16 * grp, lo = max(first, base), hi = min(first + n, base + 16);
    if (lo >= hi || (base >> a.pg.shift) >= a.pg.table_pages) return;
    const int page = a.pg.table[(int64_t)sp.b * a.pg.table_rs + (base >> a.pg.shift)];

    // ---- the rows: round q the positions base + 4 q .. + 3, if any of them is new
    const uint16_t* src = (is_k ? a.k : a.v) + h * D + 8 * c;
    const int64_t rs = is_k ? a.k_rs : a.v_rs;
    auto round_in = [&](int q) { return MANY || (base + 4 * q + 3 >= lo && base + 4 * q < hi); };
    u32x4 xin[4];
    bool live[4];
    int pos[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        live[q] = false;
        pos[q] = 0;
        if (!round_in(q)) continue;
        const int slot = base + 4 * q + sub, t = sp.s0 + min(max(slot, lo), hi - 1) - first;
        xin[q] = *reinterpret_cast<const u32x4*>(src + (int64_t)t * rs);
        pos[q] = a.pos ? a.pos[t] : slot;
        live[q] = slot >= lo && slot < hi && (KIND == TABLE_NONE || (pos[q] >= 0 && pos[q] < a.tab_rows));
    }
    constexpr bool WHOLE = MANY && KIND == TABLE_COSSIN_F32 && PAIRING == PAIR_INTERLEAVED;
    const bool whole = WHOLE && is_k && a.tab_vec && a.rot == D;
    f32x4 cv[4], sv[4];
    if (whole)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t at = (int64_t)(live[q] ? pos[q] : 0) * a.tab_stride + 4 * c;
            cv[q] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.ta) + at);
            sv[q] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.tb) + at);
        }
    if (page < 0 || page >= a.pg.n_pages || !__builtin_amdgcn_ballot_w64(live[0] || live[1] || live[2] || live[3])) return;
    const int row = base & ((1 << a.pg.shift) - 1);
    uint8_t* scale = (is_k ? g.k_sc : g.v_sc) + (int64_t)page * g.sc_ps + (int64_t)(row >> 4) * a.HK + h;
    uint8_t* rows = reinterpret_cast<uint8_t*>(is_k ? a.kp : a.vp) + (int64_t)page * a.pg.ps + (int64_t)row * a.pg.rs + (int64_t)h * a.pg.hs + 8 * c;
    const bool more = lo > base;   // earlier positions
    const int e_old = more ? (int)*scale - 127 : -100;
    float y[4][8], most = 0.0f, odd = 0.0f;   // (odd: NaN where a value is not finite)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (!round_in(q)) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            y[q][2 * j] = lo_bf16(xin[q][j]);
            y[q][2 * j + 1] = hi_bf16(xin[q][j]);
        }
        if (whole) {
            Rot2 rt[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) rt[j] = Rot2{cv[q][j], -sv[q][j], sv[q][j], cv[q][j]};
            norm_turn<KIND, PAIRING>(y[q], wv, rt, a.eps, D);
        } else if (is_k) {
            Rot2 rt[8];
            table_rot<KIND, PAIRING>(a.ta, a.tb, (int64_t)(live[q] ? pos[q] : 0) * a.tab_stride, c, a.rot, a.tab_vec, rt);
            norm_turn<KIND, PAIRING>(y[q], wv, rt, a.eps, a.rot);
        }
        float m = 0.0f, z = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m = fmaxf(m, fabsf(y[q][j]));
            z = fmaf(0.0f, y[q][j], z);
        }
        most = live[q] ? fmaxf(most, m) : most;
        odd = live[q] ? odd + z : odd;
    }
    if (__builtin_amdgcn_ballot_w64(!(odd == 0.0f) || most > 0x1.cp127f)) {
        most = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (!round_in(q)) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[q][j] = in_range(y[q][j]);
                most = live[q] ? fmaxf(most, fabsf(y[q][j])) : most;   // (the maximum with NaN is the other)
            }
        }
    }
    const int e = max(e_old, __builtin_amdgcn_readfirstlane(exponent8(wave_max(most))));
    if (lane == 0 && (!more || e != e_old)) *scale = (uint8_t)(e + 127);
    const float s = exp2_int(-e);
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (live[q]) *reinterpret_cast<u32x2*>(rows + (int64_t)(4 * q + sub) * a.pg.rs) = pack8(y[q], s);
    if (more && e > e_old) {   // the earlier rows again
        const float r = exp2_int(e_old - e);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (base + 4 * q + sub < lo) {
                u32x2* at = reinterpret_cast<u32x2*>(rows + (int64_t)(4 * q + sub) * a.pg.rs);
                const u32x2 w = *at;
                float z[8];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const f32x2 x0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[x], false), x1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[x], true);
                    z[4 * x] = x0[0]; z[4 * x + 1] = x0[1]; z[4 * x + 2] = x1[0]; z[4 * x + 3] = x1[1];
                }
                *at = pack8(z, r);
            }
    }
}

template <int KIND, int PAIRING, bool MANY>
__global__ __launch_bounds__(256) void cache_append8_kernel(CacheAppend8Args a, int waves, uint32_t rcp_parts) {
    // (keys and values first: theirs is the longer chain)
    const int group_blocks = (waves + 3) / 4;
    if ((int)blockIdx.x >= group_blocks) {
        query_rows<KIND, PAIRING>(a.at, (int64_t)((int)blockIdx.x - group_blocks) * 16 + (threadIdx.x >> 4));
        return;
    }
    const int w = 4 * (int)blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= waves) return;
    const int parts = 2 * a.at.HK, u = div_small(w, parts, rcp_parts);
    group_rows<KIND, PAIRING, MANY>(a, u, w - u * parts);
}

template <int KIND>
hipError_t append8_kind(const CacheAppend8Args& a, hipStream_t stream) {
    const int64_t query_blocks = ((int64_t)a.at.T * ((a.at.H + HPG - 1) / HPG) + 15) / 16;
    const int64_t waves = ((int64_t)(a.at.T >> 4) + 2 * (int64_t)a.at.B) * 2 * a.at.HK, blocks = query_blocks + (waves + 3) / 4;
    if (blocks > 1 << 23) return hipErrorInvalidValue;   // (a grid's work-items are counted in 32 bits)
    // us without / with: 24 tokens of 24 sequences 4.5 / 4.6, 64 of 64 6.0 / 6.6, up to 37 of 7 7.1 / 6.8, 1,125 of 11 53.5 / 54.6, 1,500 of
    // 8 with 16 kv heads 48.0 / 44.7
    const bool many = a.at.T >= 16 * (int64_t)a.at.B;
    const auto kernel = a.at.pairing == PAIR_SPLIT_HALF
                            ? (many ? cache_append8_kernel<KIND, PAIR_SPLIT_HALF, true> : cache_append8_kernel<KIND, PAIR_SPLIT_HALF, false>)
                            : (many ? cache_append8_kernel<KIND, PAIR_INTERLEAVED, true> : cache_append8_kernel<KIND, PAIR_INTERLEAVED, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a, (int)waves, rcp_small(2 * a.at.HK));
    return hipGetLastError();
}

// A workgroup copies one page's scales of one layer's keys or values.
__global__ __launch_bounds__(64) void cache_copy_scales_kernel(CacheCopyScalesArgs a) {
    const int src = a.src[blockIdx.x], dst = a.dst[blockIdx.x];
    if (src < 0 || src >= a.n_pages || dst < 0 || dst >= a.n_pages || src == dst) return;
    uint8_t* base = (blockIdx.z ? a.v_sc : a.k_sc) + (int64_t)blockIdx.y * a.layer_stride;
    for (int i = threadIdx.x; i < a.bytes; i += 64) base[(int64_t)dst * a.sc_ps + i] = base[(int64_t)src * a.sc_ps + i];
}

}  // namespace

hipError_t launch_cache_append8(const CacheAppend8Args& g, hipStream_t stream) {
    const CacheAppendArgs& a = g.at;
    switch (a.table_kind) {
        case TABLE_NONE: return append8_kind<TABLE_NONE>(g, stream);
        case TABLE_COSSIN_F32: return append8_kind<TABLE_COSSIN_F32>(g, stream);
        case TABLE_MAT2_BF16: return append8_kind<TABLE_MAT2_BF16>(g, stream);
        case TABLE_MAT2_F32: return append8_kind<TABLE_MAT2_F32>(g, stream);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_cache_copy_scales(const CacheCopyScalesArgs& a, hipStream_t stream) {
    if (a.n > 1 << 23 || a.layers > 65535) return hipErrorInvalidValue;
    hipLaunchKernelGGL(cache_copy_scales_kernel, dim3((unsigned)a.n, (unsigned)a.layers, 2), dim3(64), 0, stream, a);
    return hipGetLastError();
}

}  // namespace lr
