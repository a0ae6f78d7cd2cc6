// The passes that write a cache in pages (gfx950): the append (head norms and rotation of new tokens, their keys and values
// into pages), page copies and row moves. All three are bound by memory: every byte is read once and written once, 16 bytes
// a lane, a row of one head (256 bytes) by 16 lanes. 16,000 tokens of 32 + 2 x 8 heads appended 60 us (4.9 TB/s), 1,000 pages of 16
// rows x 8 heads copied in 16 layers 387 us (5.4 TB/s), 40 x 5 rows moved in 32 layers 12.7 to 14.2 us (3.7 to 4.1 TB/s; the chain
// starts, positions, page entries, rows); the smallest calls 3 (a page's copy) to 4.5 us (32 tokens appended: the chain of a token's
// sequence, its length, page entry and table row).
#include "lr_common.h"
#include "lr_cache_kernels.h"

namespace lr {

namespace {

#include "rope_rows.inc"
#include "div_small.inc"

// The sequence of token t: the largest b < B with starts[b] <= t, by the 16 lanes of the token's group, 16 probes a round.
// -1: none. (Every lane of the wave takes the same rounds.)
__device__ __forceinline__ int seq_of_token(const int* starts, int B, int t) {
    const int lane = threadIdx.x & 63, c = lane & 15;
    int lo = 0, width = B;
    while (width > 1) {
        const int step = (width + 15) >> 4;
        const int i = lo + c * step;
        const bool le = c * step < width && i < B && starts[min(i, B - 1)] <= t;
        const int cnt = __popcll((__builtin_amdgcn_ballot_w64(le) >> (lane & 48)) & 0xffff);
        lo += max(cnt - 1, 0) * step;
        width = step;
    }
    return starts[lo] <= t && t < starts[lo + 1] ? lo : -1;
}

// Offset (elements) of position j of sequence b in the pool, or -1 where the sequence's table or the pool does not have it.
__device__ __forceinline__ int64_t page_offset(const PageArgs& g, int b, int j) {
    if (j < 0 || (j >> g.shift) >= g.table_pages) return -1;
    const int page = g.table[(int64_t)b * g.table_rs + (j >> g.shift)];
    if (page < 0 || page >= g.n_pages) return -1;
    return (int64_t)page * g.ps + (int64_t)(j & ((1 << g.shift) - 1)) * g.rs;
}

// One 16-lane group owns one token and HPG heads of one of q, k and v; lane c dims 8c .. 8c + 7 (rope_rows.inc's layout).
template <int KIND, int PAIRING>
__global__ __launch_bounds__(256) void cache_append_kernel(CacheAppendArgs a) {
    const int tid = threadIdx.x, c = tid & 15;
    const int hq = (a.H + HPG - 1) / HPG, hk = (a.HK + HPG - 1) / HPG, hg = hq + 2 * hk;
    const int64_t gid = (int64_t)blockIdx.x * 16 + (tid >> 4), total = (int64_t)a.T * hg;
    const int64_t gg = min(gid, total - 1);
    const int t = total < ((int64_t)1 << 32) ? (int)((uint32_t)gg / (uint32_t)hg) : (int)(gg / hg);
    const int part = (int)(gg - (int64_t)t * hg);
    const bool is_q = part < hq, is_k = !is_q && part < hq + hk;
    const int h0 = HPG * (is_q ? part : is_k ? part - hq : part - hq - hk);
    const int heads = is_q ? a.H : a.HK;
    const uint16_t* src = (is_q ? a.q + (int64_t)t * a.q_rs : is_k ? a.k + (int64_t)t * a.k_rs : a.v + (int64_t)t * a.v_rs) + 8 * c;

    u32x4 xin[HPG];
#pragma unroll
    for (int i = 0; i < HPG; ++i) xin[i] = *reinterpret_cast<const u32x4*>(src + min(h0 + i, heads - 1) * D);
    const float* wsrc = is_q ? a.qw : a.kw;
    float wv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) wv[j] = 1.0f;
    if (wsrc && (is_q || is_k)) {
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(wsrc + 8 * c), w1 = *reinterpret_cast<const f32x4*>(wsrc + 8 * c + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { wv[j] = w0[j]; wv[4 + j] = w1[j]; }
    }
    const int b = seq_of_token(a.starts, a.B, t);
    bool live = gid < total && b >= 0;
    const int s0 = a.starts[max(b, 0)], s1 = a.starts[max(b, 0) + 1];
    const int slot = a.lens[max(b, 0)] - (s1 - s0) + (t - s0);
    const int64_t off = live ? page_offset(a.pg, b, slot) : -1;
    const int pos = a.pos ? a.pos[t] : slot;
    live = live && off >= 0 && (KIND == TABLE_NONE || (pos >= 0 && pos < a.tab_rows));
    if (!is_q && !is_k) {
        if (live)
#pragma unroll
            for (int i = 0; i < HPG; ++i)
                if (h0 + i < a.HK) *reinterpret_cast<u32x4*>(a.vp + off + (int64_t)(h0 + i) * a.pg.hs + 8 * c) = xin[i];
        // (no return: the other groups of the wave exchange lanes below)
    }
    Rot2 rt[8];
    const int P = a.rot >> 1;
    if constexpr (KIND != TABLE_NONE) {
        const int64_t toff = (int64_t)(live ? pos : 0) * a.tab_stride;
        if constexpr (PAIRING == PAIR_INTERLEAVED) {
            rot4<KIND>(a.ta, a.tb, toff, 4 * c, P, a.tab_vec, rt);
        } else {
            const int hc = a.rot >> 4, pc = c < hc ? c : c - hc;
            rot4<KIND>(a.ta, a.tb, toff, 8 * pc, P, a.tab_vec, rt);
            rot4<KIND>(a.ta, a.tb, toff, 8 * pc + 4, P, a.tab_vec, rt + 4);
        }
    }
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
        const int h = h0 + i;
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = lo_bf16(xin[i][j]);
            x[2 * j + 1] = hi_bf16(xin[i][j]);
        }
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
        ss = row16_sum(ss);
        const float rr = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] * rr * wv[j];
        if constexpr (KIND != TABLE_NONE) {
            if constexpr (PAIRING == PAIR_INTERLEAVED) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool on = 8 * c + 2 * j < a.rot;
                    const float x0 = x[2 * j], x1 = x[2 * j + 1];
                    const float y0 = fmaf(rt[j].f00, x0, rt[j].f01 * x1);
                    const float y1 = fmaf(rt[j].f10, x0, rt[j].f11 * x1);
                    x[2 * j] = on ? y0 : x0;
                    x[2 * j + 1] = on ? y1 : x1;
                }
            } else {
                const int hc = a.rot >> 4, base = tid & 48;
                const bool first = c < hc, second = c >= hc && c < 2 * hc;
                const int partner = base + (first ? c + hc : (second ? c - hc : c));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = __shfl(x[j], partner, 64);
                    const float a0 = first ? x[j] : y, b0 = first ? y : x[j];
                    const float ya = fmaf(rt[j].f00, a0, rt[j].f01 * b0);
                    const float yb = fmaf(rt[j].f10, a0, rt[j].f11 * b0);
                    x[j] = first ? ya : (second ? yb : x[j]);
                }
            }
        }
        if (live && (is_q || is_k) && h < heads) {
            u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
            uint16_t* dst = is_q ? a.q_out + (int64_t)t * a.qo_rs + h * D : a.kp + off + (int64_t)h * a.pg.hs;
            *reinterpret_cast<u32x4*>(dst + 8 * c) = o;
        }
    }
}

template <int KIND>
hipError_t append_kind(const CacheAppendArgs& a, unsigned blocks, hipStream_t stream) {
    if (a.pairing == PAIR_SPLIT_HALF)
        hipLaunchKernelGGL((cache_append_kernel<KIND, PAIR_SPLIT_HALF>), dim3(blocks), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((cache_append_kernel<KIND, PAIR_INTERLEAVED>), dim3(blocks), dim3(256), 0, stream, a);
    return hipGetLastError();
}

// A workgroup copies 128 rows (32 KB) of one page of one layer's keys or values. FLAT: the page's rows lie next to each other, in
// whichever order: 8 loads of 16 bytes in flight a lane, through buffers of the page's size that end a short last chunk.
constexpr int COPY_ROWS = 128;
template <bool FLAT>
__global__ __launch_bounds__(256) void cache_copy_kernel(CacheCopyArgs a, int chunks, uint32_t rcp_chunks, uint32_t rcp_hk) {
    const int pair = div_small(blockIdx.x, chunks, rcp_chunks), chunk = blockIdx.x - pair * chunks;
    const int src = a.src[pair], dst = a.dst[pair];
    if (src < 0 || src >= a.pg.n_pages || dst < 0 || dst >= a.pg.n_pages || src == dst) return;
    uint16_t* base = (blockIdx.z ? a.vp : a.kp) + (int64_t)blockIdx.y * a.layer_stride;
    uint16_t *from = base + (int64_t)src * a.pg.ps, *to = base + (int64_t)dst * a.pg.ps;
    const int rows = a.HK << a.pg.shift;
    if constexpr (FLAT) {
        const __amdgpu_buffer_rsrc_t in = __builtin_amdgcn_make_buffer_rsrc(from, 0, rows * D * 2, 0x00020000);
        const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(to, 0, rows * D * 2, 0x00020000);
        const int off = chunk * COPY_ROWS * D * 2 + 16 * (int)threadIdx.x;
        u32x4 x[COPY_ROWS / 16];
#pragma unroll
        for (int u = 0; u < COPY_ROWS / 16; ++u) x[u] = __builtin_amdgcn_raw_buffer_load_b128(in, off + 4096 * u, 0, 2);
#pragma unroll
        for (int u = 0; u < COPY_ROWS / 16; ++u) __builtin_amdgcn_raw_buffer_store_b128(x[u], out, off + 4096 * u, 0, 2);
    } else {
        const int end = min(rows, (chunk + 1) * COPY_ROWS);
        for (int r = chunk * COPY_ROWS + (threadIdx.x >> 4); r < end; r += 16) {
            const int slot = div_small(r, a.HK, rcp_hk);
            const int64_t off = (int64_t)slot * a.pg.rs + (int64_t)(r - slot * a.HK) * a.pg.hs + 8 * (threadIdx.x & 15);
            *reinterpret_cast<u32x4*>(to + off) = *reinterpret_cast<const u32x4*>(from + off);
        }
    }
}

// A workgroup moves a sequence's rows in `hw` heads of one layer's keys or values, at most 16 U rows of a head: all of them are
// read before any is written, so a row may be the source of one move and the target of another.
constexpr int MOVE_ROWS = 256;
template <int U>
__global__ __launch_bounds__(256, U == 4 ? 8 : 4) void cache_move_kernel(CacheMoveArgs a, int hw) {
    const int b = blockIdx.x, h0 = blockIdx.z * hw, nh = min(hw, a.HK - h0);
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    if (s0 < 0 || s1 <= s0) return;
    const int n = min(min(s1, a.n) - s0, a.max_rows);
    if (n <= 0) return;
    uint16_t* base = ((blockIdx.y & 1) ? a.vp : a.kp) + (int64_t)(blockIdx.y >> 1) * a.layer_stride + 8 * (threadIdx.x & 15);
    u32x4 x[U];
    int64_t to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = 16 * u + (threadIdx.x >> 4);
        to[u] = -1;
        if (r < n * nh) {
            const int m = r / nh;
            const int64_t hoff = (int64_t)(h0 + r - m * nh) * a.pg.hs;
            const int64_t from = page_offset(a.pg, b, a.src[s0 + m]), dst = page_offset(a.pg, b, a.dst[s0 + m]);
            if (from >= 0 && dst >= 0) {
                to[u] = dst + hoff;
                x[u] = *reinterpret_cast<const u32x4*>(base + from + hoff);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (to[u] >= 0) *reinterpret_cast<u32x4*>(base + to[u]) = x[u];
}

}  // namespace

hipError_t launch_cache_append(const CacheAppendArgs& a, hipStream_t stream) {
    const int64_t hg = (a.H + HPG - 1) / HPG + 2 * ((a.HK + HPG - 1) / HPG);
    const int64_t blocks = (a.T * hg + 15) / 16;
    if (blocks <= 0 || blocks > 1 << 23) return hipErrorInvalidValue;   // (a grid's work-items are counted in 32 bits)
    switch (a.table_kind) {
        case TABLE_NONE: return append_kind<TABLE_NONE>(a, (unsigned)blocks, stream);
        case TABLE_COSSIN_F32: return append_kind<TABLE_COSSIN_F32>(a, (unsigned)blocks, stream);
        case TABLE_MAT2_BF16: return append_kind<TABLE_MAT2_BF16>(a, (unsigned)blocks, stream);
        case TABLE_MAT2_F32: return append_kind<TABLE_MAT2_F32>(a, (unsigned)blocks, stream);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_cache_copy(const CacheCopyArgs& a, hipStream_t stream) {
    const int rows = a.HK << a.pg.shift, chunks = (rows + COPY_ROWS - 1) / COPY_ROWS;
    const int64_t blocks = (int64_t)a.n * chunks;
    if (blocks > 1 << 23 || a.layers > 65535) return hipErrorInvalidValue;   // (a grid's work-items are counted in 32 bits)
    const int64_t page = (int64_t)1 << a.pg.shift;
    // (a buffer's size is 32 bits)
    const bool flat = rows <= 1 << 22 && ((a.pg.hs == D && a.pg.rs == (int64_t)a.HK * D) || (a.pg.rs == D && a.pg.hs == page * D));
    const dim3 grid((unsigned)blocks, (unsigned)a.layers, 2);
    if (flat) hipLaunchKernelGGL(cache_copy_kernel<true>, grid, dim3(256), 0, stream, a, chunks, rcp_small(chunks), rcp_small(a.HK));
    else hipLaunchKernelGGL(cache_copy_kernel<false>, grid, dim3(256), 0, stream, a, chunks, rcp_small(chunks), rcp_small(a.HK));
    return hipGetLastError();
}

hipError_t launch_cache_move(const CacheMoveArgs& a, hipStream_t stream) {
    // few moves: fewer registers a lane, so that twice the workgroups hide each other's chain of loads
    const int most = min(MOVE_ROWS, max(64, 16 * ((a.max_rows * a.HK + 15) / 16)));
    const int hw = min(a.HK, max(1, most / a.max_rows));
    if (a.max_rows > MOVE_ROWS || 2 * (int64_t)a.layers > 65535 || (a.HK + hw - 1) / hw > 65535) return hipErrorInvalidValue;
    const dim3 grid((unsigned)a.B, 2 * (unsigned)a.layers, (unsigned)((a.HK + hw - 1) / hw));
    const int rows = hw * a.max_rows;
    if (rows <= 64) hipLaunchKernelGGL(cache_move_kernel<4>, grid, dim3(256), 0, stream, a, hw);
    else if (rows <= 128) hipLaunchKernelGGL(cache_move_kernel<8>, grid, dim3(256), 0, stream, a, hw);
    else hipLaunchKernelGGL(cache_move_kernel<16>, grid, dim3(256), 0, stream, a, hw);
    return hipGetLastError();
}

}  // namespace lr
