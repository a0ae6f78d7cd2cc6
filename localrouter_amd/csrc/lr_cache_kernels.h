// Internal launch interface between the C ABI of the paged caches, the windowed and the packed attention (cache_abi.hip) and their
// kernels (attn_cache.hip, attn_cache_wide.hip, attn_cache8.hip, attn_packed.hip, cache_rows.hip, cache8_rows.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lr_kernels.h"

namespace lr {

// A pool of pages: row r of page p of kv head g at base + p * ps + r * rs + g * hs (elements), and the page tables of the
// sequences: position j of sequence b lies in row j & (page_size - 1) of page table[b * table_rs + (j >> shift)]. An entry
// outside [0, n_pages) holds no rows.
struct PageArgs {
    int64_t ps, rs, hs;
    const int* table;
    int64_t table_rs;
    int n_pages, shift, table_pages;
};

// Attention of query tokens over a sequence's keys, each token over its own range of them. Sources of keys (range_attn.inc's Source):
// rows of one sequence (key j of kv head g at k + j * k_rs + g * 128), rows of sequences packed end to end, pages, pages in 8 bits.
struct RangeAttnArgs {
    const uint16_t* q;   // bf16 [T][H][128], row stride q_rs
    uint16_t* out;       // bf16 [T][H][128], row stride o_rs
    const uint16_t* k;
    const uint16_t* v;
    int64_t q_rs, o_rs, k_rs, v_rs;
    int H, HK, G;
    float c;             // scale * log2(e)
    // rows: tokens i < W at positions p0 + i; frame f = p / frame sees keys of frames (f - window, f] below nkeys, and
    // keys below sinks of frames before
    int W, p0, nkeys, frame;
    // pages: tokens starts[b] .. starts[b + 1] of sequence b are its last positions before lens[b]; at most max_rows of them
    // a sequence and T in all, keys below max_keys
    PageArgs pg;
    const int* starts;
    const int* lens;
    const uint64_t* tree;   // [T][words]: bit x of a token's words: it sees the sequence's drafted token x; null: chains
    int B, T, max_rows, max_keys, words;
    int window, sinks;      // window 0 (not of rows): every earlier key
    // packed: tokens starts[b] .. starts[b + 1] are sequence b, its keys in the same rows of k and v; T rows in all
    // pages in 8 bits: k and v are bytes (the strides of pg too), 16 rows of a page and head with a scale 2^(byte - 127): of page p,
    // row r and head g at k_sc / v_sc + p * sc_ps + (r / 16) * HK + g
    const uint8_t* k_sc;
    const uint8_t* v_sc;
    int64_t sc_ps;
    // Split over the keys: with nsplit > 1 a block of rows is nsplit workgroups, each a part of its key tiles, whose unnormalised
    // rows, references and sums go to the parts (fp32 [slot][128] and [slot][2]).
    // attn_cache.hip: every block, `per` tiles a part, slots [block][part][row]; merged by the last part of a block to end, by the
    // flags [block][part] (merge_here), or by a second launch.
    // attn_cache_wide.hip: the blocks from number `whole` on, in the order in which an XCD's workgroups start (`local` blocks an
    // XCD, or with by_xcd 0 in all: see its kernel), `per` tiles a part or, per 0, equal parts; slots [block][row][part], merged
    // by a second launch.
    // attn_cache8.hip, places > 0: `places` workgroups with equal shares of all tiles, at least `per`; two slots each.
    // teams > 0 (attn_cache_wide.hip): cut by the sequences' own lengths into pieces of equal length, up to `teams` of them an XCD
    // whose `places` workgroups are resident at once. There, places without teams: an XCD's blocks in `places` equal shares.
    int nsplit, per, whole, local, merge_here, by_xcd, teams, places;
    float* part_o;
    float* part_ml;
    uint64_t* flags;
    // rcp_small of the divisors; nblk: blocks of rows a sequence and kv head
    uint32_t rcp_g, rcp_hk, rcp_frame, rcp_split, rcp_nblk;
    int nblk, hgroups;   // attn_cache8.hip: workgroups of several kv heads each, HK / heads of them (rcp_hk its)
};

// floor(2^32 / d), 2^32 - 1 for d = 1: what the kernels divide by d with.
inline uint32_t rcp_small(int64_t d) { return d > 1 ? (uint32_t)(((uint64_t)1 << 32) / (uint64_t)d) : 0xffffffffu; }

constexpr int RANGE_TILE = 32;              // attn_cache.hip: keys a tile,
constexpr int RANGE_STAGED = 2048;          // page-table entries a workgroup holds
constexpr int RANGE_WIDE_TILE = 64;         // attn_cache_wide.hip: the same, and
constexpr int RANGE_WIDE_STAGED = 3840;     // (both of its forms: 4 and 8 waves of 32 rows);
constexpr int RANGE_WIDE_PLACES = 32;       // workgroups of 8 waves that an XCD holds at once
constexpr int RANGE_WIDE_MIN_PAGE = 16;     // rows a page at least (of 16 rows: in pools of less than 4 GB),
constexpr int64_t RANGE_WIDE_MAX_RS = 1 << 23;   // and row strides (elements) below this
constexpr int64_t RANGE_MAX_BLOCKS = 1 << 22;    // workgroups a launch: a grid's work-items are counted in 32 bits

// The attention and, with a.nsplit > 1, the merge of its parts: attn_cache.hip in blocks of br rows (16, 32, 64 or 128), or
// attn_cache_wide.hip in workgroups of `waves` waves of 32 rows (the cut's tiles are each kernel's own).
hipError_t launch_range_attn(const RangeAttnArgs& a, bool paged, int br, hipStream_t stream);
hipError_t launch_range_wide(const RangeAttnArgs& a, bool paged, int waves, hipStream_t stream);
// Sequences packed end to end: attn_cache.hip's kernel of few rows in blocks of br (16 or 32), or attn_packed.hip's workgroups of `waves`
// waves of 32 rows. (nblk: the most blocks a sequence may have.)
hipError_t launch_packed_attn(const RangeAttnArgs& a, int br, hipStream_t stream);
hipError_t launch_packed_wide(const RangeAttnArgs& a, int waves, hipStream_t stream);
// Pages in 8 bits: attn_cache8.hip in blocks of br rows (16 or 32) of hw kv heads, kh waves each, or attn_cache_wide.hip.
constexpr int RANGE8_STAGED = 1024;
hipError_t launch_range8(const RangeAttnArgs& a, int br, int kh, int hw, hipStream_t stream);
hipError_t launch_range_wide8(const RangeAttnArgs& a, int waves, hipStream_t stream);

// cache_rows.hip
struct CacheAppendArgs {
    const uint16_t* q;   // bf16 [T][H][128] (null: no queries)
    const uint16_t* k;   // bf16 [T][HK][128]
    const uint16_t* v;
    uint16_t* q_out;
    uint16_t* kp;        // pages
    uint16_t* vp;
    int64_t q_rs, k_rs, v_rs, qo_rs;
    PageArgs pg;
    const int* starts;
    const int* lens;
    const int* pos;      // table row of each token; null: its position in its sequence
    int B, T, H, HK;
    const float* qw;     // fp32 [128] or null for ones
    const float* kw;
    int table_kind, pairing, rot, tab_rows, tab_vec;
    const void* ta;
    const void* tb;
    int64_t tab_stride;
    float eps;
};
hipError_t launch_cache_append(const CacheAppendArgs& a, hipStream_t stream);

// cache8_rows.hip: the same into pages in 8 bits (k and v pages as bytes, the strides of pg too) and their scales (RangeAttnArgs').
constexpr int GROUP8 = 16;   // rows of a page and head that share a scale
struct CacheAppend8Args {
    CacheAppendArgs at;      // (kp and vp: bytes)
    uint8_t* k_sc;
    uint8_t* v_sc;
    int64_t sc_ps;
};
hipError_t launch_cache_append8(const CacheAppend8Args& a, hipStream_t stream);

struct CacheCopyArgs {
    uint16_t* kp;        // (pages of `es` bytes an element: strides are elements)
    uint16_t* vp;
    PageArgs pg;         // no table
    int64_t layer_stride;
    const int* src;
    const int* dst;
    int n, layers, HK, es;
};
hipError_t launch_cache_copy(const CacheCopyArgs& a, hipStream_t stream);

// cache8_rows.hip: `bytes` scales of each page, of both tensors, in every layer.
struct CacheCopyScalesArgs {
    uint8_t* k_sc;
    uint8_t* v_sc;
    int64_t sc_ps, layer_stride;
    const int* src;
    const int* dst;
    int n, layers, n_pages, bytes;
};
hipError_t launch_cache_copy_scales(const CacheCopyScalesArgs& a, hipStream_t stream);

struct CacheMoveArgs {
    uint16_t* kp;
    uint16_t* vp;
    PageArgs pg;
    int64_t layer_stride;
    const int* starts;
    const int* src;
    const int* dst;
    int B, n, max_rows, layers, HK;
};
hipError_t launch_cache_move(const CacheMoveArgs& a, hipStream_t stream);

}  // namespace lr
