// The C ABI of the paged cache (include/lr_cache.h) and of the windowed attention (lr_attention_window_bf16 of
// include/lr_attn.h): argument validation, then launches on the caller's stream. Nothing here synchronises, allocates or keeps
// state.
#include <limits.h>

#include <algorithm>

#include "../../include/lr_cache.h"
#include "../../include/lr_cache8.h"
#include "abi_checks.h"
#include "lr_cache_kernels.h"

namespace {

using namespace lr::abi;

constexpr int MAX_POS = 1 << 30;

inline int shift_of(int page_size) { return __builtin_ctz((unsigned)page_size); }
inline bool page_size_ok(int ps) { return ps >= 1 && ps <= 65536 && (ps & (ps - 1)) == 0; }

// One level of a set of rows: `stride` elements times any of lo .. hi.
struct Level {
    int64_t stride, lo, hi;
};

// Whether d, less some sum of the levels' steps, is within `width` elements of 0: whether two rows of that width (a head's: 128) that far
// apart meet. Levels by falling stride; where a level's stride holds the extent of those below it (nested layouts) two of its steps are
// tried, else as many as reach, `left` in all: past that the answer is that they do.
bool rows_meet(int64_t d, const Level* levels, int n, int64_t width, int& left) {
    if (n == 0) return --left < 0 || (d > -width && d < width);
    const Level& l = levels[0];
    if (l.lo == l.hi) return rows_meet(d - l.lo * l.stride, levels + 1, n - 1, width, left);
    int64_t below = width - 1;
    for (int i = 1; i < n; ++i) below += std::max(-levels[i].lo, levels[i].hi) * levels[i].stride;
    const int64_t least = d - below;   // <= x * stride <= d + below
    for (int64_t x = std::max(least / l.stride + (least > 0 && least % l.stride), l.lo); x <= l.hi && x * l.stride <= d + below; ++x)
        if (rows_meet(d - x * l.stride, levels + 1, n - 1, width, left)) return true;
    return false;
}
// Whether no row of keys is one of values, d elements from them, nor a row of one layer one of another's. levels: the differences of two
// rows' numbers in every dimension, in any order, those of the layers (`layer` apart) among them.
bool apart(int64_t d, Level* levels, int n, int layers, int64_t layer, int64_t width) {
    std::sort(levels, levels + n, [](const Level& x, const Level& y) { return x.stride > y.stride; });
    int left = 4096;   // (nested layouts: at most 16)
    if (rows_meet(d, levels, n, width, left)) return false;
    if (layers == 1) return true;
    for (int i = 0; i < n; ++i)
        if (levels[i].stride == layer && levels[i].hi == layers - 1 && levels[i].lo == 1 - layers) {   // (another level of the same numbers is as good)
            levels[i].lo = 1;
            break;
        }
    return !rows_meet(0, levels, n, width, left);
}

// A pool of pages of elements of `es` bytes: aligned bases, strides that hold what they step over, no row of keys and values, or of
// two layers, the same.
bool pool_ok(const void* k, const void* v, int64_t page, int64_t row, int64_t head, int n_pages, int page_size, int HK,
             int layers = 1, int64_t layer = 0, int es = 2) {
    const int unit = 16 / es;
    if (!k || !v || !aligned(k, 16) || !aligned(v, 16) || n_pages < 1 || HK < 1 || !page_size_ok(page_size)) return false;
    if (page % unit || row % unit || head % unit || page < lr::D || row < lr::D || head < lr::D) return false;
    if (layers < 1 || layers > 65535 || layer % unit || (layers > 1 && layer < lr::D)) return false;
    auto far = [](int64_t stride, int64_t count) { return stride > ((int64_t)1 << 48) / count; };   // (no address space holds it)
    if (far(page, n_pages) || far(row, page_size) || far(head, HK) || far(layer, layers)) return false;
    // rows of a page token by token or head by head, pages apart from each other
    const bool by_token = row >= (HK - 1) * head + lr::D && page >= (page_size - 1) * row + (HK - 1) * head + lr::D;
    const bool by_head = head >= (page_size - 1) * row + lr::D && page >= (HK - 1) * head + (page_size - 1) * row + lr::D;
    if (!by_token && !by_head) return false;
    Level levels[4] = {{page, 1 - n_pages, n_pages - 1}, {row, 1 - page_size, page_size - 1}, {head, 1 - HK, HK - 1},
                       {layer, 1 - layers, layers - 1}};
    return apart((reinterpret_cast<intptr_t>(v) - reinterpret_cast<intptr_t>(k)) / es, levels, 4, layers, layer, lr::D);
}
// Whether a row of x (T of them, hx heads, x_rs apart) meets one of q (hq heads, q_rs apart): tensors that interleave, as the views of
// one packed projection do, share a span but no row.
bool packed_rows_meet(const void* q, int64_t q_rs, int hq, const void* x, int64_t x_rs, int hx, int T) {
    if (!overlap(rows_span(q, T, q_rs, hq), rows_span(x, T, x_rs, hx))) return false;
    const int64_t d = (reinterpret_cast<intptr_t>(x) - reinterpret_cast<intptr_t>(q)) / 2, last = T - 1;
    int left = 4096;
    if (last == 0 || q_rs == x_rs) {
        const Level levels[2] = {{q_rs, -last, last}, {lr::D, 1 - hx, hq - 1}};
        return rows_meet(d, levels, 2, lr::D, left);
    }
    Level levels[3] = {{q_rs, 0, last}, {x_rs, -last, 0}, {lr::D, 1 - hx, hq - 1}};
    if (x_rs > q_rs) std::swap(levels[0], levels[1]);
    return rows_meet(d, levels, 3, lr::D, left);
}
Span pool_span(const void* p, int layers, int64_t layer, int64_t page, int64_t row, int64_t head, int n_pages, int page_size,
               int HK, int es = 2) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return Span{lo, lo + es * (uintptr_t)((layers - 1) * layer + (n_pages - 1) * page + (page_size - 1) * row +
                                         (HK - 1) * head + lr::D)};
}
// The scales of a pool in 8 bits: pages of page_size / GROUP8 * HK bytes, `page` apart, layers `layer` apart; no byte of keys and values,
// or of two layers, the same.
bool page8_ok(int page_size, int64_t row) { return page_size >= lr::GROUP8 && row < lr::RANGE_WIDE_MAX_RS; }
int64_t scales_bytes(int page_size, int HK) { return (int64_t)(page_size / lr::GROUP8) * HK; }
Span scales_span(const void* p, int layers, int64_t layer, int64_t page, int n_pages, int page_size, int HK) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return Span{lo, lo + (uintptr_t)((layers - 1) * layer + (n_pages - 1) * page + scales_bytes(page_size, HK))};
}
bool scales_ok(const void* k, const void* v, int64_t page, int n_pages, int page_size, int HK, int layers = 1, int64_t layer = 0) {
    const int64_t bytes = scales_bytes(page_size, HK);
    if (!k || !v || page < bytes || page > ((int64_t)1 << 48) / n_pages || (layers > 1 && (layer < bytes || layer > ((int64_t)1 << 48) / layers)))
        return false;
    Level levels[2] = {{page, 1 - n_pages, n_pages - 1}, {layer, 1 - layers, layers - 1}};
    return apart(reinterpret_cast<intptr_t>(v) - reinterpret_cast<intptr_t>(k), levels, 2, layers, layer, bytes);
}
bool table_args_ok(const int* table, int64_t stride, int pages, int page_size, const int* starts, int B) {
    return table && aligned(table, 4) && starts && aligned(starts, 4) && B >= 1 && pages >= 1 && stride >= pages &&
           (int64_t)pages * page_size <= MAX_POS;
}
lr::PageArgs page_args(int64_t page, int64_t row, int64_t head, int n_pages, int page_size, const int* table, int64_t stride,
                       int pages) {
    lr::PageArgs g{};
    g.ps = page; g.rs = row; g.hs = head;
    g.table = table; g.table_rs = stride; g.table_pages = pages;
    g.n_pages = n_pages; g.shift = shift_of(page_size);
    return g;
}

// ------------------------------------------------------------------------------------------------ range attention
// How a call is cut: the kernel (wide: 0, or the waves of the kernel of attn_cache_wide.hip; br: attn_cache.hip's rows a block) and its
// blocks over the keys (RangeAttnArgs: nsplit, per, whole, local, nblk, teams, places), the rows of the parts and their flags.
struct Cut {
    int wide, br, nsplit, per, nblk, merge_here, by_xcd, teams, places, kh, hw;
    int64_t whole, local, part_rows, flags;   // (blocks of every sequence and kv head: past 32 bits before the launch is refused)
};

// The most key tiles of bt keys that a block of rows needs: of `span` keys beside the first `sinks`, of `keys` in all.
int64_t tiles_of(int64_t keys, int64_t span, int64_t sinks, int bt) {
    return std::min((keys + bt - 1) / bt, (std::min(sinks, keys) + bt - 1) / bt + span / bt + 2);
}

// Whether blocks of 32 rows are taken, each reading its keys by itself, in place of 64 or of attn_cache_wide.hip's 128 and 256: one
// round of the CUs, and few keys in all. Us with blocks of 32 / without: 64 rows over 8 kv heads, 1 sequence of 500 keys 10.4 /
// 16.6, of 16,000 22 / 30, 8 and 16 of 4,000 33 / 42 and 62 / 66, 8 of 16,000 (64,000 tiles) 120 / 112; 128 rows over 8, 1 of 300
// 9.5 / 15.2, of 16,000 (16,000 tiles) 26 / 31, 4 of 1,900 20 / 26, of 16,000 94 / 82; 96 over 2, 4 of 6,000 (4,500) 17 / 24, of
// 16,000 (12,000) 39 / 30; 600 over 4, 1 of 1,900 17 / 24, of 16,000 49 / 47; 16 of 300 (1,216 blocks) 42 / 21.
bool few_rows(int64_t rows, int64_t pairs, int64_t tiles) {
    const int64_t blocks = (rows + 31) / 32 * pairs;
    return rows <= 32 || (blocks <= 256 && blocks * tiles <= (rows <= 64 ? 32000 : 12000));
}

// attn_cache.hip: every block in parts of `per` tiles, one workgroup a CU; rows of a kv head a sequence, pairs: sequences x kv heads.
// Blocks of 16 and 32 rows (the kernel of few rows) up to 32 rows a kv head, and of 32 above while there are few blocks with few
// keys, which every block reads (few_rows). Elsewhere blocks of 64 and 128 rows.
// Parts of the kernel of few rows: as few as cost least, when a round of eight tiles takes 1.2 to 1.6 us. Of at most 16 rows the last
// part to end merges them all in ~2.5 us, eight more of them in another 1.2 (rows of 600 keys 1 part 6.3, 3 7.3; 1,100 3 7.8, 5 7.4;
// pages of 500 1 7.6, 2 8.6, 4 8.1; 1,900 2 parts 12.4, 4 9.9, 8 8.7, 15 9.5; 6,000 6 14.1, 12 12.4, 24 13.1; 16,000 over 2 heads
// 16 14.5, 32 13.0, 63 15.4, over 8 16 18.5, 32 19.1). Of more rows a second launch does,
// in ~2.5 us and with each part's stores (20 rows: 500 keys 1 part 10.1, 2 11.5; 1,900 4 13.1, 8 11.8, 16 12.7; 6,000 8 16.7,
// 16 15.9, 32 18.2). In the same launch / by a second: 24 parts of 4 rows 13.1 / 14.5, 63 of 8 15.4 / 17.5, 32 of 16 20.9 / 22.1, 8 of
// 20 12.5 / 11.8, 8 of 32 13.4 / 11.9, 2 of 64 19.1 / 16.0.
// The other kernel: parts of 8 tiles at least, merged by a second launch.
Cut cut_small(int64_t rows, int64_t pairs, int64_t tiles, int page_size) {
    const int64_t br = rows <= 16 ? 16 : few_rows(rows, pairs, tiles) ? 32 : rows <= 64 ? 64 : 128, base = (rows + br - 1) / br * pairs;
    const int64_t staged = page_size ? lr::RANGE_STAGED / std::max(1, lr::RANGE_TILE / page_size) : INT_MAX;
    int64_t ns = std::max<int64_t>(1, std::min(256 / base, (tiles + 4) / 8));
    if (br <= 32) {
        auto cost = [&](int64_t n) {
            const double rounds = (double)(((tiles + n - 1) / n + 7) / 8);
            if (br == 16) return 1.25 * rounds + (n > 1 ? 1.4 + 1.2 * (double)((n + 7) / 8) : 0.0);
            return 1.4 * rounds + (n > 1 ? 2.4 + 0.18 * (double)n : 0.0);
        };
        const int64_t most = std::max<int64_t>(1, std::min(256 / base, (tiles + 7) / 8));
        ns = 1;
        for (int64_t n = 2; n <= most; ++n)
            if (cost(n) < cost(ns)) ns = n;
    }
    const int64_t per = std::max<int64_t>(1, std::min((tiles + ns - 1) / ns, staged));
    ns = std::max<int64_t>(1, (tiles + per - 1) / per);
    Cut c{};
    c.br = (int)br; c.nsplit = (int)ns; c.per = (int)per;
    c.nblk = (int)((rows + br - 1) / br);
    c.merge_here = br == 16 && ns * std::min(rows, br) <= 1024;
    c.part_rows = ns > 1 ? base * ns * br : 0;
    c.flags = c.merge_here && ns > 1 ? base * ns : 0;
    return c;
}

// attn_cache_wide.hip. Two workgroups of 4 waves are resident on a CU, 64 on an XCD. Where the last round of them is not full,
// its blocks may be cut: a block alone on its CU takes ~1.1 us a tile, beside another 1.8, and parts cost a launch (~6 us) and
// their rows written and read (2,319 tokens x 32 heads over 8, 512 + 72 blocks, windows of 1,024, 2,048 and 8,192: 66.6, 114 and 400
// us uncut, 63.4, 99 and 309 cut). `waves`: given by the caller (8-bit
// pages), or 0; a block of 8 that it gives takes 1.9 us a tile, of 4 1.8 also alone (4 chunks of 100 tokens over 3,000, 32 heads over 8, whole 56
// us, in parts 47).
Cut cut_wide(int64_t rows, int64_t pairs, int64_t tiles, int page_size, bool by_xcd, int waves = 0) {
    const int64_t big = (rows + 255) / 256 * pairs;
    Cut c{};
    // 8 waves: half the keys and values moved into LDS. Long ranges that fill the rounds of 256 such workgroups (us, 8 / 4
    // waves: 4,096 tokens x 32 heads, windows of 8,192 and 1,024 tokens 493 / 511 and 100 / 92; 3,000 x 32, 1.5 rounds, 91 / 82).
    c.wide = waves ? waves : tiles >= 64 && big >= 256 && (big % 256 == 0 || big >= 1024) ? 8 : 4;
    const int br = 32 * c.wide, xcds = by_xcd ? 8 : 1, round = (c.wide == 8 ? 256 : 512) / xcds;
    c.by_xcd = by_xcd;
    c.nblk = (int)((rows + br - 1) / br);
    c.local = (pairs + xcds - 1) / xcds * c.nblk;
    c.whole = c.local;
    c.nsplit = 1;
    const int64_t staged = page_size ? lr::RANGE_WIDE_STAGED / std::max(1, lr::RANGE_WIDE_TILE / page_size) : INT_MAX;
    int64_t tail = c.local % round, ns = 1;
    // (under pages the lengths are the device's: only launches of less than a round are cut, into parts of a fixed length)
    if (page_size && c.local > round) tail = 0;
    if (tail) {
        auto cost = [&](int64_t n) {
            return (double)((tiles + n - 1) / n) * (waves == 8 ? 1.9 : waves == 4 || 2 * tail * n > round ? 1.8 : 1.1) +
                   (n > 1 ? 6.0 + 2.0 * (double)(tail * xcds * br * n) * lr::D * 4 / 5e6 : 0.0);
        };
        for (int64_t n = 2; n <= std::min<int64_t>(std::min(round / tail, tiles / 2), 64); ++n)
            if (cost(n) < cost(ns)) ns = n;
    }
    if (page_size) {
        const int64_t per = std::max<int64_t>(1, std::min((tiles + ns - 1) / ns, staged));
        ns = std::max<int64_t>(1, (tiles + per - 1) / per);
        c.per = (int)per;
        tail = c.local;
    }
    if (ns > 1) {
        c.nsplit = (int)ns;
        c.whole = c.local - tail;
        c.part_rows = tail * xcds * br * ns;
    }
    return c;
}

// attn_cache_wide.hip's pieces of equal length, for batches of long sequences in at most three rounds of blocks of more than 128 rows
// (us with whole blocks / pieces; 8 kv heads, lengths from N / 2, from N / 20, all N): 16 x 256 rows, N 8,000 162 / 138, 132 / 103,
// 174 / 168; N 30,000 535 / 445, 507 / 355, 605 / 521; 40 x 256, N 30,000 1160 / 957, 897 / 689, 1965 / 1257; 16 x 512, N 8,000
// 222 / 219, 217 / 160, 270 / 263; N 30,000 820 / 785, 782 / 629, 926 / 932. Not short ones (40 x 256, N 2,000 61 / 91 from N / 20),
// nor of 128 rows (16 x 128, N 30,000 368 / 385, 339 / 303, 409 / 474). Workgroups of 256 rows where they hold as few empty rows as
// those of 128 (16 x 320 rows over 2 heads, N 30,000, of 256 / of 128: 258 / 179, 209 / 168, 303 / 224; whole blocks 193, 189, 206).
void cut_pieces(Cut& c, int64_t rows, int64_t pairs, int64_t tiles, int page_size) {
    if (rows <= 128 || pairs % 8 || tiles < 64) return;
    const int waves = (rows + 255) / 256 * 2 == (rows + 127) / 128 ? 8 : 4;
    const int64_t P = pairs / 8, places = waves == 8 ? 32 : 64, nblk = (rows + 32 * waves - 1) / (32 * waves);
    // (nblk: of more blocks a pair is balanced without, and the parts would take gigabytes)
    if (P > 48 || nblk > places / 8 || P * nblk > 3 * places || P * nblk * tiles < 60 * places) return;
    const int64_t teams = std::min<int64_t>(places, 64 - P), least = std::max<int64_t>(1, std::min(teams, places / nblk));
    const int64_t longest = std::max<int64_t>(16, (P * tiles + least - 1) / least);   // what a workgroup holds page entries for
    if (longest * std::max(1, lr::RANGE_WIDE_TILE / page_size) > lr::RANGE_WIDE_STAGED) return;
    c.wide = waves; c.nblk = (int)nblk; c.by_xcd = 1;
    c.nsplit = 1; c.per = 0;
    c.teams = (int)teams; c.places = (int)places;
    c.part_rows = 8 * (P + teams) * nblk * 32 * waves;
}

Cut window_cut(int W, int H, int HK, int nkeys, int window, int sinks, int frame, bool narrow) {
    const int64_t rows = (int64_t)W * (H / HK), tokens = std::min<int64_t>(W, 256 / (H / HK) + 2);
    const int64_t span = std::min((int64_t)window + 2, (int64_t)MAX_POS) * frame + tokens;
    const int64_t tiles = tiles_of(nkeys, span, sinks, lr::RANGE_TILE);
    if (narrow && rows > 64 && !few_rows(rows, HK, tiles))
        return cut_wide(rows, HK, tiles_of(nkeys, span, sinks, lr::RANGE_WIDE_TILE), 0, HK % 8 == 0);
    return cut_small(rows, HK, tiles, 0);
}
Cut cache_cut(int B, int max_rows, int max_keys, int H, int HK, int page_size, int window, int sinks, bool narrow) {
    const int64_t rows = (int64_t)max_rows * (H / HK), pairs = (int64_t)B * HK;
    const int64_t span = window ? (int64_t)window + max_rows + 1 : max_keys;
    const int64_t tiles = tiles_of(max_keys, span, sinks, lr::RANGE_TILE);
    if (narrow && rows > 64 && page_size >= lr::RANGE_WIDE_MIN_PAGE && !few_rows(rows, pairs, tiles)) {
        const int64_t wide_tiles = tiles_of(max_keys, span, sinks, lr::RANGE_WIDE_TILE);
        Cut c = cut_wide(rows, pairs, wide_tiles, page_size, pairs % 8 == 0 || pairs >= 64);
        if (B > 1 && !window) cut_pieces(c, rows, pairs, wide_tiles, page_size);
        return c;
    }
    return cut_small(rows, pairs, tiles, page_size);
}
// Sequences packed end to end; the host knows how many and how many rows in all. Blocks of 16 rows (attn_cache.hip, whose eight waves
// share a block's keys) while all of them are resident at once; else blocks of 32 rows or the stream of blocks of 128 (attn_packed.hip),
// by what they cost when the sequences are of one length: a round of blocks of 32 starts and ends in ~5 us and takes 0.75 per 256
// keys of its longest; the blocks of 128 take ~6 and 1.2 per 64 keys of the longest, or what the GPU does in all. Us with 16 / 32 / 128
// rows: one of 1,000 tokens, one head, 9.2 / 11.7 / 25.7; one of 300, 32 heads over 8, 14.0 / 11.2 / 13.2; 891 tokens of 2, 32 over 8, 37
// / 28 / 19; 4,017 of 2, 4 over 1, 41 / 28 / 60; one of 7,000, 4 over 1, 149 / 91 / 141, 8 over 8 273 / 173 / 156; 611 of 18, 16 over 8,
// 12.5 / 11.0 / 7.8. Under a window a block reads that and its own tokens (us with 32 / 128 rows, windows of 64, 256 and 1,024: one of 7,000, 4
// over 1, 25 / 12, 34 / 17, 48 / 32; one of 4,000, 8 over 2, 24 / 12, 32 / 17, 46 / 31; one of 500, 32 over 8, 64 11.2 / 10.6, but one of
// 8,000, one head, 7.6 / 12.2, 9.5 / 16.8, 14.0 / 30.9).
// Blocks of 256 where there are many and each XCD has kv heads of its own, whose keys its workgroups move half as often (us with 128 /
// 256 rows: 10,900 tokens of 19, 32 over 8, 120 / 116; 58,000 of 60, 16 over 8, 441 / 414; one of 4,096, 32 over 8, 147 / 139; of 53,000 of 38,
// 8 over 8, 283 / 289; 43,000 of 27, 8 over 2, 217 / 223).
Cut packed_cut(int B, int T, int H, int HK, int window, int sinks) {
    const int64_t G = H / HK, rows = (int64_t)T * G;
    auto blocks = [&](int64_t br) { return (rows / br + B) * HK; };
    Cut c{};
    c.nsplit = 1; c.per = MAX_POS;
    const double len = (double)T / B;
    // the most keys of a block of br rows, and twice their mean: the first tokens see fewer, of a prompt without a window half as many
    auto most = [&](int64_t br) { return window ? std::min(len, (double)window + (double)sinks + (double)br / (double)G) : len; };
    auto twice = [&](int64_t br) { return most(br) < len ? 2 * most(br) - most(br) * most(br) / len : len; };
    const double t32 = 1.1 * (double)blocks(32) / 256 * (5.0 + 0.0029 * twice(32)),
                 t128 = std::max(6.0 + 1.2 / 64 * most(128), (double)blocks(128) / 512 * (6.0 + 1.75 / 128 * twice(128)));
    if ((B == 1 ? (rows + 15) / 16 : rows / 16 + (3 * B + 3) / 4) * HK <= 256) c.br = 16;   // (all resident, but for a few of ragged batches)
    else if (t32 <= t128) c.br = 32;
    else c.wide = blocks(128) >= 1024 && HK % 8 == 0 && G > 1 ? 8 : 4;
    const int64_t br = c.wide ? 32 * c.wide : c.br;
    c.nblk = (int)((rows + br - 1) / br);
    return c;
}
// Pages in 8 bits, few rows (attn_cache8.hip): blocks of 16 or 32 rows of hw kv heads, kh waves a head.
// Batches of one block a sequence and kv head with much to read: equal shares of all tiles, whatever the lengths, for one workgroup a CU
// of 8 waves and two heads, or of an odd number of heads two of 4 waves and one. Us with whole pairs or parts as below / shares, 32 heads
// over 8, lengths from half to N: 4 sequences, N 24,000 39.8 / 41.6; 16, 6,000 33.1 / 37.7; 64, 1,500 32.7 / 38.6; 32, 6,000 66.8 / 58.9;
// 16, 24,000 146 / 121; 64, 6,000 144 / 124, 24,000 558 / 440 (5.5 TB/s); 27 rows, 16 of 6,000 38.9 / 47.7, 40 112 / 104, 20 of 12,000
// 123 / 98.8.
// Blocks of 16 rows also where that makes more of them, unless it is the bytes that count: keys are read once a block, but its chain of
// steps and the merge of its parts are shorter (us in blocks of 32 / 16, 32 heads over 8: 8 tokens over 60 keys 7.6 / 5.7, 400 11.1 / 8.7, 3,000
// 15.1 / 12.3, 30,000 25.6 / 24.6; 16 sequences of 8 over 1,000 17.7 / 12.2; 8 of 8 over 3,000 20.2 / 19.9, but 4 over 9,000 23.7 / 24.5; 480
// blocks of 64 keys 8.0 / 6.9, 512 of 400 11.4 / 11.3).
// Otherwise parts, as few as cost least (cut_small's costs: what a round takes is the chain of loads and instructions, not the bytes),
// by 8 waves of one head; of at most 4 tiles, or of more blocks than CUs, by 4 (8 sequences of 4 tokens over 60 keys 5.9 / 5.7); of more
// than three a CU by 2 of each of two heads, whose rows are next to each other (us with 8 / 4 / 2 x 2: 64 x 300 keys 14.2 / 10.8 / 11.0,
// 64 x 1,500 35.9 / 32.7 / 35.2, 128 x 1,500 80 / 68 / 61.5, 256 x 1,500 158 / 137 / 129; 32 x 1,500 20.1 / 20.9 / 33.4).
Cut cut_small8(int64_t rows, int64_t B, int64_t HK, int64_t tiles, int page_size) {
    Cut c{};
    const int64_t blocks16 = (rows + 15) / 16 * B * HK;
    c.br = rows <= 16 || (blocks16 <= 512 && blocks16 * tiles <= 14000) ? 16 : 32;
    const int64_t nblk = (rows + c.br - 1) / c.br, base = nblk * B * HK;
    c.nblk = (int)nblk;
    c.nsplit = 1;
    const int64_t staged = lr::RANGE8_STAGED / std::max(1, lr::RANGE_TILE / page_size), paired = HK % 2 ? 1 : 2;
    if (nblk == 1 && B <= 64 && base * tiles >= 32768 && base * tiles <= MAX_POS) {
        const int64_t places = paired == 2 ? 256 : 512, share = (base / paired * tiles + places - 1) / places;
        if (share <= staged) {   // (what a workgroup holds page entries for)
            c.kh = 4; c.hw = (int)paired;
            c.places = (int)places;
            c.per = 4;   // at least so many tiles a share
            // (us of blocks of 32 rows merged by a second launch / by the last part to end: 40 sequences of up to 6,000 104 / 102, 64 151 / 145, but
            // 20 of 12,000, whose pairs have more parts, 99.5 / 99.7, 16 of 24,000 140.8 / 142.4)
            c.merge_here = c.br == 16 || 2 * (base / paired) >= places;
            c.part_rows = 2 * places * c.br * paired;
            c.flags = c.merge_here ? 2 * places : 0;
            return c;
        }
    }
    int64_t ns = 1;
    c.kh = base <= 256 && tiles > 4 ? 8 : 4; c.hw = 1;
    if (base > 768 && paired == 2 && c.br == 16) c.kh = c.hw = 2;
    if (base <= 256) {
        auto cost = [&](int64_t n) {
            const double rounds = (double)(((tiles + n - 1) / n + 7) / 8);
            if (c.br == 16) return 1.25 * rounds + (n > 1 ? 1.4 + 1.2 * (double)((n + 7) / 8) : 0.0);
            return 1.4 * rounds + (n > 1 ? 2.4 + 0.18 * (double)n : 0.0);
        };
        const int64_t most = std::max<int64_t>(1, std::min(256 / base, (tiles + 7) / 8));
        for (int64_t n = 2; n <= most; ++n)
            if (cost(n) < cost(ns)) ns = n;
    }
    const int64_t per = std::max<int64_t>(1, std::min((tiles + ns - 1) / ns, staged));
    ns = std::max<int64_t>(1, (tiles + per - 1) / per);
    c.nsplit = (int)std::min<int64_t>(ns, INT_MAX); c.per = (int)per;
    c.merge_here = c.br == 16 && ns * std::min<int64_t>(rows, c.br) <= 1024;
    c.part_rows = ns > 1 ? base * ns * c.br : 0;
    c.flags = c.merge_here && ns > 1 ? base / c.hw * ns : 0;
    return c;
}
Cut cache8_cut(int B, int max_rows, int max_keys, int H, int HK, int page_size, int window, int sinks) {
    const int64_t rows = (int64_t)max_rows * (H / HK), pairs = (int64_t)B * HK;
    const int64_t span = window ? (int64_t)window + max_rows + 1 : max_keys;
    const int64_t tiles = tiles_of(max_keys, span, sinks, lr::RANGE_TILE);
    // The kernel of few rows while it has few blocks with few keys, which every block reads (us with it / without: 1 sequence of 256 tokens
    // behind 1,750, 32 heads over 8, 22 / 32, of 128 behind 3,900 29 / 37, 4 of 100 behind 900 22 / 34, 1 of 400 from an empty cache 13 / 18; 4
    // of 64 behind 3,000, 24,000 tiles in all, 29 / 35, 1 of 128 behind 7,900, 32,000, 42 / 44; 4 of 64 behind 9,000, 72,000, 73 / 55; 784 blocks
    // of 34 tiles 39 / 37, 1,152 of 30 42 / 37).
    const int64_t blocks32 = (rows + 31) / 32 * pairs;
    if (rows <= 64 || (blocks32 <= 600 && blocks32 * tiles <= 30000)) return cut_small8(rows, B, HK, tiles, page_size);
    const int64_t wide_tiles = tiles_of(max_keys, span, sinks, lr::RANGE_WIDE_TILE);
    // Workgroups of 8 waves, which convert each key half as often, unless ranges are short or rows would be empty (us with 4 / 8 waves:
    // one of 2,048 tokens behind 28,000 987 / 925, of 16,384 from an empty cache 2,207 / 2,091, 3 trees of 94 over 17,000 105 / 93; from
    // an empty cache 2,048 tokens 62.7 / 69.8, 3,000 103 / 107; 64 x 256 156 / 181).
    const int64_t n128 = (rows + 127) / 128, n256 = (rows + 255) / 256;
    const int waves = wide_tiles >= 64 && 16 * n256 <= 9 * n128 ? 8 : 4;
    Cut c = cut_wide(rows, pairs, wide_tiles, page_size, pairs % 8 == 0 || pairs >= 64, waves);
    if (B > 1 && !window) cut_pieces(c, rows, pairs, wide_tiles, page_size);
    // Blocks in equal shares (attn_cache_wide.hip, BlockPieces) where whole blocks, or their parts, would leave a quarter of an XCD's 32
    // places empty (us whole or in parts / in shares: 22 blocks of 90 tiles 185 / 160, 18 of 125 237 / 171, 33 of 141 432 / 319, 46 of 188
    // 606 / 547, 11 of 79 95 / 87; 24 of 66 133 / 136, and fuller: 27 of 141 272 / 270, 30 of 141 271 / 299, 61 of 250 851 / 925). They count as
    // equally long: chunks behind three times as many positions as their own, or more (71 of 141, half of them its own: 586 / 551, but
    // 54 of 141 431 / 488).
    const int64_t P = pairs / 8, blocks = P * n256, all = blocks * wide_tiles;
    if (waves == 8 && pairs % 8 == 0 && P <= 64 && blocks <= 128 && !window && !c.teams && 4 * (int64_t)max_rows <= max_keys) {
        const int64_t places = lr::RANGE_WIDE_PLACES, share = std::max<int64_t>(16, (all + places - 1) / places);
        const int64_t used = blocks * std::max<int64_t>(1, places / blocks), rounds = (blocks + places - 1) / places * places;
        if (4 * used <= 3 * rounds && std::min(share, wide_tiles) * std::max(1, lr::RANGE_WIDE_TILE / page_size) <= lr::RANGE_WIDE_STAGED) {
            c = Cut{};
            c.wide = 8; c.nblk = (int)n256; c.by_xcd = 1;
            c.nsplit = 1; c.places = (int)places;
            c.part_rows = 8 * (places + blocks) * 256;
        }
    }
    return c;
}
// Whether the grid of attn_cache_wide.hip's launch holds its workgroups (attn_cache.hip's counts its own, launch_blocks).
bool launch_fits(const Cut& c) {
    return !c.wide || (c.by_xcd ? 8 : 1) * (c.whole + (c.local - c.whole) * c.nsplit) <= lr::RANGE_MAX_BLOCKS;
}
size_t part_bytes(const Cut& c) {
    return (((size_t)c.part_rows * lr::D * 4 + 255) & ~(size_t)255) + (((size_t)(c.part_rows + c.flags) * 8 + 255) & ~(size_t)255);
}
void set_cut(lr::RangeAttnArgs& a, void* ws, const Cut& c) {
    a.nsplit = c.nsplit; a.per = c.per; a.nblk = c.nblk;
    a.whole = (int)c.whole; a.local = (int)c.local;   // (launch_fits; attn_cache.hip has no use for them)
    a.merge_here = c.merge_here; a.by_xcd = c.by_xcd;
    a.teams = c.teams; a.places = c.places;
    a.rcp_split = lr::rcp_small(c.nsplit);
    a.rcp_nblk = lr::rcp_small(c.nblk);
    a.rcp_g = lr::rcp_small(a.G);
    a.rcp_hk = lr::rcp_small(a.HK);
    a.part_o = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + (((size_t)c.part_rows * lr::D * 4 + 255) & ~(size_t)255));
    a.flags = reinterpret_cast<uint64_t*>(a.part_ml + 2 * c.part_rows);
}

int launch(const lr::RangeAttnArgs& a, bool paged, const Cut& c, lr_stream_t stream) {
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return (int)(c.wide ? lr::launch_range_wide(a, paged, c.wide, s) : lr::launch_range_attn(a, paged, c.br, s));
}

bool window_sizes_ok(int W, int H, int HK, int nkeys, int window, int sinks, int frame) {
    return W >= 1 && H >= 1 && HK >= 1 && H % HK == 0 && nkeys >= 1 && nkeys <= MAX_POS && window >= 1 && sinks >= 0 &&
           frame >= 1 && (int64_t)W * (H / HK) <= MAX_POS;
}
bool cache_sizes_ok(int B, int T, int max_rows, int max_keys, int H, int HK, int page_size, int window, int sinks) {
    return B >= 1 && B <= 65535 && T >= 1 && T <= MAX_POS && max_rows >= 1 && max_rows <= MAX_POS && max_keys >= 1 &&
           max_keys <= MAX_POS && H >= 1 && HK >= 1 && H % HK == 0 && page_size_ok(page_size) && window >= 0 && sinks >= 0 &&
           (int64_t)max_rows * (H / HK) <= MAX_POS;
}

// What both attentions over pages check, and their arguments but for the cut; es: bytes of a page's element. spans: the rows of out and
// q, and the pools.
bool attention_args(lr::RangeAttnArgs& a, Span (&spans)[4], int es, const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                    const void* k_pages, const void* v_pages, int64_t page_stride, int64_t row_stride, int64_t head_stride, int n_pages,
                    int page_size, const int* page_table, int64_t table_stride, int table_pages, const int* starts, const int* lens, int B,
                    int T, int max_rows, int max_keys, int H, int HK, const uint64_t* tree, int words, int window, int sinks, float scale) {
    if (!cache_sizes_ok(B, T, max_rows, max_keys, H, HK, page_size, window, sinks) || !scale_ok(scale)) return false;
    if (!rows_ok(q, q_row_stride, H) || !rows_ok(out, out_row_stride, H)) return false;
    if (!pool_ok(k_pages, v_pages, page_stride, row_stride, head_stride, n_pages, page_size, HK, 1, 0, es)) return false;
    if (!table_args_ok(page_table, table_stride, table_pages, page_size, starts, B) || !lens || !aligned(lens, 4))
        return false;
    if (tree && (words < 1 || words > 64 || !aligned(tree, 8))) return false;
    const Span so = rows_span(out, T, out_row_stride, H), sq = rows_span(q, T, q_row_stride, H),
               sk = pool_span(k_pages, 1, 0, page_stride, row_stride, head_stride, n_pages, page_size, HK, es),
               sv = pool_span(v_pages, 1, 0, page_stride, row_stride, head_stride, n_pages, page_size, HK, es);
    if (overlap(so, sq) || overlap(so, sk) || overlap(so, sv)) return false;
    spans[0] = so; spans[1] = sq; spans[2] = sk; spans[3] = sv;
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k_pages);
    a.v = static_cast<const uint16_t*>(v_pages);
    a.out = static_cast<uint16_t*>(out);
    a.q_rs = q_row_stride; a.o_rs = out_row_stride;
    a.H = H; a.HK = HK; a.G = H / HK;
    a.c = scale * 1.4426950408889634f;
    a.pg = page_args(page_stride, row_stride, head_stride, n_pages, page_size, page_table, table_stride, table_pages);
    a.starts = starts; a.lens = lens; a.tree = tree; a.words = tree ? words : 0;
    a.B = B; a.T = T; a.max_rows = max_rows; a.max_keys = max_keys;
    a.window = std::min(window, MAX_POS); a.sinks = window ? std::min(sinks, MAX_POS) : 0;
    return true;
}
// The workspace of a call that is cut as c, apart from everything it reads and writes.
bool workspace_ok(const Cut& c, void* workspace, size_t workspace_bytes, const Span* spans, int n) {
    const size_t need = part_bytes(c);
    if (!need) return true;
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < need) return false;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(workspace);
    for (int i = 0; i < n; ++i)
        if (overlap(Span{lo, lo + need}, spans[i])) return false;
    return true;
}

// What both appends check, and their arguments; es: bytes of a page's element.
bool append_args(lr::CacheAppendArgs& a, int es, const void* q, const void* k, const void* v, int64_t q_row_stride, int64_t k_row_stride,
                 int64_t v_row_stride, void* q_out, int64_t q_out_row_stride, void* k_pages, void* v_pages, int64_t page_stride,
                 int64_t row_stride, int64_t head_stride, int n_pages, int page_size, const int* page_table, int64_t table_stride,
                 int table_pages, const int* starts, const int* lens, const int* positions, int B, int T, int H, int HK,
                 const float* q_norm_w, const float* k_norm_w, int table_kind, const void* table_a, const void* table_b,
                 int64_t table_row_stride, int table_rows, int pairing, int rot_dim, float eps) {
    const int rot = rot_dim == 0 ? lr::D : rot_dim;
    if (T < 1 || T > MAX_POS || HK < 1 || (q && H < 1) || !(eps >= 0.0f) || !isfinite(eps)) return false;
    if (!rows_ok(k, k_row_stride, HK) || !rows_ok(v, v_row_stride, HK)) return false;
    if (q && (!rows_ok(q, q_row_stride, H) || !rows_ok(q_out, q_out_row_stride, H))) return false;
    if (!pool_ok(k_pages, v_pages, page_stride, row_stride, head_stride, n_pages, page_size, HK, 1, 0, es)) return false;
    if (!table_args_ok(page_table, table_stride, table_pages, page_size, starts, B) || !lens || !aligned(lens, 4) ||
        (positions && !aligned(positions, 4)))
        return false;
    if ((q_norm_w && !aligned(q_norm_w, 16)) || (k_norm_w && !aligned(k_norm_w, 16))) return false;
    if (!table_ok(table_kind, table_a, table_b, table_row_stride, rot, pairing, 16)) return false;
    if (table_kind != LR_TABLE_NONE && table_rows < 1) return false;
    const Span pk = pool_span(k_pages, 1, 0, page_stride, row_stride, head_stride, n_pages, page_size, HK, es),
               pv = pool_span(v_pages, 1, 0, page_stride, row_stride, head_stride, n_pages, page_size, HK, es),
               sk = rows_span(k, T, k_row_stride, HK), sv = rows_span(v, T, v_row_stride, HK);
    if (overlap(pk, sk) || overlap(pk, sv) || overlap(pv, sk) || overlap(pv, sv)) return false;
    if (q) {
        const Span sq = rows_span(q, T, q_row_stride, H), so = rows_span(q_out, T, q_out_row_stride, H);
        if (overlap(pk, sq) || overlap(pv, sq) || overlap(pk, so) || overlap(pv, so)) return false;
        if (!(q_out == q && q_out_row_stride == q_row_stride) && overlap(sq, so)) return false;
        // (in place on the queries of a packed projection, whose keys and values have columns of their own)
        if (q_out == q && q_out_row_stride == q_row_stride
                ? packed_rows_meet(q, q_row_stride, H, k, k_row_stride, HK, T) || packed_rows_meet(q, q_row_stride, H, v, v_row_stride, HK, T)
                : overlap(so, sk) || overlap(so, sv))
            return false;
    }
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.q_out = static_cast<uint16_t*>(q_out);
    a.kp = static_cast<uint16_t*>(k_pages);
    a.vp = static_cast<uint16_t*>(v_pages);
    a.q_rs = q_row_stride; a.k_rs = k_row_stride; a.v_rs = v_row_stride; a.qo_rs = q_out_row_stride;
    a.pg = page_args(page_stride, row_stride, head_stride, n_pages, page_size, page_table, table_stride, table_pages);
    a.starts = starts; a.lens = lens; a.pos = positions;
    a.B = B; a.T = T; a.H = q ? H : 0; a.HK = HK;
    a.qw = q_norm_w; a.kw = k_norm_w;
    a.table_kind = table_kind; a.pairing = pairing; a.rot = rot; a.tab_rows = table_rows;
    a.tab_vec = tab_vec(table_kind, table_a, table_b, table_row_stride);
    a.ta = table_a; a.tb = table_b; a.tab_stride = table_row_stride; a.eps = eps;
    return true;
}

}  // namespace

extern "C" {

size_t lr_attention_window_ws_bytes(int W, int H, int HK, int nkeys, int window, int sinks, int frame) {
    if (!window_sizes_ok(W, H, HK, nkeys, window, sinks, frame)) return 0;
    return std::max(part_bytes(window_cut(W, H, HK, nkeys, window, sinks, frame, true)),
                    part_bytes(window_cut(W, H, HK, nkeys, window, sinks, frame, false)));
}

int lr_attention_window_bf16(const void* q, const void* k, const void* v, void* out, int p0, int W, int H, int HK, int nkeys,
                             int window, int sinks, int frame, float scale, int64_t q_row_stride, int64_t k_row_stride,
                             int64_t v_row_stride, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                             lr_stream_t stream) {
    if (!window_sizes_ok(W, H, HK, nkeys, window, sinks, frame) || p0 < 0 || (int64_t)p0 + W > MAX_POS || !scale_ok(scale))
        return ERR_ARGS;
    if (!rows_ok(q, q_row_stride, H) || !rows_ok(out, out_row_stride, H) || !rows_ok(k, k_row_stride, HK) ||
        !rows_ok(v, v_row_stride, HK))
        return ERR_ARGS;
    const Span so = rows_span(out, W, out_row_stride, H), sq = rows_span(q, W, q_row_stride, H),
               sk = rows_span(k, nkeys, k_row_stride, HK), sv = rows_span(v, nkeys, v_row_stride, HK);
    if (overlap(so, sq) || overlap(so, sk) || overlap(so, sv)) return ERR_ARGS;
    lr::RangeAttnArgs a{};
    const bool narrow = k_row_stride < lr::RANGE_WIDE_MAX_RS && v_row_stride < lr::RANGE_WIDE_MAX_RS;
    const Cut cut = window_cut(W, H, HK, nkeys, window, sinks, frame, narrow);
    if (!launch_fits(cut)) return ERR_ARGS;
    const size_t need = part_bytes(cut);
    if (need) {
        if (!workspace || !aligned(workspace, 256) || workspace_bytes < need) return ERR_ARGS;
        const uintptr_t lo = reinterpret_cast<uintptr_t>(workspace);
        const Span w{lo, lo + need};
        if (overlap(w, so) || overlap(w, sq) || overlap(w, sk) || overlap(w, sv)) return ERR_ARGS;
    }
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.out = static_cast<uint16_t*>(out);
    a.q_rs = q_row_stride; a.k_rs = k_row_stride; a.v_rs = v_row_stride; a.o_rs = out_row_stride;
    a.H = H; a.HK = HK; a.G = H / HK;
    a.c = scale * 1.4426950408889634f;
    set_cut(a, workspace, cut);
    a.W = W; a.p0 = p0; a.nkeys = nkeys; a.frame = std::min(frame, MAX_POS);   // (positions are below it either way)
    a.rcp_frame = lr::rcp_small(a.frame);
    a.window = std::min(window, MAX_POS); a.sinks = std::min(sinks, MAX_POS);
    return launch(a, false, cut, stream);
}

int lr_attention_packed_bf16(const void* q, const void* k, const void* v, void* out, const int* starts, int B, int T, int H, int HK,
                             int window, int sinks, float scale, int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride,
                             int64_t out_row_stride, lr_stream_t stream) {
    if (B < 1 || B > 65535 || T < 1 || T > MAX_POS || H < 1 || HK < 1 || H % HK || (int64_t)T * (H / HK) > MAX_POS || window < 0 ||
        sinks < 0 || !scale_ok(scale) || !starts || !aligned(starts, 4))
        return ERR_ARGS;
    if (!rows_ok(q, q_row_stride, H) || !rows_ok(out, out_row_stride, H) || !rows_ok(k, k_row_stride, HK) ||
        !rows_ok(v, v_row_stride, HK) || k_row_stride >= lr::RANGE_WIDE_MAX_RS || v_row_stride >= lr::RANGE_WIDE_MAX_RS)
        return ERR_ARGS;
    const Span so = rows_span(out, T, out_row_stride, H);
    if (overlap(so, rows_span(q, T, q_row_stride, H)) || overlap(so, rows_span(k, T, k_row_stride, HK)) ||
        overlap(so, rows_span(v, T, v_row_stride, HK)))
        return ERR_ARGS;
    lr::RangeAttnArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.out = static_cast<uint16_t*>(out);
    a.q_rs = q_row_stride; a.k_rs = k_row_stride; a.v_rs = v_row_stride; a.o_rs = out_row_stride;
    a.H = H; a.HK = HK; a.G = H / HK;
    a.c = scale * 1.4426950408889634f;
    a.starts = starts; a.B = B; a.T = T;
    a.window = std::min(window, MAX_POS); a.sinks = window ? std::min(sinks, MAX_POS) : 0;
    const Cut cut = packed_cut(B, T, H, HK, a.window, a.sinks);
    set_cut(a, nullptr, cut);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return (int)(cut.wide ? lr::launch_packed_wide(a, cut.wide, s) : lr::launch_packed_attn(a, cut.br, s));
}

size_t lr_cache_attention_ws_bytes(int B, int T, int max_rows, int max_keys, int H, int HK, int page_size, int window,
                                   int sinks) {
    if (!cache_sizes_ok(B, T, max_rows, max_keys, H, HK, page_size, window, sinks)) return 0;
    return std::max(part_bytes(cache_cut(B, max_rows, max_keys, H, HK, page_size, window, sinks, true)),
                    part_bytes(cache_cut(B, max_rows, max_keys, H, HK, page_size, window, sinks, false)));
}

int lr_cache_attention_bf16(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride, const void* k_pages,
                            const void* v_pages, int64_t page_stride, int64_t row_stride, int64_t head_stride, int n_pages,
                            int page_size, const int* page_table, int64_t table_stride, int table_pages, const int* starts,
                            const int* lens, int B, int T, int max_rows, int max_keys, int H, int HK, const uint64_t* tree,
                            int words, int window, int sinks, float scale, void* workspace, size_t workspace_bytes,
                            lr_stream_t stream) {
    lr::RangeAttnArgs a{};
    Span spans[4];
    if (!attention_args(a, spans, 2, q, q_row_stride, out, out_row_stride, k_pages, v_pages, page_stride, row_stride, head_stride, n_pages,
                        page_size, page_table, table_stride, table_pages, starts, lens, B, T, max_rows, max_keys, H, HK, tree, words,
                        window, sinks, scale))
        return ERR_ARGS;
    const bool narrow =
        row_stride < lr::RANGE_WIDE_MAX_RS && (page_size > lr::RANGE_WIDE_MIN_PAGE || spans[2].hi - spans[2].lo < (1ull << 32));
    const Cut cut = cache_cut(B, max_rows, max_keys, H, HK, page_size, window, sinks, narrow);
    if (!launch_fits(cut) || !workspace_ok(cut, workspace, workspace_bytes, spans, 4)) return ERR_ARGS;
    set_cut(a, workspace, cut);
    return launch(a, true, cut, stream);
}

size_t lr_cache_attention_f8_ws_bytes(int B, int T, int max_rows, int max_keys, int H, int HK, int page_size, int window, int sinks) {
    if (!cache_sizes_ok(B, T, max_rows, max_keys, H, HK, page_size, window, sinks) || page_size < lr::GROUP8) return 0;
    return part_bytes(cache8_cut(B, max_rows, max_keys, H, HK, page_size, window, sinks));
}

int lr_cache_attention_f8(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride, const void* k_pages, const void* v_pages,
                          int64_t page_stride, int64_t row_stride, int64_t head_stride, int n_pages, int page_size, const void* k_scales,
                          const void* v_scales, int64_t scale_page_stride, const int* page_table, int64_t table_stride, int table_pages,
                          const int* starts, const int* lens, int B, int T, int max_rows, int max_keys, int H, int HK,
                          const uint64_t* tree, int words, int window, int sinks, float scale, void* workspace, size_t workspace_bytes,
                          lr_stream_t stream) {
    lr::RangeAttnArgs a{};
    Span spans[6];
    Span(&four)[4] = reinterpret_cast<Span(&)[4]>(spans);
    if (!attention_args(a, four, 1, q, q_row_stride, out, out_row_stride, k_pages, v_pages, page_stride, row_stride, head_stride, n_pages,
                        page_size, page_table, table_stride, table_pages, starts, lens, B, T, max_rows, max_keys, H, HK, tree, words,
                        window, sinks, scale) ||
        !page8_ok(page_size, row_stride) || !scales_ok(k_scales, v_scales, scale_page_stride, n_pages, page_size, HK))
        return ERR_ARGS;
    spans[4] = scales_span(k_scales, 1, 0, scale_page_stride, n_pages, page_size, HK);
    spans[5] = scales_span(v_scales, 1, 0, scale_page_stride, n_pages, page_size, HK);
    for (int i : {0, 2, 3})
        if (overlap(spans[i], spans[4]) || overlap(spans[i], spans[5])) return ERR_ARGS;
    const Cut cut = cache8_cut(B, max_rows, max_keys, H, HK, page_size, window, sinks);
    if (!launch_fits(cut) || !workspace_ok(cut, workspace, workspace_bytes, spans, 6)) return ERR_ARGS;
    set_cut(a, workspace, cut);
    if (!cut.wide) {
        a.hgroups = HK / cut.hw;
        a.rcp_hk = lr::rcp_small(a.hgroups);
    }
    a.k_sc = static_cast<const uint8_t*>(k_scales);
    a.v_sc = static_cast<const uint8_t*>(v_scales);
    a.sc_ps = scale_page_stride;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return (int)(cut.wide ? lr::launch_range_wide8(a, cut.wide, s) : lr::launch_range8(a, cut.br, cut.kh, cut.hw, s));
}

int lr_cache_append_bf16(const void* q, const void* k, const void* v, int64_t q_row_stride, int64_t k_row_stride,
                         int64_t v_row_stride, void* q_out, int64_t q_out_row_stride, void* k_pages, void* v_pages,
                         int64_t page_stride, int64_t row_stride, int64_t head_stride, int n_pages, int page_size,
                         const int* page_table, int64_t table_stride, int table_pages, const int* starts, const int* lens,
                         const int* positions, int B, int T, int H, int HK, const float* q_norm_w, const float* k_norm_w,
                         int table_kind, const void* table_a, const void* table_b, int64_t table_row_stride, int table_rows,
                         int pairing, int rot_dim, float eps, lr_stream_t stream) {
    lr::CacheAppendArgs a{};
    if (!append_args(a, 2, q, k, v, q_row_stride, k_row_stride, v_row_stride, q_out, q_out_row_stride, k_pages, v_pages, page_stride,
                     row_stride, head_stride, n_pages, page_size, page_table, table_stride, table_pages, starts, lens, positions, B, T, H,
                     HK, q_norm_w, k_norm_w, table_kind, table_a, table_b, table_row_stride, table_rows, pairing, rot_dim, eps))
        return ERR_ARGS;
    return (int)lr::launch_cache_append(a, reinterpret_cast<hipStream_t>(stream));
}

int lr_cache_append_f8(const void* q, const void* k, const void* v, int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride,
                       void* q_out, int64_t q_out_row_stride, void* k_pages, void* v_pages, int64_t page_stride, int64_t row_stride,
                       int64_t head_stride, int n_pages, int page_size, void* k_scales, void* v_scales, int64_t scale_page_stride,
                       const int* page_table, int64_t table_stride, int table_pages, const int* starts, const int* lens,
                       const int* positions, int B, int T, int H, int HK, const float* q_norm_w, const float* k_norm_w, int table_kind,
                       const void* table_a, const void* table_b, int64_t table_row_stride, int table_rows, int pairing, int rot_dim,
                       float eps, lr_stream_t stream) {
    lr::CacheAppend8Args a{};
    if (!append_args(a.at, 1, q, k, v, q_row_stride, k_row_stride, v_row_stride, q_out, q_out_row_stride, k_pages, v_pages, page_stride,
                     row_stride, head_stride, n_pages, page_size, page_table, table_stride, table_pages, starts, lens, positions, B, T, H,
                     HK, q_norm_w, k_norm_w, table_kind, table_a, table_b, table_row_stride, table_rows, pairing, rot_dim, eps) ||
        B > 65535 || !page8_ok(page_size, row_stride) || !scales_ok(k_scales, v_scales, scale_page_stride, n_pages, page_size, HK))
        return ERR_ARGS;
    const Span pools[2] = {pool_span(k_pages, 1, 0, page_stride, row_stride, head_stride, n_pages, page_size, HK, 1),
                           pool_span(v_pages, 1, 0, page_stride, row_stride, head_stride, n_pages, page_size, HK, 1)};
    for (void* p : {k_scales, v_scales}) {
        const Span sc = scales_span(p, 1, 0, scale_page_stride, n_pages, page_size, HK);
        if (overlap(sc, pools[0]) || overlap(sc, pools[1]) || overlap(sc, rows_span(k, T, k_row_stride, HK)) ||
            overlap(sc, rows_span(v, T, v_row_stride, HK)) ||
            (q && (overlap(sc, rows_span(q, T, q_row_stride, H)) || overlap(sc, rows_span(q_out, T, q_out_row_stride, H)))))
            return ERR_ARGS;
    }
    a.k_sc = static_cast<uint8_t*>(k_scales);
    a.v_sc = static_cast<uint8_t*>(v_scales);
    a.sc_ps = scale_page_stride;
    return (int)lr::launch_cache_append8(a, reinterpret_cast<hipStream_t>(stream));
}

int lr_cache_copy_pages(void* k_pages, void* v_pages, int layers, int64_t layer_stride, int64_t page_stride,
                        int64_t row_stride, int64_t head_stride, int n_pages, int page_size, int HK, const int* src,
                        const int* dst, int n, lr_stream_t stream) {
    if (!pool_ok(k_pages, v_pages, page_stride, row_stride, head_stride, n_pages, page_size, HK, layers, layer_stride))
        return ERR_ARGS;
    if (n < 1 || !src || !dst || !aligned(src, 4) || !aligned(dst, 4)) return ERR_ARGS;
    lr::CacheCopyArgs a{};
    a.kp = static_cast<uint16_t*>(k_pages);
    a.vp = static_cast<uint16_t*>(v_pages);
    a.pg = page_args(page_stride, row_stride, head_stride, n_pages, page_size, nullptr, 0, 0);
    a.layer_stride = layer_stride;
    a.src = src; a.dst = dst; a.n = n; a.layers = layers; a.HK = HK; a.es = 2;
    return (int)lr::launch_cache_copy(a, reinterpret_cast<hipStream_t>(stream));
}

int lr_cache_copy_pages_f8(void* k_pages, void* v_pages, int layers, int64_t layer_stride, int64_t page_stride, int64_t row_stride,
                           int64_t head_stride, int n_pages, int page_size, int HK, void* k_scales, void* v_scales,
                           int64_t scale_layer_stride, int64_t scale_page_stride, const int* src, const int* dst, int n,
                           lr_stream_t stream) {
    if (!pool_ok(k_pages, v_pages, page_stride, row_stride, head_stride, n_pages, page_size, HK, layers, layer_stride, 1) ||
        !page8_ok(page_size, row_stride) ||
        !scales_ok(k_scales, v_scales, scale_page_stride, n_pages, page_size, HK, layers, scale_layer_stride))
        return ERR_ARGS;
    if (n < 1 || !src || !dst || !aligned(src, 4) || !aligned(dst, 4)) return ERR_ARGS;
    for (void* p : {k_scales, v_scales}) {
        const Span sc = scales_span(p, layers, scale_layer_stride, scale_page_stride, n_pages, page_size, HK);
        for (void* x : {k_pages, v_pages})
            if (overlap(sc, pool_span(x, layers, layer_stride, page_stride, row_stride, head_stride, n_pages, page_size, HK, 1)))
                return ERR_ARGS;
    }
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    lr::CacheCopyArgs a{};
    a.kp = static_cast<uint16_t*>(k_pages);
    a.vp = static_cast<uint16_t*>(v_pages);
    a.pg = page_args(page_stride, row_stride, head_stride, n_pages, page_size, nullptr, 0, 0);
    a.layer_stride = layer_stride;
    a.src = src; a.dst = dst; a.n = n; a.layers = layers; a.HK = HK; a.es = 1;
    const hipError_t e = lr::launch_cache_copy(a, s);
    if (e != hipSuccess) return (int)e;
    lr::CacheCopyScalesArgs c{};
    c.k_sc = static_cast<uint8_t*>(k_scales);
    c.v_sc = static_cast<uint8_t*>(v_scales);
    c.sc_ps = scale_page_stride; c.layer_stride = scale_layer_stride;
    c.src = src; c.dst = dst; c.n = n; c.layers = layers; c.n_pages = n_pages;
    c.bytes = (int)scales_bytes(page_size, HK);
    return (int)lr::launch_cache_copy_scales(c, s);
}

int lr_cache_move_rows(void* k_pages, void* v_pages, int layers, int64_t layer_stride, int64_t page_stride,
                       int64_t row_stride, int64_t head_stride, int n_pages, int page_size, int HK, const int* page_table,
                       int64_t table_stride, int table_pages, const int* starts, const int* src, const int* dst, int B, int n,
                       int max_rows, lr_stream_t stream) {
    if (!pool_ok(k_pages, v_pages, page_stride, row_stride, head_stride, n_pages, page_size, HK, layers, layer_stride))
        return ERR_ARGS;
    if (!table_args_ok(page_table, table_stride, table_pages, page_size, starts, B)) return ERR_ARGS;
    if (layers > 32767 || n < 1 || !src || !dst || !aligned(src, 4) || !aligned(dst, 4) || max_rows < 1 || max_rows > 256)
        return ERR_ARGS;
    lr::CacheMoveArgs a{};
    a.kp = static_cast<uint16_t*>(k_pages);
    a.vp = static_cast<uint16_t*>(v_pages);
    a.pg = page_args(page_stride, row_stride, head_stride, n_pages, page_size, page_table, table_stride, table_pages);
    a.layer_stride = layer_stride;
    a.starts = starts; a.src = src; a.dst = dst; a.B = B; a.n = n; a.max_rows = max_rows; a.layers = layers; a.HK = HK;
    return (int)lr::launch_cache_move(a, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
