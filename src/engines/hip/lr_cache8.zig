//! Extern bindings of include/lr_cache8.h (liblr_attn.so): a key / value cache in pages of 8 bits. Conventions as lr_cache.zig.

const Stream = ?*anyopaque;

pub extern "lr_attn" fn lr_cache_append_f8(q: u64, k: u64, v: u64, q_rs: i64, k_rs: i64, v_rs: i64, q_out: u64, q_out_rs: i64,
    k_pages: u64, v_pages: u64, page_stride: i64, row_stride: i64, head_stride: i64, n_pages: c_int, page_size: c_int,
    k_scales: u64, v_scales: u64, scale_page_stride: i64, page_table: u64, table_stride: i64, table_pages: c_int,
    starts: u64, lens: u64, positions: u64, b: c_int, t: c_int, h: c_int, hk: c_int, q_norm_w: u64, k_norm_w: u64,
    table_kind: c_int, table_a: u64, table_b: u64, table_rs: i64, table_rows: c_int, pairing: c_int, rot: c_int, eps: f32,
    s: Stream) c_int;
pub extern "lr_attn" fn lr_cache_attention_f8_ws_bytes(b: c_int, t: c_int, max_rows: c_int, max_keys: c_int, h: c_int,
    hk: c_int, page_size: c_int, window: c_int, sinks: c_int) usize;
pub extern "lr_attn" fn lr_cache_attention_f8(q: u64, q_rs: i64, out: u64, out_rs: i64, k_pages: u64, v_pages: u64,
    page_stride: i64, row_stride: i64, head_stride: i64, n_pages: c_int, page_size: c_int, k_scales: u64, v_scales: u64,
    scale_page_stride: i64, page_table: u64, table_stride: i64, table_pages: c_int, starts: u64, lens: u64, b: c_int,
    t: c_int, max_rows: c_int, max_keys: c_int, h: c_int, hk: c_int, tree: u64, words: c_int, window: c_int, sinks: c_int,
    scale: f32, ws: u64, ws_bytes: usize, s: Stream) c_int;
pub extern "lr_attn" fn lr_cache_copy_pages_f8(k_pages: u64, v_pages: u64, layers: c_int, layer_stride: i64,
    page_stride: i64, row_stride: i64, head_stride: i64, n_pages: c_int, page_size: c_int, hk: c_int, k_scales: u64,
    v_scales: u64, scale_layer_stride: i64, scale_page_stride: i64, src: u64, dst: u64, n: c_int, s: Stream) c_int;
