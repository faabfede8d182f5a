//! Raw bindings to `libcybq.so`: one `extern "C"` declaration per entry point of
//! `include/cybq.h`, same order, same argument names.  Pointers named `x`, `y`, `out`,
//! `residual`, `gamma`, `src`, `q_out`, `scales_out`, `q_dev`, `scales_dev` are DEVICE
//! pointers; `q` / `scales` of `cybq_weight_upload` are host pointers (the mmap'd `.model`
//! file).  `stream` is a `hipStream_t` (null = the default stream).  Every function returns
//! `CYBQ_OK` (0) or a negative status; nothing unwinds across the boundary.
#![allow(non_camel_case_types)]

use core::ffi::{c_char, c_float, c_int, c_void};

#[repr(C)]
pub struct cybq_ctx {
    _opaque: [u8; 0],
}
#[repr(C)]
pub struct cybq_weight {
    _opaque: [u8; 0],
}

#[repr(C)]
pub struct cybq_cache {
    _opaque: [u8; 0],
}
/// `starts`, `lengths` and `tables` are device pointers.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct cybq_batch {
    pub seqs: i64,
    pub rows: i64,
    pub max_new: i64,
    pub table_pages: i64,
    pub starts: *const i32,
    pub lengths: *const i32,
    pub tables: *const i32,
}

pub const CYBQ_GROUP: c_int = 32;
pub const CYBQ_MAX_EXPERTS: c_int = 1024;
pub const CYBQ_MAX_TOP_K: c_int = 64;

// enum cybq_status
pub const CYBQ_OK: c_int = 0;
pub const CYBQ_ERR_INVALID: c_int = -1;
pub const CYBQ_ERR_SHAPE: c_int = -2;
pub const CYBQ_ERR_ALIGN: c_int = -3;
pub const CYBQ_ERR_NO_DEVICE: c_int = -4;
pub const CYBQ_ERR_HIP: c_int = -5;
pub const CYBQ_ERR_NOMEM: c_int = -6;
pub const CYBQ_ERR_UNSUPPORTED: c_int = -7;

// enum cybq_quant
pub const CYBQ_Q4: c_int = 4;
pub const CYBQ_Q8: c_int = 8;
// enum cybq_layout
pub const CYBQ_LAYOUT_PLANAR: c_int = 0;
pub const CYBQ_LAYOUT_BLOCK_AOS: c_int = 1;
// enum cybq_dtype
pub const CYBQ_F32: c_int = 0;
pub const CYBQ_F16: c_int = 1;
pub const CYBQ_BF16: c_int = 2;
// enum cybq_prefill_mode
pub const CYBQ_PREFILL_FAST: c_int = 0;
pub const CYBQ_PREFILL_EXACT: c_int = 1;
// enum cybq_decode_mode
pub const CYBQ_DECODE_STREAM: c_int = 0;
pub const CYBQ_DECODE_EXACT: c_int = 1;
// enum cybq_epilogue
pub const CYBQ_EPI_NONE: c_int = 0;
pub const CYBQ_EPI_ADD: c_int = 1;
pub const CYBQ_EPI_SWIGLU: c_int = 2;
// enum cybq_score
pub const CYBQ_SCORE_SOFTMAX: c_int = 0;
pub const CYBQ_SCORE_SIGMOID: c_int = 1;
// enum cybq_cache_kind
pub const CYBQ_CACHE_F16: c_int = 1;
pub const CYBQ_CACHE_BF16: c_int = 2;
pub const CYBQ_CACHE_Q4: c_int = 4;
pub const CYBQ_CACHE_Q8: c_int = 8;
// enum cybq_rope_style
pub const CYBQ_ROPE_HALVES: c_int = 0;
pub const CYBQ_ROPE_PAIRS: c_int = 1;

extern "C" {
    pub fn cybq_init(device: c_int, out: *mut *mut cybq_ctx) -> c_int;
    pub fn cybq_destroy(ctx: *mut cybq_ctx);
    pub fn cybq_strerror(status: c_int) -> *const c_char;
    pub fn cybq_last_error(ctx: *const cybq_ctx) -> *const c_char;
    pub fn cybq_version() -> *const c_char;

    pub fn cybq_weight_upload(ctx: *mut cybq_ctx, quant: c_int, layout: c_int, N: i64, K: i64, q: *const c_void,
                              scales: *const c_void, out: *mut *mut cybq_weight) -> c_int;
    pub fn cybq_weight_upload_many(ctx: *mut cybq_ctx, count: i64, quant: *const c_int, layout: *const c_int,
                                   N: *const i64, K: *const i64, q: *const *const c_void,
                                   scales: *const *const c_void, out: *mut *mut cybq_weight) -> c_int;
    pub fn cybq_weight_clone(ctx: *mut cybq_ctx, src: *const cybq_weight, out: *mut *mut cybq_weight) -> c_int;
    pub fn cybq_weight_free(ctx: *mut cybq_ctx, w: *mut cybq_weight) -> c_int;
    pub fn cybq_trim(ctx: *mut cybq_ctx) -> c_int;
    pub fn cybq_weight_info(w: *const cybq_weight, quant: *mut c_int, N: *mut i64, K: *mut i64,
                            device_bytes: *mut i64) -> c_int;

    pub fn cybq_matmul(ctx: *mut cybq_ctx, w: *const cybq_weight, x: *const c_void, xdt: c_int, M: i64,
                       y: *mut c_void, ydt: c_int, stream: *mut c_void) -> c_int;
    pub fn cybq_matmul_static(ctx: *mut cybq_ctx, w: *const cybq_weight, x: *const c_void, xdt: c_int, M: i64,
                              y: *mut c_void, ydt: c_int, stream: *mut c_void) -> c_int;
    pub fn cybq_set_prefill_mode(ctx: *mut cybq_ctx, mode: c_int) -> c_int;
    pub fn cybq_set_decode_mode(ctx: *mut cybq_ctx, mode: c_int) -> c_int;
    pub fn cybq_matmul_many(ctx: *mut cybq_ctx, count: i64, w: *const *const cybq_weight, x: *const *const c_void,
                            y: *const *mut c_void, xdt: c_int, M: i64, ydt: c_int, stream: *mut c_void) -> c_int;
    pub fn cybq_weight_fuse_pairs(ctx: *mut cybq_ctx, gate: *const cybq_weight, up: *const cybq_weight,
                                  out: *mut *mut cybq_weight) -> c_int;
    pub fn cybq_matmul_ex(ctx: *mut cybq_ctx, w: *const cybq_weight, x: *const c_void, xdt: c_int, M: i64,
                          y: *mut c_void, ydt: c_int, epilogue: c_int, residual: *const c_void,
                          stream: *mut c_void) -> c_int;
    pub fn cybq_matmul_norm(ctx: *mut cybq_ctx, w: *const cybq_weight, x: *const c_void, xdt: c_int, M: i64,
                            gamma: *const c_void, gdt: c_int, eps: c_float, y: *mut c_void, ydt: c_int,
                            epilogue: c_int, residual: *const c_void, stream: *mut c_void) -> c_int;
    pub fn cybq_matmul_many_ex(ctx: *mut cybq_ctx, count: i64, w: *const *const cybq_weight,
                               x: *const *const c_void, y: *const *mut c_void, epilogue: *const c_int,
                               residual: *const *const c_void, xdt: c_int, M: i64, ydt: c_int,
                               stream: *mut c_void) -> c_int;
    pub fn cybq_matmul_many_norm(ctx: *mut cybq_ctx, count: i64, w: *const *const cybq_weight,
                                 x: *const *const c_void, gamma: *const *const c_void, gdt: c_int, eps: c_float,
                                 y: *const *mut c_void, epilogue: *const c_int, residual: *const *const c_void,
                                 xdt: c_int, M: i64, ydt: c_int, stream: *mut c_void) -> c_int;
    pub fn cybq_route(ctx: *mut cybq_ctx, logits: *const c_void, ldt: c_int, T: i64, E: i64,
                      top_k: i64, score: c_int, bias: *const c_float, groups: i64,
                      top_groups: i64, group_best: c_int, renormalise: c_int, scale: c_float,
                      ids: *mut i32, weights: *mut c_float, stream: *mut c_void) -> c_int;
    pub fn cybq_matmul_experts(ctx: *mut cybq_ctx, w: *const cybq_weight, E: i64,
                               x: *const c_void, xdt: c_int, T: i64, top_k: i64,
                               ids: *const i32, y: *mut c_void, ydt: c_int, epilogue: c_int,
                               stream: *mut c_void) -> c_int;
    pub fn cybq_matmul_experts_sum(ctx: *mut cybq_ctx, w: *const cybq_weight, E: i64,
                                   x: *const c_void, xdt: c_int, T: i64, top_k: i64,
                                   ids: *const i32, weights: *const c_float,
                                   residual: *const c_void, y: *mut c_void, ydt: c_int,
                                   stream: *mut c_void) -> c_int;
    pub fn cybq_cache_create(ctx: *mut cybq_ctx, kind: c_int, layers: i64, kv_heads: i64, head_dim: i64,
                             page_tokens: i64, pages: i64, out: *mut *mut cybq_cache) -> c_int;
    pub fn cybq_cache_free(ctx: *mut cybq_ctx, cache: *mut cybq_cache) -> c_int;
    pub fn cybq_cache_info(cache: *const cybq_cache, kind: *mut c_int, layers: *mut i64, kv_heads: *mut i64,
                           head_dim: *mut i64, page_tokens: *mut i64, pages: *mut i64, page_bytes: *mut i64,
                           layer_bytes: *mut i64, memory: *mut *mut c_void) -> c_int;
    pub fn cybq_cache_append(ctx: *mut cybq_ctx, cache: *mut cybq_cache, layer: i64, batch: *const cybq_batch,
                             q: *const c_void, q_stride: i64, q_heads: i64, k: *const c_void, k_stride: i64,
                             v: *const c_void, v_stride: i64, dt: c_int, rope: *const c_float,
                             rope_positions: i64, rope_dims: i64, style: c_int, q_out: *mut c_void, qdt: c_int,
                             stream: *mut c_void) -> c_int;
    pub fn cybq_cache_read(ctx: *mut cybq_ctx, cache: *const cybq_cache, layer: i64, batch: *const cybq_batch,
                           k: *mut c_void, v: *mut c_void, dt: c_int, stream: *mut c_void) -> c_int;
    pub fn cybq_attention(ctx: *mut cybq_ctx, cache: *const cybq_cache, layer: i64, batch: *const cybq_batch,
                          q: *const c_void, q_stride: i64, qdt: c_int, q_heads: i64, scale: c_float, window: i64,
                          y: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn cybq_dequant(ctx: *mut cybq_ctx, w: *const cybq_weight, out: *mut c_float, stream: *mut c_void) -> c_int;
    pub fn cybq_quantize(ctx: *mut cybq_ctx, quant: c_int, src: *const c_float, N: i64, K: i64, q_out: *mut c_void,
                         scales_out: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn cybq_weight_from_device(ctx: *mut cybq_ctx, quant: c_int, N: i64, K: i64, q_dev: *const c_void,
                                   scales_dev: *const c_void, stream: *mut c_void,
                                   out: *mut *mut cybq_weight) -> c_int;
}
