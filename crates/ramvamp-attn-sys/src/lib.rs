// Generated by gen_bindings.py from include/*.h; do not edit by hand.
//! Raw bindings to libramvamp_attn (the MI355X attention hot path's C ABI):
//! one declaration per symbol of include/ramvamp_attn.h, ramvamp_gemv.h,
//! ramvamp_block.h, ramvamp_router.h, ramvamp_paged.h and ramvamp_floors.h. The safe wrapper
//! that keeps the reference's signatures is crates/ramvamp-attn.
#![allow(non_camel_case_types, clippy::missing_safety_doc)]
use std::os::raw::{c_char, c_int, c_void};

pub const RV_ABI_VERSION: u32 = 1;
pub const RV_OK: i32 = 0;
pub const RV_KV_INVALID_DIMS: i32 = 1;
pub const RV_KV_LAYER_OUT_OF_RANGE: i32 = 2;
pub const RV_KV_ROW_LEN_MISMATCH: i32 = 3;
pub const RV_KV_CAPACITY_EXCEEDED: i32 = 4;
pub const RV_KV_POSITION_OUT_OF_RANGE: i32 = 5;
pub const RV_KV_RAGGED_LAYERS: i32 = 6;
pub const RV_KV_TRUNCATE_BEYOND_LENGTH: i32 = 7;
pub const RV_ATTN_Q_LEN_INDIVISIBLE: i32 = 16;
pub const RV_ATTN_GQA_GROUP_MISMATCH: i32 = 17;
pub const RV_ATTN_OUT_LEN_MISMATCH: i32 = 18;
pub const RV_ATTN_EMPTY_LAYER: i32 = 19;
pub const RV_ATTN_KV_HEAD_RANGE: i32 = 20;
pub const RV_ATTN_SCRATCH_TOO_SHORT: i32 = 21;
pub const RV_PRIM_INVALID_HEAD_DIM: i32 = 24;
pub const RV_PRIM_LENGTH_MISMATCH: i32 = 25;
pub const RV_PRIM_EMPTY: i32 = 26;
pub const RV_ERR_NULL_ARG: i32 = 32;
pub const RV_ERR_UNSUPPORTED: i32 = 33;
pub const RV_ERR_HIP: i32 = 34;
pub const RV_ERR_BAD_ELEM: i32 = 35;
pub const RV_HOST_PTRS: u32 = 0x1;
pub const RV_SYNC: u32 = 0x2;
pub const RV_PREFILL_EXACT: u32 = 0x00;
pub const RV_PREFILL_F16: u32 = 0x10;
pub const RV_PREFILL_BF16: u32 = 0x20;
pub const RV_PREFILL_MODE_MASK: u32 = 0x30;
pub const RV_NOALLOC_SCRATCH_BYTES: usize = (8 << 20);
pub const RV_TUNE_DECODE_SPLIT_LEN: i32 = 1;
pub const RV_TUNE_PREFILL_KV_SPLIT: i32 = 2;
pub const RV_TUNE_DECODE_WAVES: i32 = 3;
pub const RV_TUNE_PREFILL_ROWS: i32 = 4;
pub const RV_TUNE_DECODE_HG: i32 = 5;
pub const RV_TUNE_DECODE_IMPL: i32 = 6;
pub const RV_TUNE_KERNEL_TIMING: i32 = 7;
pub const RV_TUNE_DECODE_DEPTH: i32 = 9;
pub const RV_TUNE_DECODE_MERGE: i32 = 11;
pub const RV_TUNE_ROWS_COLUMNS: i32 = 12;
pub const RV_ELEM_F16: i32 = 1;
pub const RV_ELEM_F32: i32 = 2;
pub const RV_ELEM_Q8_0: i32 = 4;
pub const RV_QF_Q4_K: u32 = 1;
pub const RV_QF_Q5_K: u32 = 2;
pub const RV_QF_Q6_K: u32 = 3;
pub const RV_QF_Q8_0: u32 = 4;
pub const RV_QF_Q8_K: u32 = 5;
pub const RV_QUANT_INDIVISIBLE_ROW: i32 = 40;
pub const RV_QUANT_ROW_BYTES_NOT_BLOCK_MULTIPLE: i32 = 41;
pub const RV_QUANT_BLOCK_COUNT_MISMATCH: i32 = 42;
pub const RV_QUANT_QUANTIZE_LEN_MISMATCH: i32 = 43;
pub const RV_QUANT_UNSUPPORTED_FORMAT: i32 = 44;
pub const RV_FWD_INVALID_TOP_K: i32 = 48;
pub const RV_PAGED_PAGE_OUT_OF_RANGE: i32 = 56;
pub const RV_PAGED_SEQUENCE_OUT_OF_RANGE: i32 = 57;
pub const RV_PAGED_POSITION_OUT_OF_RANGE: i32 = 58;
pub const RV_ROPE_HALF: u32 = 0;
pub const RV_ROPE_INTERLEAVED: u32 = 1;
pub const RV_ROPE_UNSCALED: u32 = 0;
pub const RV_ROPE_LINEAR: u32 = 1;
pub const RV_ROPE_NTK: u32 = 2;
pub const RV_ROPE_YARN: u32 = 3;
pub const RV_TUNE_PAGED_JOIN: i32 = 1;
pub const RV_FLOOR_MFMA_F16_16X16X32: i32 = 0;
pub const RV_FLOOR_MFMA_F16_32X32X16: i32 = 1;
pub const RV_FLOOR_MFMA_F32_16X16X4: i32 = 2;
pub const RV_FLOOR_VALU_FMA: i32 = 0;
pub const RV_FLOOR_VALU_EXP: i32 = 1;

pub type rv_elem = i32;
#[repr(C)]
pub struct rv_kv {
    _private: [u8; 0],
}
#[repr(C)]
pub struct rv_rope {
    _private: [u8; 0],
}
#[repr(C)]
pub struct rv_paged {
    _private: [u8; 0],
}
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rv_error {
    pub code: i32,
    pub a: u64,
    pub b: u64,
    pub c: u64,
    pub d: u64,
    pub what: *const c_char,
}
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rv_block_q8_k {
    pub d: f32,
    pub qs: [i8; 256],
    pub bsums: [i16; 16],
}
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rv_block_q8_0 {
    pub d: f32,
    pub qs: [i8; 32],
}
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rv_attn_block_weights {
    pub attn_norm: *const f32,
    pub q_format: u32,
    pub wq: *const u8,
    pub wq_len: usize,
    pub wk: *const u8,
    pub wk_len: usize,
    pub v_format: u32,
    pub wv: *const u8,
    pub wv_len: usize,
    pub q_norm: *const f32,
    pub k_norm: *const f32,
    pub o_format: u32,
    pub wo: *const u8,
    pub wo_len: usize,
    pub q_norm_len: usize,
    pub k_norm_len: usize,
}
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rv_page_table {
    pub ids: *const i32,
    pub n_seqs: usize,
    pub pages: usize,
    pub stride: usize,
}

extern "C" {
    pub fn rv_abi_version() -> u32;
    pub fn rv_status_name(code: i32) -> *const c_char;
    pub fn rv_scratch_len(n_q_heads: usize, n_kv_heads: usize, head_dim: usize, max_positions: usize) -> usize;
    pub fn rv_kv_projected_bytes(n_layers: usize, n_kv_heads: usize, head_dim: usize, capacity: usize, elem: rv_elem, bytes: *mut u64, err: *mut rv_error) -> i32;
    pub fn rv_kv_new(n_layers: usize, n_kv_heads: usize, head_dim: usize, capacity: usize, elem: rv_elem, device: c_int, out: *mut *mut rv_kv, err: *mut rv_error) -> i32;
    pub fn rv_kv_free(kv: *mut rv_kv);
    pub fn rv_kv_set_stream(kv: *mut rv_kv, hip_stream: *mut c_void, err: *mut rv_error) -> i32;
    pub fn rv_kv_synchronize(kv: *mut rv_kv, err: *mut rv_error) -> i32;
    pub fn rv_kv_n_layers(kv: *const rv_kv) -> usize;
    pub fn rv_kv_n_kv_heads(kv: *const rv_kv) -> usize;
    pub fn rv_kv_head_dim(kv: *const rv_kv) -> usize;
    pub fn rv_kv_capacity(kv: *const rv_kv) -> usize;
    pub fn rv_kv_kv_dim(kv: *const rv_kv) -> usize;
    pub fn rv_kv_elem(kv: *const rv_kv) -> i32;
    pub fn rv_kv_len(kv: *const rv_kv, layer: usize, len: *mut usize, err: *mut rv_error) -> i32;
    pub fn rv_kv_is_empty(kv: *const rv_kv) -> c_int;
    pub fn rv_kv_seq_len(kv: *const rv_kv, len: *mut usize, err: *mut rv_error) -> i32;
    pub fn rv_kv_append(kv: *mut rv_kv, layer: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_kv_append_rows(kv: *mut rv_kv, layer: usize, k: *const f32, v: *const f32, rows: usize, row_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_kv_clear(kv: *mut rv_kv);
    pub fn rv_kv_truncate(kv: *mut rv_kv, new_len: usize, err: *mut rv_error) -> i32;
    pub fn rv_kv_truncate_layer(kv: *mut rv_kv, layer: usize, new_len: usize, err: *mut rv_error) -> i32;
    pub fn rv_kv_append_each(kv: *mut rv_kv, layer0: usize, n: usize, k: *const f32, v: *const f32, row_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_kv_read_rows(kv: *const rv_kv, layer: usize, pos: usize, rows: usize, k: *mut f32, v: *mut f32, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_kv_k_layer(kv: *const rv_kv, layer: usize, dev: *mut *const c_void, n_elems: *mut usize, err: *mut rv_error) -> i32;
    pub fn rv_kv_v_layer(kv: *const rv_kv, layer: usize, dev: *mut *const c_void, n_elems: *mut usize, err: *mut rv_error) -> i32;
    pub fn rv_kv_read_row(kv: *const rv_kv, plane_v: c_int, layer: usize, pos: usize, dst: *mut c_void, err: *mut rv_error) -> i32;
    pub fn rv_decode_attention(kv: *const rv_kv, q: *const f32, q_len: usize, layer: usize, scale: f32, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_decode_attention_in(kv: *const rv_kv, q: *const f32, q_len: usize, layer: usize, scale: f32, scratch_len: usize, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_decode_attention_kv_range_in(kv: *const rv_kv, q: *const f32, q_len: usize, layer: usize, scale: f32, kv_lo: usize, kv_hi: usize, scratch_len: usize, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_decode_attention_noalloc(kv: *const rv_kv, q: *const f32, q_len: usize, layer: usize, scale: f32, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attention_at(kv: *const rv_kv, q: *const f32, q_len: usize, layer: usize, positions: usize, scale: f32, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attention_at_in(kv: *const rv_kv, q: *const f32, q_len: usize, layer: usize, positions: usize, scale: f32, scratch_len: usize, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attention_at_kv_range_in(kv: *const rv_kv, q: *const f32, q_len: usize, layer: usize, positions: usize, scale: f32, kv_lo: usize, kv_hi: usize, scratch_len: usize, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attention_at_rows(kv: *const rv_kv, q_rows: *const f32, rows: usize, q_dim: usize, layer: usize, start: usize, scale: f32, out: *mut f32, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_decode_attention_shared(prefix: *const rv_kv, prefix_layer: usize, prefix_positions: usize, tails: *const rv_kv, tail_layer: usize, q_rows: *const f32, n_seqs: usize, q_dim: usize, scale: f32, out: *mut f32, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_decode_step_shared(prefix: *const rv_kv, prefix_layer: usize, prefix_positions: usize, tails: *mut rv_kv, tail_layer: usize, n_seqs: usize, q_rows: *const f32, k_rows: *const f32, v_rows: *const f32, q_dim: usize, q_norm_w: *const f32, q_norm_len: usize, k_norm_w: *const f32, k_norm_len: usize, eps: f32, theta: f32, scale: f32, out: *mut f32, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_decode_step(kv: *mut rv_kv, layer: usize, q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, q_norm_w: *const f32, q_norm_len: usize, k_norm_w: *const f32, k_norm_len: usize, eps: f32, theta: f32, position: usize, scale: f32, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_decode_step_dev(kv: *mut rv_kv, layer: usize, q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, q_norm_w: *const f32, q_norm_len: usize, k_norm_w: *const f32, k_norm_len: usize, eps: f32, theta: f32, d_position: *const u32, max_position: usize, scale: f32, out: *mut f32, out_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_kv_commit(kv: *mut rv_kv, layer: usize, rows: usize, err: *mut rv_error) -> i32;
    pub fn rv_kv_device_status(kv: *mut rv_kv, err: *mut rv_error) -> i32;
    pub fn rv_position_advance(kv: *mut rv_kv, d_position: *mut u32, n: u32, err: *mut rv_error) -> i32;
    pub fn rv_prefill_chunk(kv: *mut rv_kv, layer: usize, q_rows: *const f32, k_rows: *const f32, v_rows: *const f32, rows: usize, q_dim: usize, q_norm_w: *const f32, q_norm_len: usize, k_norm_w: *const f32, k_norm_len: usize, eps: f32, theta: f32, start: usize, scale: f32, out: *mut f32, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_kv_set_tuning(kv: *mut rv_kv, knob: i32, value: i64, err: *mut rv_error) -> i32;
    pub fn rv_kv_kernel_time(kv: *mut rv_kv, total_ms: *mut f64, launches: *mut u64, err: *mut rv_error) -> i32;
    pub fn rv_kv_device_bytes(kv: *mut rv_kv, now: *mut u64, bound: *mut u64, err: *mut rv_error) -> i32;
    pub fn rv_kv_projected_device_bytes(n_layers: usize, n_kv_heads: usize, head_dim: usize, capacity: usize, elem: rv_elem, bytes: *mut u64, err: *mut rv_error) -> i32;
    pub fn rv_kv_xcd_dealing(kv: *mut rv_kv, ok: *mut i32, err: *mut rv_error) -> i32;
    pub fn rv_quant_block_weights(format: u32) -> usize;
    pub fn rv_quant_block_bytes(format: u32) -> usize;
    pub fn rv_quant_row_bytes(format: u32, in_dim: usize, row_bytes: *mut usize, err: *mut rv_error) -> i32;
    pub fn rv_quantize_row_q8_0(x: *const f32, x_len: usize, out: *mut rv_block_q8_0, n_blocks: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_quantize_row_q8_k(x: *const f32, x_len: usize, out: *mut rv_block_q8_k, n_blocks: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_gemv_q8_k_rows(format: u32, weight: *const u8, weight_len: usize, in_dim: usize, out_dim: usize, acts: *const rv_block_q8_k, act_blocks: usize, row_lo: usize, row_hi: usize, out: *mut f32, out_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_gemv_q8_k(format: u32, weight: *const u8, weight_len: usize, in_dim: usize, out_dim: usize, acts: *const rv_block_q8_k, act_blocks: usize, out: *mut f32, out_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_gemv_q8_0_rows(weight: *const u8, weight_len: usize, in_dim: usize, out_dim: usize, acts: *const rv_block_q8_0, act_blocks: usize, row_lo: usize, row_hi: usize, out: *mut f32, out_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_gemv_q8_0(weight: *const u8, weight_len: usize, in_dim: usize, out_dim: usize, acts: *const rv_block_q8_0, act_blocks: usize, out: *mut f32, out_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_gemv_q8_k_batched(format: u32, weight: *const u8, weight_len: usize, in_dim: usize, out_dim: usize, acts: *const rv_block_q8_k, act_blocks: usize, n_acts: usize, row_lo: usize, row_hi: usize, out: *mut f32, out_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_gemv_q8_0_batched(weight: *const u8, weight_len: usize, in_dim: usize, out_dim: usize, acts: *const rv_block_q8_0, act_blocks: usize, n_acts: usize, row_lo: usize, row_hi: usize, out: *mut f32, out_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attn_in_proj_rows_scratch_bytes(n_rows: usize, hidden: usize) -> usize;
    pub fn rv_attn_in_proj_rows(normed_rows: *const f32, n_rows: usize, hidden: usize, q_format: u32, wq: *const u8, wq_len: usize, q_rows: *mut f32, q_dim: usize, wk: *const u8, wk_len: usize, k_rows: *mut f32, kv_dim: usize, v_format: u32, wv: *const u8, wv_len: usize, v_rows: *mut f32, scratch: *mut c_void, scratch_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attn_out_proj_rows_scratch_bytes(n_rows: usize, q_dim: usize) -> usize;
    pub fn rv_attn_out_proj_rows(attn_rows: *const f32, n_rows: usize, q_dim: usize, o_format: u32, wo: *const u8, wo_len: usize, residual_rows: *mut f32, hidden: usize, scratch: *mut c_void, scratch_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attn_in_proj_scratch_bytes(hidden: usize) -> usize;
    pub fn rv_attn_in_proj(normed: *const f32, hidden: usize, q_format: u32, wq: *const u8, wq_len: usize, q: *mut f32, q_dim: usize, wk: *const u8, wk_len: usize, k: *mut f32, kv_dim: usize, v_format: u32, wv: *const u8, wv_len: usize, v: *mut f32, scratch: *mut c_void, scratch_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attn_out_proj_scratch_bytes(q_dim: usize) -> usize;
    pub fn rv_attn_out_proj(attn_out: *const f32, q_dim: usize, o_format: u32, wo: *const u8, wo_len: usize, o: *mut f32, hidden: usize, scratch: *mut c_void, scratch_len: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attn_block_scratch_bytes(hidden: usize, q_dim: usize, kv_dim: usize) -> usize;
    pub fn rv_attn_block_decode(kv: *mut rv_kv, layer: usize, residual: *mut f32, hidden: usize, q_dim: usize, w: *const rv_attn_block_weights, eps: f32, theta: f32, position: usize, scale: f32, scratch: *mut c_void, scratch_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attn_block_decode_dev(kv: *mut rv_kv, layer: usize, residual: *mut f32, hidden: usize, q_dim: usize, w: *const rv_attn_block_weights, eps: f32, theta: f32, d_position: *const u32, max_position: usize, scale: f32, scratch: *mut c_void, scratch_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_attn_block_prefill_scratch_bytes(n_rows: usize, hidden: usize, q_dim: usize, kv_dim: usize) -> usize;
    pub fn rv_attn_block_prefill(kv: *mut rv_kv, layer: usize, residual_rows: *mut f32, n_rows: usize, hidden: usize, q_dim: usize, w: *const rv_attn_block_weights, eps: f32, theta: f32, start: usize, scale: f32, scratch: *mut c_void, scratch_len: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_router_topk(x: *const f32, n_rows: usize, hidden: usize, router: *const f32, router_len: usize, n_experts: usize, top_k: usize, norm_topk_prob: c_int, experts: *mut u32, weights: *mut f32, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_rope_new(head_dim: usize, rotary_dim: usize, layout: u32, theta: f64, scaling: u32, factor: f64, trained_positions: usize, beta_fast: f64, beta_slow: f64, out: *mut *mut rv_rope, err: *mut rv_error) -> i32;
    pub fn rv_rope_free(rope: *mut rv_rope);
    pub fn rv_rope_frequencies(rope: *const rv_rope, freq: *mut f64, n: usize, gain: *mut f64, err: *mut rv_error) -> i32;
    pub fn rv_rope_rows(rope: *const rv_rope, x: *const f32, x_stride: usize, rows: usize, width: usize, positions: *const i32, out: *mut f32, out_stride: usize, stream: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_paged_projected_bytes(n_layers: usize, n_kv_heads: usize, head_dim: usize, n_pages: usize, page_rows: usize, elem: rv_elem, bytes: *mut u64, err: *mut rv_error) -> i32;
    pub fn rv_paged_new(n_layers: usize, n_kv_heads: usize, head_dim: usize, n_pages: usize, page_rows: usize, elem: rv_elem, device: c_int, out: *mut *mut rv_paged, err: *mut rv_error) -> i32;
    pub fn rv_paged_free(pg: *mut rv_paged);
    pub fn rv_paged_set_tuning(pg: *mut rv_paged, knob: i32, value: i64, err: *mut rv_error) -> i32;
    pub fn rv_paged_set_stream(pg: *mut rv_paged, hip_stream: *mut c_void, err: *mut rv_error) -> i32;
    pub fn rv_paged_synchronize(pg: *mut rv_paged, err: *mut rv_error) -> i32;
    pub fn rv_paged_device_status(pg: *mut rv_paged, err: *mut rv_error) -> i32;
    pub fn rv_paged_append_rows(pg: *mut rv_paged, layer: usize, rope: *const rv_rope, k: *const f32, k_stride: usize, v: *const f32, v_stride: usize, rows: usize, positions: *const i32, seqs: *const i32, table: *const rv_page_table, k_norm_w: *const f32, k_norm_len: usize, eps: f32, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_paged_read_rows(pg: *mut rv_paged, layer: usize, rows: usize, positions: *const i32, seqs: *const i32, table: *const rv_page_table, k: *mut c_void, v: *mut c_void, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_paged_attention(pg: *mut rv_paged, layer: usize, q: *const f32, q_stride: usize, n_seqs: usize, q_dim: usize, table: *const rv_page_table, lens: *const i32, scale: f32, out: *mut f32, out_stride: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_paged_decode_step(pg: *mut rv_paged, layer: usize, rope: *const rv_rope, q: *const f32, q_stride: usize, k: *const f32, k_stride: usize, v: *const f32, v_stride: usize, n_seqs: usize, q_dim: usize, q_norm_w: *const f32, q_norm_len: usize, k_norm_w: *const f32, k_norm_len: usize, eps: f32, table: *const rv_page_table, positions: *const i32, scale: f32, out: *mut f32, out_stride: usize, flags: u32, err: *mut rv_error) -> i32;
    pub fn rv_floor_empty(stream: *mut c_void, err: *mut rv_error) -> i32;
    pub fn rv_floor_stream_read(src: *const c_void, bytes: usize, n_wg: u32, sink: *mut f32, stream: *mut c_void, err: *mut rv_error) -> i32;
    pub fn rv_floor_mfma(form: i32, chains: u32, iters: u32, n_wg: u32, sink: *mut f32, stream: *mut c_void, err: *mut rv_error) -> i32;
    pub fn rv_floor_mfma_valu(kind: i32, valu_per_mfma: u32, iters: u32, n_wg: u32, sink: *mut f32, stream: *mut c_void, err: *mut rv_error) -> i32;
}
