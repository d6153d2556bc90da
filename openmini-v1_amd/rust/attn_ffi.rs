//! FFI to the attention step of libopenmini_qmm.so: a line-for-line transcription of
//! include/openmini_attn.h (C types only).  Lives beside ffi.rs, whose status codes and
//! check() these calls share.  tests/test_attn_abi.py checks every declaration here
//! against the header.
#![allow(non_camel_case_types, dead_code)]

use std::os::raw::{c_int, c_void};

// openmini_attn_dtype_t
pub const F32: i32 = 0;
pub const F16: i32 = 1;
pub const BF16: i32 = 2;
pub const F8_E4M3: i32 = 3;

#[repr(C)]
pub struct Rope {
    _p: [u8; 0],
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct KvCache {
    pub d_k: *mut c_void,
    pub d_v: *mut c_void,
    pub dtype: i32,
    pub kv_heads: i32,
    pub head_dim: i32,
    pub page_size: i32,
    pub n_pages: i64,
    pub page_stride: i64,
    pub token_stride: i64,
    pub head_stride: i64,
    pub k_scale: f32,
    pub v_scale: f32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct KvPlanArgs {
    pub d_cached: *const i32,
    pub d_new: *const i32,
    pub requests: i64,
    pub d_free: *const i32,
    pub n_free: i64,
    pub d_head: *const i32,
    pub d_tables: *mut i32,
    pub table_stride: i64,
    pub max_pages: i64,
    pub page_size: i64,
    pub max_tokens: i64,
    pub d_starts: *mut i32,
    pub d_lens: *mut i32,
    pub d_rows: *mut i32,
    pub d_positions: *mut i32,
    pub d_slots: *mut i32,
    pub d_row_lens: *mut i32,
    pub d_counts: *mut i32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct RopeArgs {
    pub d_x: *const c_void,
    pub d_y: *mut c_void,
    pub x_stride: i64,
    pub y_stride: i64,
    pub x_dtype: i32,
    pub y_dtype: i32,
    pub tokens: i64,
    pub heads: i32,
    pub head_dim: i32,
    pub inverse: i32,
    pub d_positions: *const i32,
    pub position_stride: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct RopeAppendArgs {
    pub d_q: *const c_void,
    pub d_k: *const c_void,
    pub d_v: *const c_void,
    pub q_stride: i64,
    pub k_stride: i64,
    pub v_stride: i64,
    pub d_q_out: *mut c_void,
    pub q_out_stride: i64,
    pub in_dtype: i32,
    pub q_out_dtype: i32,
    pub tokens: i64,
    pub q_heads: i32,
    pub d_positions: *const i32,
    pub position_stride: i64,
    pub d_slots: *const i32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct AttnArgs {
    pub d_q: *const c_void,
    pub q_stride: i64,
    pub d_out: *mut c_void,
    pub out_stride: i64,
    pub d_lse: *mut f32,
    pub q_dtype: i32,
    pub out_dtype: i32,
    pub q_heads: i32,
    pub scale: f32,
    pub window: i64,
    pub rows: i64,
    pub d_lens: *const i32,
    pub d_rows: *const i32,
    pub d_tables: *const i32,
    pub table_stride: i64,
    pub max_pages: i64,
    pub requests: i64,
    pub d_work: *mut c_void,
    pub work_bytes: usize,
}

extern "C" {
    pub fn openmini_kv_plan(args: *const KvPlanArgs, stream: *mut c_void) -> c_int;
    pub fn openmini_rope_create(inv_freq: *const f64, axis: *const i32, pairs: c_int, axes: c_int, adjacent: c_int, scale: f32, out_rope: *mut *mut Rope) -> c_int;
    pub fn openmini_rope_free(rope: *mut Rope);
    pub fn openmini_rope_apply(rope: *const Rope, args: *const RopeArgs, stream: *mut c_void) -> c_int;
    pub fn openmini_rope_append(rope: *const Rope, cache: *const KvCache, args: *const RopeAppendArgs, stream: *mut c_void) -> c_int;
    pub fn openmini_attn_workspace_bytes(q_heads: c_int, kv_heads: c_int, head_dim: c_int) -> usize;
    pub fn openmini_attn_decode(cache: *const KvCache, args: *const AttnArgs, stream: *mut c_void) -> c_int;
}
