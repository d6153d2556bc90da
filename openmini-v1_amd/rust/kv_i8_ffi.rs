//! FFI to the calls of libopenmini_qmm.so on caches of 8-bit integers, to prompt attention and to
//! reading a cache back: a line-for-line transcription of include/openmini_kv_i8.h (C types
//! only).  Lives beside attn_ffi.rs, whose structures it shares.  tests/test_kv_i8_abi.py checks
//! every declaration here against the header.
#![allow(non_camel_case_types, dead_code)]

use super::attn_ffi::{AttnArgs, KvCache, Rope, RopeAppendArgs};
use std::os::raw::{c_int, c_void};

// OPENMINI_ATTN_I8
pub const I8: i32 = 4;

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct KvScales {
    pub d_k: *mut f32,
    pub d_v: *mut f32,
    pub block: i32,
    pub page_stride: i64,
    pub block_stride: i64,
    pub head_stride: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct KvReadArgs {
    pub d_tables: *const i32,
    pub table_stride: i64,
    pub max_pages: i64,
    pub requests: i64,
    pub d_starts: *const i32,
    pub d_first: *const i32,
    pub tokens: i64,
    pub d_k_out: *mut c_void,
    pub d_v_out: *mut c_void,
    pub k_stride: i64,
    pub v_stride: i64,
    pub out_dtype: i32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct PromptArgs {
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
    pub d_starts: *const i32,
    pub d_tables: *const i32,
    pub table_stride: i64,
    pub max_pages: i64,
    pub requests: i64,
    pub d_work: *mut c_void,
    pub work_bytes: usize,
}

extern "C" {
    pub fn openmini_rope_append_i8(rope: *const Rope, cache: *const KvCache, scales: *const KvScales, args: *const RopeAppendArgs, stream: *mut c_void) -> c_int;
    pub fn openmini_attn_decode_i8(cache: *const KvCache, scales: *const KvScales, args: *const AttnArgs, stream: *mut c_void) -> c_int;
    pub fn openmini_kv_read(cache: *const KvCache, scales: *const KvScales, args: *const KvReadArgs, stream: *mut c_void) -> c_int;
    pub fn openmini_attn_prompt_workspace_bytes(q_heads: c_int, kv_heads: c_int, head_dim: c_int) -> usize;
    pub fn openmini_attn_prompt(cache: *const KvCache, scales: *const KvScales, args: *const PromptArgs, stream: *mut c_void) -> c_int;
}
