//! Raw bindings of the paged KV cache, `include/lmx/paged.h`, field for field.
//! The status codes, dtypes and stream type are the crate root's.

use core::ffi::c_void;

use crate::HipStream;

pub const LMXP_F16: u32 = 1;
pub const LMXP_I8: u32 = 2;

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct LmxpPool {
    pub n_pages: u32,
    pub page_size: u32,
    pub n_kv_heads: u32,
    pub head_dim: u32,
    pub store: u32,
    pub k: *mut c_void,
    pub v: *mut c_void,
    pub k_scale: *mut f32,
    pub v_scale: *mut f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct LmxpBatch {
    pub n_seq: u32,
    pub n_tokens: u32,
    pub max_new: u32,
    pub max_ctx: u32,
    pub table_stride: u32,
    pub cu: *const i32,
    pub ctx_lens: *const i32,
    pub page_table: *const i32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct LmxpPrologueDesc {
    pub n_heads: u32,
    pub n_rot: u32,
    pub v_norm: u32,
    pub q_head_stride: u32,
    pub q_row_stride: u32,
    pub kv_row_stride: u32,
    pub rms_eps: f32,
    pub rope_base: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct LmxpAttnDesc {
    pub n_heads: u32,
    pub window: u32,
    pub q_head_stride: u32,
    pub q_row_stride: u32,
    pub scale: f32,
}

extern "C" {
    pub fn lmxp_append(p: *const LmxpPool, b: *const LmxpBatch, k_new: *const c_void, v_new: *const c_void, src_dt: i32, row_stride: u32, stream: HipStream) -> i32;
    pub fn lmxp_read(p: *const LmxpPool, b: *const LmxpBatch, k_out: *mut c_void, v_out: *mut c_void, out_dt: i32, row_stride: u32, stream: HipStream) -> i32;
    pub fn lmxp_prologue(p: *const LmxpPool, b: *const LmxpBatch, d: *const LmxpPrologueDesc, q: *const f32, k_new: *const f32, v_new: *const f32, q_gain: *const f32, k_gain: *const f32, rope_factors: *const f32, q_out: *mut c_void, q_out_dt: i32, stream: HipStream) -> i32;
    pub fn lmxp_attn_workspace_bytes(p: *const LmxpPool, b: *const LmxpBatch, d: *const LmxpAttnDesc) -> usize;
    pub fn lmxp_attn(p: *const LmxpPool, b: *const LmxpBatch, d: *const LmxpAttnDesc, q: *const c_void, dt: i32, out: *mut c_void, ws: *mut c_void, ws_bytes: usize, stream: HipStream) -> i32;
}
