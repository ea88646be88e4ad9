//! Raw bindings of steps with drafted tokens, `include/lmx/spec.h`, field for field.
//! Pools, batches and the paged descriptions are `paged`'s.

use core::ffi::c_void;

use crate::paged::{LmxpAttnDesc, LmxpBatch, LmxpPool, LmxpPrologueDesc};
use crate::HipStream;

pub const LMXS_MAX_ROWS: u32 = 1024;

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct LmxsPlanDesc {
    pub n_seq: u32,
    pub n_tokens: u32,
    pub page_size: u32,
    pub table_stride: u32,
    pub n_pages: u32,
    pub trim: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct LmxsRope {
    pub interleaved: u32,
    pub turn_scale: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct LmxsVerifyDesc {
    pub n_seq: u32,
    pub n_tokens: u32,
    pub max_new: u32,
    pub vocab: u32,
    pub p_stride: u32,
    pub q_stride: u32,
    pub greedy: u32,
}

extern "C" {
    pub fn lmxs_plan(d: *const LmxsPlanDesc, lens: *const i32, new_rows: *const i32, page_table: *mut i32, held: *mut i32, free_pages: *mut i32, n_free: *mut i32, cu: *mut i32, ctx_lens: *mut i32, slots: *mut i64, pos: *mut i32, stream: HipStream) -> i32;
    pub fn lmxs_tree(b: *const LmxpBatch, parent: *const i32, words: u32, window: u32, pos: *mut i32, seen: *mut u64, stream: HipStream) -> i32;
    pub fn lmxs_prologue(p: *const LmxpPool, b: *const LmxpBatch, d: *const LmxpPrologueDesc, r: *const LmxsRope, pos: *const i32, q: *const f32, k_new: *const f32, v_new: *const f32, q_gain: *const f32, k_gain: *const f32, rope_factors: *const f32, q_out: *mut c_void, q_out_dt: i32, stream: HipStream) -> i32;
    pub fn lmxs_attn_workspace_bytes(p: *const LmxpPool, b: *const LmxpBatch, d: *const LmxpAttnDesc) -> usize;
    pub fn lmxs_attn(p: *const LmxpPool, b: *const LmxpBatch, d: *const LmxpAttnDesc, seen: *const u64, words: u32, pos: *const i32, q: *const c_void, dt: i32, out: *mut c_void, ws: *mut c_void, ws_bytes: usize, stream: HipStream) -> i32;
    pub fn lmxs_verify_workspace_bytes(d: *const LmxsVerifyDesc) -> usize;
    pub fn lmxs_verify(d: *const LmxsVerifyDesc, cu: *const i32, tokens: *const i32, parent: *const i32, p: *const c_void, q: *const c_void, dt: i32, u: *const f32, r: *const f32, path: *mut i32, accepted: *mut i32, token: *mut i32, lens: *mut i32, ws: *mut c_void, ws_bytes: usize, stream: HipStream) -> i32;
    pub fn lmxs_keep(pools: *const *const LmxpPool, n_pools: u32, b: *const LmxpBatch, path: *const i32, path_stride: u32, accepted: *const i32, stream: HipStream) -> i32;
}
