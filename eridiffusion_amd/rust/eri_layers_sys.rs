//! Raw `extern "C"` declarations of include/eri_layers.h: embedding lookup and its gradient, dropout, and the residual's
//! addition with root-mean-square norm, forward and backward.  Plain pointers, sizes and ints, as in eri_optim8_sys.rs.
#![allow(non_camel_case_types)]
use core::ffi::{c_int, c_void};

pub const ERI_DTYPE_F8E4M3: i32 = 16;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriEmbedding {
    pub ids: *const c_void, pub table: *const c_void, pub out: *mut c_void, pub tokens: u64, pub vocab: u64, pub dim: u64,
    pub table_stride: u64, pub out_stride: u64, pub ids_64: i32, pub dtype_tag: i32, pub scale: f32, pub reserved: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriEmbeddingGrad {
    pub ids: *const c_void, pub grad: *const c_void, pub out: *mut c_void, pub workspace: *mut c_void, pub workspace_bytes: u64,
    pub tokens: u64, pub vocab: u64, pub dim: u64, pub grad_stride: u64, pub out_stride: u64, pub padding_id: i64, pub ids_64: i32,
    pub grad_dtype: i32, pub out_dtype: i32, pub accumulate: i32, pub scale: f32, pub reserved: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriDropoutKey { pub seed: u64, pub offset: u64, pub offset_ptr: *const u64, pub p: f64 }

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriDropout {
    pub x: *const c_void, pub y: *mut c_void, pub rows: u64, pub cols: u64, pub x_stride: u64, pub y_stride: u64,
    pub key: EriDropoutKey, pub dtype_tag: i32, pub reserved: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriRmsNorm {
    pub x: *const c_void, pub residual: *const c_void, pub weight: *const c_void, pub y: *mut c_void, pub h: *mut c_void,
    pub rstd: *mut f32, pub scales: *mut f32, pub rows: u64, pub cols: u64, pub x_stride: u64, pub residual_stride: u64,
    pub y_stride: u64, pub h_stride: u64, pub key: EriDropoutKey, pub eps: f32, pub x_dtype: i32, pub residual_dtype: i32,
    pub weight_dtype: i32, pub y_dtype: i32, pub scale_group: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriRmsNormGrad {
    pub grad: *const c_void, pub h: *const c_void, pub rstd: *const f32, pub weight: *const c_void, pub grad_h: *const c_void,
    pub grad_x: *mut c_void, pub grad_residual: *mut c_void, pub grad_weight: *mut c_void, pub workspace: *mut c_void,
    pub workspace_bytes: u64, pub rows: u64, pub cols: u64, pub grad_stride: u64, pub h_stride: u64, pub grad_h_stride: u64,
    pub grad_x_stride: u64, pub grad_residual_stride: u64, pub key: EriDropoutKey, pub grad_dtype: i32, pub h_dtype: i32,
    pub x_dtype: i32, pub weight_dtype: i32, pub grad_weight_dtype: i32, pub reserved: i32,
}

extern "C" {
    pub fn eri_embedding(args: *const EriEmbedding, stream: *mut c_void) -> c_int;
    pub fn eri_embedding_grad_workspace(tokens: u64, vocab: u64, dim: u64, bytes: *mut u64) -> c_int;
    pub fn eri_embedding_grad(args: *const EriEmbeddingGrad, stream: *mut c_void) -> c_int;
    pub fn eri_dropout(args: *const EriDropout, stream: *mut c_void) -> c_int;
    pub fn eri_rms_norm(args: *const EriRmsNorm, stream: *mut c_void) -> c_int;
    pub fn eri_rms_norm_grad_workspace(rows: u64, cols: u64, bytes: *mut u64) -> c_int;
    pub fn eri_rms_norm_grad(args: *const EriRmsNormGrad, stream: *mut c_void) -> c_int;
}
