//! Raw `extern "C"` declarations of include/eri_losses.h: log probabilities of given tokens with entropy and top alternatives, and
//! distillation from a teacher's top tokens, each with the logits' gradient.  Plain pointers, sizes and ints, as in eri_optim8_sys.rs.
#![allow(non_camel_case_types)]
use core::ffi::{c_int, c_void};

pub const ERI_TOP_MOST: i32 = 64;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriTokenLogprobs {
    pub logits: *const c_void, pub ids: *const c_void, pub logprob: *mut f32, pub entropy: *mut f32, pub stats: *mut f32, pub top: *mut f32,
    pub top_ids: *mut i64, pub workspace: *mut c_void, pub workspace_bytes: u64, pub rows: u64, pub vocab: u64, pub logits_stride: u64,
    pub temperature: f32, pub ids_64: i32, pub dtype_tag: i32, pub top_n: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriTokenLogprobsGrad {
    pub logits: *const c_void, pub ids: *const c_void, pub stats: *const f32, pub grad: *const f32, pub grad_entropy: *const f32,
    pub entropy: *const f32, pub out: *mut c_void, pub rows: u64, pub vocab: u64, pub logits_stride: u64, pub out_stride: u64,
    pub temperature: f32, pub ids_64: i32, pub dtype_tag: i32, pub out_dtype: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriDistillTop {
    pub logits: *const c_void, pub ids: *const c_void, pub teacher: *const c_void, pub loss: *mut f32, pub stats: *mut f32,
    pub workspace: *mut c_void, pub workspace_bytes: u64, pub rows: u64, pub vocab: u64, pub logits_stride: u64, pub ids_stride: u64,
    pub teacher_stride: u64, pub temperature: f32, pub ids_64: i32, pub dtype_tag: i32, pub teacher_dtype: i32, pub k: i32, pub rest: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct EriDistillTopGrad {
    pub logits: *const c_void, pub ids: *const c_void, pub teacher: *const c_void, pub stats: *const f32, pub grad: *const f32,
    pub out: *mut c_void, pub rows: u64, pub vocab: u64, pub logits_stride: u64, pub ids_stride: u64, pub teacher_stride: u64,
    pub out_stride: u64, pub temperature: f32, pub ids_64: i32, pub dtype_tag: i32, pub teacher_dtype: i32, pub out_dtype: i32, pub k: i32,
}

extern "C" {
    pub fn eri_token_logprobs_workspace(rows: u64, vocab: u64, top_n: i32, bytes: *mut u64) -> c_int;
    pub fn eri_token_logprobs(args: *const EriTokenLogprobs, stream: *mut c_void) -> c_int;
    pub fn eri_token_logprobs_grad(args: *const EriTokenLogprobsGrad, stream: *mut c_void) -> c_int;
    pub fn eri_distill_top_workspace(rows: u64, vocab: u64, bytes: *mut u64) -> c_int;
    pub fn eri_distill_top(args: *const EriDistillTop, stream: *mut c_void) -> c_int;
    pub fn eri_distill_top_grad(args: *const EriDistillTopGrad, stream: *mut c_void) -> c_int;
}
