//! Raw bindings of `include/momiru_ops.h`: the operators around the MatMul
//! node (linear layers, tokens sorted by expert, the experts' products) of the
//! same library. Layouts and conventions as in `ffi`.
//!
//! NOT COMPILED HERE: the image this library was built in has no Rust
//! toolchain. `tests/test_ops_contract.py` checks this file as text against the
//! header and the ctypes mirror.

#![allow(non_camel_case_types)]

use core::ffi::{c_char, c_void};

use super::ffi::mmr_view;

pub const MMR_DTYPE_F32: i32 = 0;
pub const MMR_DTYPE_BF16: i32 = 1;
pub const MMR_DTYPE_F16: i32 = 2;
pub const MMR_DTYPE_I32: i32 = 3;

pub const MMR_ACT_NONE: i32 = 0;
pub const MMR_ACT_RELU: i32 = 1;
pub const MMR_ACT_RELU6: i32 = 2;
pub const MMR_ACT_GELU_ERF: i32 = 3;
pub const MMR_ACT_GELU_TANH: i32 = 4;
pub const MMR_ACT_SILU: i32 = 5;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_tensor {
    pub view: mmr_view,
    pub dtype: i32,
    pub reserved: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_linear_desc {
    pub lhs: mmr_tensor,
    pub rhs: mmr_tensor,
    pub out: mmr_tensor,
    pub bias: mmr_tensor,
    pub residual: mmr_tensor,
    pub pre: mmr_tensor,
    pub transpose_lhs: i32,
    pub transpose_rhs: i32,
    pub activation: i32,
    pub math_mode: i32,
    pub device_ordinal: i32,
    pub reserved: i32,
    pub stream: *mut c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_linear_grad_desc {
    pub d_out: mmr_tensor,
    pub lhs: mmr_tensor,
    pub rhs: mmr_tensor,
    pub pre: mmr_tensor,
    pub d_lhs: mmr_tensor,
    pub d_rhs: mmr_tensor,
    pub d_bias: mmr_tensor,
    pub transpose_lhs: i32,
    pub transpose_rhs: i32,
    pub activation: i32,
    pub math_mode: i32,
    pub device_ordinal: i32,
    pub reserved: i32,
    pub stream: *mut c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_expert_layout {
    pub tokens: i64,
    pub top_k: i64,
    pub experts: i64,
    pub row_align: i64,
    pub slots: mmr_tensor,
    pub sources: mmr_tensor,
    pub offsets: mmr_tensor,
    pub counts: mmr_tensor,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_dispatch_desc {
    pub layout: mmr_expert_layout,
    pub ids: mmr_tensor,
    pub x: mmr_tensor,
    pub rows: mmr_tensor,
    pub device_ordinal: i32,
    pub reserved: i32,
    pub stream: *mut c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_combine_desc {
    pub layout: mmr_expert_layout,
    pub rows: mmr_tensor,
    pub weights: mmr_tensor,
    pub residual: mmr_tensor,
    pub out: mmr_tensor,
    pub device_ordinal: i32,
    pub reserved: i32,
    pub stream: *mut c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_combine_grad_desc {
    pub layout: mmr_expert_layout,
    pub d_out: mmr_tensor,
    pub rows: mmr_tensor,
    pub weights: mmr_tensor,
    pub d_rows: mmr_tensor,
    pub d_weights: mmr_tensor,
    pub device_ordinal: i32,
    pub reserved: i32,
    pub stream: *mut c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_expert_linear_desc {
    pub layout: mmr_expert_layout,
    pub rows: mmr_tensor,
    pub weights: mmr_tensor,
    pub bias: mmr_tensor,
    pub out: mmr_tensor,
    pub pre: mmr_tensor,
    pub transpose_rhs: i32,
    pub activation: i32,
    pub device_ordinal: i32,
    pub reserved: i32,
    pub stream: *mut c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mmr_expert_linear_grad_desc {
    pub layout: mmr_expert_layout,
    pub d_out: mmr_tensor,
    pub rows: mmr_tensor,
    pub weights: mmr_tensor,
    pub pre: mmr_tensor,
    pub d_rows: mmr_tensor,
    pub d_weights: mmr_tensor,
    pub d_bias: mmr_tensor,
    pub transpose_rhs: i32,
    pub activation: i32,
    pub device_ordinal: i32,
    pub reserved: i32,
    pub stream: *mut c_void,
}

#[repr(C)]
pub struct mmr_op_handle {
    _private: [u8; 0],
}

extern "C" {
    pub fn mmr_expert_rows(tokens: i64, top_k: i64, experts: i64, row_align: i64, rows: *mut i64) -> i32;
    pub fn mmr_linear_bind(desc: *const mmr_linear_desc, out: *mut *mut mmr_op_handle) -> i32;
    pub fn mmr_linear_grad_bind(desc: *const mmr_linear_grad_desc, out: *mut *mut mmr_op_handle) -> i32;
    pub fn mmr_dispatch_bind(desc: *const mmr_dispatch_desc, out: *mut *mut mmr_op_handle) -> i32;
    pub fn mmr_combine_bind(desc: *const mmr_combine_desc, out: *mut *mut mmr_op_handle) -> i32;
    pub fn mmr_combine_grad_bind(desc: *const mmr_combine_grad_desc, out: *mut *mut mmr_op_handle) -> i32;
    pub fn mmr_expert_linear_bind(desc: *const mmr_expert_linear_desc, out: *mut *mut mmr_op_handle) -> i32;
    pub fn mmr_expert_linear_grad_bind(desc: *const mmr_expert_linear_grad_desc, out: *mut *mut mmr_op_handle) -> i32;
    pub fn mmr_op_run(h: *mut mmr_op_handle) -> i32;
    pub fn mmr_op_run_on(h: *mut mmr_op_handle, stream: *mut c_void) -> i32;
    pub fn mmr_op_quiesce(h: *mut mmr_op_handle, timeout_ns: u64) -> i32;
    pub fn mmr_op_destroy(h: *mut mmr_op_handle) -> i32;
    pub fn mmr_op_plan(h: *const mmr_op_handle) -> *const c_char;
}
