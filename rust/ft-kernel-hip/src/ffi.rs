// GENERATED by generate_bindings.py from include/ft_kernel_hip.h. Do not edit: change the header and regenerate.
//
// The C ABI of libft_kernel_hip.so, declaration for declaration: status codes and tags, the plain-data structs,
// the opaque handles, and every exported function.

#![allow(non_camel_case_types, non_snake_case, dead_code, clippy::too_many_arguments)]

use std::os::raw::{c_char, c_void};

/// A `hipStream_t`; null selects the library's own ordered stream.
pub type fth_stream = *mut c_void;
/// A `hipEvent_t`.
pub type fth_event = *mut c_void;

pub const FTH_OK: i32 = 0;
pub const FTH_ERR_DTYPE_MISMATCH: i32 = 1;
pub const FTH_ERR_DEVICE_MISMATCH: i32 = 2;
pub const FTH_ERR_SHAPE_MISMATCH: i32 = 3;
pub const FTH_ERR_UNSUPPORTED_LAYOUT: i32 = 4;
pub const FTH_ERR_STORAGE_SPAN_OVERFLOW: i32 = 5;
pub const FTH_ERR_INSUFFICIENT_STORAGE: i32 = 6;
pub const FTH_ERR_INVALID_DIMENSION: i32 = 7;
pub const FTH_ERR_SHAPE_OVERFLOW: i32 = 8;
pub const FTH_ERR_EMPTY_REDUCTION_DIM: i32 = 9;
pub const FTH_ERR_UNAVAILABLE: i32 = 100;
pub const FTH_ERR_KERNEL: i32 = 101;
pub const FTH_ERR_SIZE_OVERFLOW: i32 = 102;
pub const FTH_ERR_BUFFER_TOO_LARGE: i32 = 103;
pub const FTH_ERR_STREAM: i32 = 104;
pub const FTH_ERR_INVALID_ARGUMENT: i32 = 105;
pub const FTH_ERR_OUTPUT_TOO_SMALL: i32 = 106;
pub const FTH_ERR_CORRUPT: i32 = 107;
pub const FTH_ERR_IO: i32 = 108;
pub const FTH_ERR_INVALID_MAGIC: i32 = 109;
pub const FTH_ERR_UNSUPPORTED_VERSION: i32 = 110;
pub const FTH_DTYPE_F64: i32 = 0;
pub const FTH_DTYPE_F32: i32 = 1;
pub const FTH_DTYPE_F16: i32 = 2;
pub const FTH_DTYPE_BF16: i32 = 3;
pub const FTH_DTYPE_I8: i32 = 16;
pub const FTH_DTYPE_E4M3: i32 = 17;
pub const FTH_DEVICE_CPU: i32 = 0;
pub const FTH_DEVICE_CUDA: i32 = 1;
pub const FTH_DEVICE_HIP: i32 = 2;
pub const FTH_EPI_NONE: i32 = 0;
pub const FTH_EPI_BIAS: i32 = 1;
pub const FTH_EPI_GELU: i32 = 2;
pub const FTH_EPI_RESIDUAL: i32 = 4;
pub const FTH_EPI_GELU_TANH: i32 = 8;
pub const FTH_ACT_GELU_ERF: i32 = 0;
pub const FTH_ACT_GELU_TANH: i32 = 1;
pub const FTH_MAX_DIMS: usize = 8;

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_meta {
    pub ndim: i32,
    pub dtype: i32,
    pub device: i32,
    pub reserved: i32,
    pub shape: [u64; 8],
    pub strides: [u64; 8],
    pub storage_offset: u64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_error_info {
    pub code: i32,
    pub lhs_ndim: i32,
    pub rhs_ndim: i32,
    pub reserved: i32,
    pub lhs_shape: [u64; 8],
    pub rhs_shape: [u64; 8],
    pub a: u64,
    pub b: u64,
    pub side: [c_char; 16],
    pub message: [c_char; 200],
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_gemm_desc {
    pub m: i64,
    pub n: i64,
    pub k: i64,
    pub lda: i64,
    pub ldb: i64,
    pub ldc: i64,
    pub batch: i64,
    pub stride_a: i64,
    pub stride_b: i64,
    pub stride_c: i64,
    pub trans_b: i32,
    pub epilogue: i32,
    pub trans_a: i32,
    pub reserved: i32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_sdpa_desc {
    pub num_bh: i64,
    pub heads: i64,
    pub seq_q: i64,
    pub seq_k: i64,
    pub d_k: i64,
    pub d_v: i64,
    pub q_batch_stride: i64,
    pub q_head_stride: i64,
    pub q_row_stride: i64,
    pub k_batch_stride: i64,
    pub k_head_stride: i64,
    pub k_row_stride: i64,
    pub v_batch_stride: i64,
    pub v_head_stride: i64,
    pub v_row_stride: i64,
    pub o_batch_stride: i64,
    pub o_head_stride: i64,
    pub o_row_stride: i64,
    pub causal: i32,
    pub kv_group: i32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_paged_cache {
    pub num_pages: i64,
    pub page_size: i64,
    pub kv_heads: i64,
    pub head_dim: i64,
    pub page_stride: i64,
    pub head_stride: i64,
    pub row_stride: i64,
    pub num_seqs: i64,
    pub max_pages: i64,
    pub table_stride: i64,
    pub dtype: i32,
    pub reserved: i32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_paged_append_desc {
    pub tokens: i64,
    pub q_heads: i64,
    pub q_row_stride: i64,
    pub q_head_stride: i64,
    pub k_row_stride: i64,
    pub k_head_stride: i64,
    pub v_row_stride: i64,
    pub v_head_stride: i64,
    pub out_row_stride: i64,
    pub out_head_stride: i64,
    pub rotary_dim: i64,
    pub max_pos: i64,
    pub interleaved: i32,
    pub reserved: i32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_paged_sdpa_desc {
    pub q_heads: i64,
    pub new_tokens: i64,
    pub max_len: i64,
    pub q_seq_stride: i64,
    pub q_row_stride: i64,
    pub q_head_stride: i64,
    pub o_seq_stride: i64,
    pub o_row_stride: i64,
    pub o_head_stride: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_paged_scales {
    pub block: i64,
    pub page_stride: i64,
    pub head_stride: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_logits_desc {
    pub rows: i64,
    pub vocab: i64,
    pub logits_stride: i64,
    pub out_stride: i64,
    pub history_stride: i64,
    pub bias_stride: i64,
    pub mask_stride: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_sample_desc {
    pub rows: i64,
    pub vocab: i64,
    pub logits_stride: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_layer_weights {
    pub ln1_w: *const f32,
    pub ln1_b: *const f32,
    pub wq: *const f32,
    pub bq: *const f32,
    pub wk: *const f32,
    pub bk: *const f32,
    pub wv: *const f32,
    pub bv: *const f32,
    pub wo: *const f32,
    pub bo: *const f32,
    pub ln2_w: *const f32,
    pub ln2_b: *const f32,
    pub w1: *const f32,
    pub b1: *const f32,
    pub w2: *const f32,
    pub b2: *const f32,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fth_safetensors_tensor {
    pub dtype: i32,
    pub ndim: i32,
    pub shape: [u64; 8],
    pub numel: u64,
    pub byte_len: u64,
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct fth_tensor {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct fth_batch {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct fth_encoder {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct fth_safetensors {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct fth_gpt2 {
    _private: [u8; 0],
}

pub type fth_statedict = fth_safetensors;

#[link(name = "ft_kernel_hip")]
extern "C" {
    pub fn fth_last_error(out: *mut fth_error_info) -> i32;
    pub fn fth_status_name(code: i32) -> *const c_char;
    pub fn fth_is_available() -> i32;
    pub fn fth_device_info(arch: *mut c_char, arch_cap: usize, compute_units: *mut i32, hbm_bytes: *mut u64, engine_clock_khz: *mut i32, memory_clock_khz: *mut i32) -> i32;
    pub fn fth_malloc(dptr: *mut *mut c_void, bytes: usize) -> i32;
    pub fn fth_free(dptr: *mut c_void) -> i32;
    pub fn fth_memcpy_h2d(dst_dev: *mut c_void, src_host: *const c_void, bytes: usize) -> i32;
    pub fn fth_memcpy_d2h(dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> i32;
    pub fn fth_memcpy_d2d(dst_dev: *mut c_void, src_dev: *const c_void, bytes: usize) -> i32;
    pub fn fth_memset_zero(dst_dev: *mut c_void, bytes: usize) -> i32;
    pub fn fth_device_memory_info(free_bytes: *mut u64, total_bytes: *mut u64) -> i32;
    pub fn fth_device_workspace_info(live_bytes: *mut u64, retired_bytes: *mut u64) -> i32;
    pub fn fth_host_malloc(hptr: *mut *mut c_void, bytes: usize) -> i32;
    pub fn fth_host_free(hptr: *mut c_void) -> i32;
    pub fn fth_memcpy_async(dst: *mut c_void, src: *const c_void, bytes: usize, kind: i32, s: fth_stream) -> i32;
    pub fn fth_stream_create(s: *mut fth_stream) -> i32;
    pub fn fth_stream_destroy(s: fth_stream) -> i32;
    pub fn fth_stream_synchronize(s: fth_stream) -> i32;
    pub fn fth_device_synchronize() -> i32;
    pub fn fth_event_create(e: *mut fth_event) -> i32;
    pub fn fth_event_destroy(e: fth_event) -> i32;
    pub fn fth_event_record(e: fth_event, s: fth_stream) -> i32;
    pub fn fth_event_synchronize(e: fth_event) -> i32;
    pub fn fth_event_elapsed_ms(start: fth_event, stop: fth_event, ms: *mut f32) -> i32;
    pub fn fth_dev_softmax_lastdim_f32(x: *const f32, y: *mut f32, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_softmax_lastdim_f64(x: *const f64, y: *mut f64, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_softmax_strided_f32(x: *const f32, y: *mut f32, outer: i64, reduce: i64, inner: i64, s: fth_stream) -> i32;
    pub fn fth_dev_softmax_strided_f64(x: *const f64, y: *mut f64, outer: i64, reduce: i64, inner: i64, s: fth_stream) -> i32;
    pub fn fth_dev_layer_norm_f32(x: *const f32, weight: *const f32, bias: *const f32, y: *mut f32, batch: i64, norm_size: i64, eps: f32, s: fth_stream) -> i32;
    pub fn fth_dev_layer_norm_f64(x: *const f64, weight: *const f64, bias: *const f64, y: *mut f64, batch: i64, norm_size: i64, eps: f64, s: fth_stream) -> i32;
    pub fn fth_dev_add_layer_norm_f32(a: *const f32, b: *const f32, weight: *const f32, bias: *const f32, y: *mut f32, batch: i64, norm_size: i64, eps: f32, s: fth_stream) -> i32;
    pub fn fth_dev_rms_norm_f32(x: *const f32, weight: *const f32, y: *mut f32, batch: i64, norm_size: i64, eps: f32, s: fth_stream) -> i32;
    pub fn fth_dev_rms_norm_f64(x: *const f64, weight: *const f64, y: *mut f64, batch: i64, norm_size: i64, eps: f64, s: fth_stream) -> i32;
    pub fn fth_dev_gelu_f32(x: *const f32, y: *mut f32, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_gelu_f64(x: *const f64, y: *mut f64, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_gelu_tanh_f32(x: *const f32, y: *mut f32, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_gelu_tanh_f64(x: *const f64, y: *mut f64, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_add_f32(a: *const f32, b: *const f32, y: *mut f32, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_add_f64(a: *const f64, b: *const f64, y: *mut f64, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_copy_f32(x: *const f32, y: *mut f32, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_copy_f64(x: *const f64, y: *mut f64, n: i64, s: fth_stream) -> i32;
    pub fn fth_dev_bias_add_f32(x: *const f32, bias: *const f32, y: *mut f32, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_bias_add_f64(x: *const f64, bias: *const f64, y: *mut f64, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_bias_residual_add_f32(x: *const f32, bias: *const f32, residual: *const f32, y: *mut f32, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_bias_residual_add_f64(x: *const f64, bias: *const f64, residual: *const f64, y: *mut f64, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_index_select_f32(input: *const f32, outer: i64, dim_size: i64, inner: i64, indices: *const f64, num_indices: i64, out: *mut f32, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_index_select_f64(input: *const f64, outer: i64, dim_size: i64, inner: i64, indices: *const f64, num_indices: i64, out: *mut f64, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_embedding_add_f32(wte: *const f32, vocab: i64, wpe: *const f32, max_pos: i64, ids: *const f64, tokens: i64, seq: i64, width: i64, out: *mut f32, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_argmax_f32(x: *const f32, outer: i64, reduce: i64, inner: i64, out: *mut f32, s: fth_stream) -> i32;
    pub fn fth_dev_argmax_f64(x: *const f64, outer: i64, reduce: i64, inner: i64, out: *mut f64, s: fth_stream) -> i32;
    pub fn fth_dev_linear_argmax_workspace_floats(rows: i64, out_features: i64) -> i64;
    pub fn fth_dev_linear_argmax_f32(x: *const f32, w: *const f32, rows: i64, out_features: i64, in_features: i64, logits: *mut f32, argmax: *mut f32, workspace: *mut f32, workspace_floats: i64, s: fth_stream) -> i32;
    pub fn fth_dev_permute_0213_f32(src: *const f32, dst: *mut f32, d0: i64, d1: i64, d2: i64, d3: i64, s: fth_stream) -> i32;
    pub fn fth_dev_permute_0213_f64(src: *const f64, dst: *mut f64, d0: i64, d1: i64, d2: i64, d3: i64, s: fth_stream) -> i32;
    pub fn fth_dev_transpose_2d_f32(src: *const f32, dst: *mut f32, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_transpose_2d_f64(src: *const f64, dst: *mut f64, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_transpose_batched_f32(src: *const f32, dst: *mut f32, batch: i64, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_transpose_batched_f64(src: *const f64, dst: *mut f64, batch: i64, rows: i64, cols: i64, s: fth_stream) -> i32;
    pub fn fth_dev_gemm_f32(d: *const fth_gemm_desc, alpha: f32, a: *const f32, b: *const f32, c: *mut f32, bias: *const f32, residual: *const f32, s: fth_stream) -> i32;
    pub fn fth_dev_gemm_f64(d: *const fth_gemm_desc, alpha: f64, a: *const f64, b: *const f64, c: *mut f64, bias: *const f64, residual: *const f64, s: fth_stream) -> i32;
    pub fn fth_dev_log_softmax_strided_f32(x: *const f32, y: *mut f32, outer: i64, reduce: i64, inner: i64, s: fth_stream) -> i32;
    pub fn fth_dev_log_softmax_strided_f64(x: *const f64, y: *mut f64, outer: i64, reduce: i64, inner: i64, s: fth_stream) -> i32;
    pub fn fth_dev_cross_entropy_forward_f32(logits: *const f32, target: *const i64, batch: i64, classes: i64, loss: *mut f32, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_cross_entropy_forward_f64(logits: *const f64, target: *const i64, batch: i64, classes: i64, loss: *mut f64, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_cross_entropy_backward_f32(logits: *const f32, target: *const i64, dloss: *const f32, batch: i64, classes: i64, dlogits: *mut f32, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_cross_entropy_backward_f64(logits: *const f64, target: *const i64, dloss: *const f64, batch: i64, classes: i64, dlogits: *mut f64, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_quantize_rows_i8(x: *const f32, rows: i64, cols: i64, q: *mut i8, scales: *mut f32, s: fth_stream) -> i32;
    pub fn fth_dev_linear_int8_workspace_bytes(m: i64, k: i64) -> usize;
    pub fn fth_dev_linear_int8_dynamic_f32(x: *const f32, m: i64, k: i64, w_i8: *const i8, w_scales: *const f32, n: i64, bias: *const f32, out: *mut f32, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_linear_int8_prequantized_f32(x_i8: *const i8, a_scales: *const f32, m: i64, k: i64, w_i8: *const i8, w_scales: *const f32, n: i64, bias: *const f32, out: *mut f32, s: fth_stream) -> i32;
    pub fn fth_dev_norm_backward_workspace_bytes(rows: i64, cols: i64, dtype: i32) -> usize;
    pub fn fth_dev_layer_norm_backward_f32(dy: *const f32, x: *const f32, weight: *const f32, rows: i64, cols: i64, eps: f32, dx: *mut f32, dweight: *mut f32, dbias: *mut f32, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_layer_norm_backward_f64(dy: *const f64, x: *const f64, weight: *const f64, rows: i64, cols: i64, eps: f64, dx: *mut f64, dweight: *mut f64, dbias: *mut f64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_layer_norm_backward_noalloc_max_bytes() -> usize;
    pub fn fth_dev_layer_norm_backward_f32_noalloc(dy: *const f32, x: *const f32, weight: *const f32, rows: i64, cols: i64, eps: f32, dx: *mut f32, dweight: *mut f32, dbias: *mut f32, s: fth_stream) -> i32;
    pub fn fth_dev_rms_norm_backward_f32(dy: *const f32, x: *const f32, weight: *const f32, rows: i64, cols: i64, eps: f32, dx: *mut f32, dweight: *mut f32, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_rms_norm_backward_f64(dy: *const f64, x: *const f64, weight: *const f64, rows: i64, cols: i64, eps: f64, dx: *mut f64, dweight: *mut f64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_linear_backward_workspace_bytes(batch: i64, out_features: i64, dtype: i32) -> usize;
    pub fn fth_dev_linear_backward_f32(dy: *const f32, x: *const f32, weight: *const f32, batch: i64, in_features: i64, out_features: i64, dx: *mut f32, dweight: *mut f32, dbias: *mut f32, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_linear_backward_f64(dy: *const f64, x: *const f64, weight: *const f64, batch: i64, in_features: i64, out_features: i64, dx: *mut f64, dweight: *mut f64, dbias: *mut f64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_backward_workspace_bytes(num_bh: i64, seq_q: i64, seq_k: i64, dtype: i32) -> usize;
    pub fn fth_dev_sdpa_backward_f32(q: *const f32, k: *const f32, v: *const f32, dout: *const f32, num_bh: i64, seq_q: i64, seq_k: i64, d_k: i64, d_v: i64, scale: f32, causal: i32, dq: *mut f32, dk: *mut f32, dv: *mut f32, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_backward_f64(q: *const f64, k: *const f64, v: *const f64, dout: *const f64, num_bh: i64, seq_q: i64, seq_k: i64, d_k: i64, d_v: i64, scale: f64, causal: i32, dq: *mut f64, dk: *mut f64, dv: *mut f64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_backward_unit_dout_workspace_bytes(num_bh: i64, seq_q: i64, seq_k: i64, d_v: i64, dtype: i32) -> usize;
    pub fn fth_dev_sdpa_backward_unit_dout_f32(q: *const f32, k: *const f32, v: *const f32, num_bh: i64, seq_q: i64, seq_k: i64, d_k: i64, d_v: i64, scale: f32, causal: i32, dq: *mut f32, dk: *mut f32, dv: *mut f32, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_backward_unit_dout_f64(q: *const f64, k: *const f64, v: *const f64, num_bh: i64, seq_q: i64, seq_k: i64, d_k: i64, d_v: i64, scale: f64, causal: i32, dq: *mut f64, dk: *mut f64, dv: *mut f64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_backward_masked_f32(q: *const f32, k: *const f32, v: *const f32, dout: *const f32, num_bh: i64, seq_q: i64, seq_k: i64, d_k: i64, d_v: i64, scale: f32, mask: *const f32, mask_bh_stride: i64, dq: *mut f32, dk: *mut f32, dv: *mut f32, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_backward_masked_f64(q: *const f64, k: *const f64, v: *const f64, dout: *const f64, num_bh: i64, seq_q: i64, seq_k: i64, d_k: i64, d_v: i64, scale: f64, mask: *const f64, mask_bh_stride: i64, dq: *mut f64, dk: *mut f64, dv: *mut f64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_sdpa_desc_contiguous(d: *mut fth_sdpa_desc, num_bh: i64, seq_q: i64, seq_k: i64, d_k: i64, d_v: i64, causal: i32);
    pub fn fth_dev_sdpa_forward_f32(d: *const fth_sdpa_desc, scale: f32, q: *const f32, k: *const f32, v: *const f32, out: *mut f32, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_forward_f64(d: *const fth_sdpa_desc, scale: f64, q: *const f64, k: *const f64, v: *const f64, out: *mut f64, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_forward_masked_f32(d: *const fth_sdpa_desc, scale: f32, q: *const f32, k: *const f32, v: *const f32, mask: *const f32, mask_bh_stride: i64, out: *mut f32, s: fth_stream) -> i32;
    pub fn fth_dev_sdpa_forward_masked_f64(d: *const fth_sdpa_desc, scale: f64, q: *const f64, k: *const f64, v: *const f64, mask: *const f64, mask_bh_stride: i64, out: *mut f64, s: fth_stream) -> i32;
    pub fn fth_dev_paged_cache_contiguous(c: *mut fth_paged_cache, num_pages: i64, page_size: i64, kv_heads: i64, head_dim: i64, num_seqs: i64, max_pages: i64, dtype: i32);
    pub fn fth_dev_paged_append_f32(c: *const fth_paged_cache, d: *const fth_paged_append_desc, q: *const f32, k: *const f32, v: *const f32, cosines: *const f32, sines: *const f32, block_table: *const i32, seq_ids: *const i32, positions: *const i32, q_out: *mut f32, k_cache: *mut c_void, v_cache: *mut c_void, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_paged_sdpa_workspace_bytes(c: *const fth_paged_cache, d: *const fth_paged_sdpa_desc) -> usize;
    pub fn fth_dev_paged_sdpa_f32(c: *const fth_paged_cache, d: *const fth_paged_sdpa_desc, scale: f32, q: *const f32, k_cache: *const c_void, v_cache: *const c_void, block_table: *const i32, lens: *const i32, out: *mut f32, bad_index: *mut i64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_paged_scales_contiguous(sc: *mut fth_paged_scales, c: *const fth_paged_cache, block: i64);
    pub fn fth_dev_paged_append_scaled_f32(c: *const fth_paged_cache, sc: *const fth_paged_scales, d: *const fth_paged_append_desc, q: *const f32, k: *const f32, v: *const f32, cosines: *const f32, sines: *const f32, block_table: *const i32, seq_ids: *const i32, positions: *const i32, q_out: *mut f32, k_cache: *mut c_void, v_cache: *mut c_void, k_scales: *mut f32, v_scales: *mut f32, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_paged_sdpa_scaled_workspace_bytes(c: *const fth_paged_cache, sc: *const fth_paged_scales, d: *const fth_paged_sdpa_desc) -> usize;
    pub fn fth_dev_paged_sdpa_scaled_f32(c: *const fth_paged_cache, sc: *const fth_paged_scales, d: *const fth_paged_sdpa_desc, scale: f32, q: *const f32, k_cache: *const c_void, v_cache: *const c_void, k_scales: *const f32, v_scales: *const f32, block_table: *const i32, lens: *const i32, out: *mut f32, bad_index: *mut i64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_dev_logits_process_f32(d: *const fth_logits_desc, logits: *const f32, history: *const i32, history_len: *const i32, prompt_len: *const i32, repetition: *const f32, frequency: *const f32, presence: *const f32, bias: *const f32, mask: *const u32, out: *mut f32, bad_index: *mut i64, s: fth_stream) -> i32;
    pub fn fth_dev_sample_workspace_bytes(d: *const fth_sample_desc) -> usize;
    pub fn fth_dev_sample_f32(d: *const fth_sample_desc, logits: *const f32, temperature: *const f32, top_k: *const i32, top_p: *const f32, min_p: *const f32, uniform: *const f64, tokens: *mut i32, logprobs: *mut f32, bad_index: *mut i64, workspace: *mut c_void, workspace_bytes: usize, s: fth_stream) -> i32;
    pub fn fth_matmul_tensor_contiguous_f32(lhs: *const f32, lhs_len: usize, rhs: *const f32, rhs_len: usize, lhs_meta: *const fth_meta, rhs_meta: *const fth_meta, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_matmul_tensor_contiguous_f64(lhs: *const f64, lhs_len: usize, rhs: *const f64, rhs_len: usize, lhs_meta: *const fth_meta, rhs_meta: *const fth_meta, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_bmm_tensor_contiguous_f32(lhs: *const f32, lhs_len: usize, rhs: *const f32, rhs_len: usize, lhs_meta: *const fth_meta, rhs_meta: *const fth_meta, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_bmm_tensor_contiguous_f64(lhs: *const f64, lhs_len: usize, rhs: *const f64, rhs_len: usize, lhs_meta: *const fth_meta, rhs_meta: *const fth_meta, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_addmm_tensor_contiguous_f32(input: *const f32, input_len: usize, mat1: *const f32, mat1_len: usize, mat2: *const f32, mat2_len: usize, input_meta: *const fth_meta, mat1_meta: *const fth_meta, mat2_meta: *const fth_meta, beta: f32, alpha: f32, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_addmm_tensor_contiguous_f64(input: *const f64, input_len: usize, mat1: *const f64, mat1_len: usize, mat2: *const f64, mat2_len: usize, input_meta: *const fth_meta, mat1_meta: *const fth_meta, mat2_meta: *const fth_meta, beta: f64, alpha: f64, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_linear_tensor_f32(x: *const f32, x_len: usize, weight: *const f32, weight_len: usize, bias: *const f32, bias_len: usize, batch: usize, in_features: usize, out_features: usize, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_linear_tensor_f64(x: *const f64, x_len: usize, weight: *const f64, weight_len: usize, bias: *const f64, bias_len: usize, batch: usize, in_features: usize, out_features: usize, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_matmul_rhs_transposed_contiguous_f32(m: usize, k: usize, n: usize, lhs: *const f32, lhs_len: usize, rhs_nk: *const f32, rhs_len: usize, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_matmul_rhs_transposed_contiguous_f64(m: usize, k: usize, n: usize, lhs: *const f64, lhs_len: usize, rhs_nk: *const f64, rhs_len: usize, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_softmax_dim_tensor_contiguous_f32(input: *const f32, input_len: usize, meta: *const fth_meta, dim: usize, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_softmax_dim_tensor_contiguous_f64(input: *const f64, input_len: usize, meta: *const fth_meta, dim: usize, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_layer_norm_forward_f32(x: *const f32, x_len: usize, weight: *const f32, bias: *const f32, batch: usize, norm_size: usize, eps: f32, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_layer_norm_forward_f64(x: *const f64, x_len: usize, weight: *const f64, bias: *const f64, batch: usize, norm_size: usize, eps: f64, out: *mut f64, out_cap: usize) -> i32;
    pub fn fth_add_layer_norm_forward_f32(a: *const f32, b: *const f32, ab_len: usize, weight: *const f32, bias: *const f32, batch: usize, norm_size: usize, eps: f32, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_rms_norm_forward_f32(x: *const f32, x_len: usize, weight: *const f32, batch: usize, norm_size: usize, eps: f32, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_rms_norm_forward_f64(x: *const f64, x_len: usize, weight: *const f64, batch: usize, norm_size: usize, eps: f64, out: *mut f64, out_cap: usize) -> i32;
    pub fn fth_quantize_per_output_channel_i8(w: *const f32, w_len: usize, rows: usize, cols: usize, q: *mut i8, q_cap: usize, scales: *mut f32, scales_cap: usize) -> i32;
    pub fn fth_quantize_rows_i8(x: *const f32, x_len: usize, rows: usize, cols: usize, q: *mut i8, q_cap: usize, scales: *mut f32, scales_cap: usize) -> i32;
    pub fn fth_linear_int8_dynamic_f32(x: *const f32, x_len: usize, m: usize, k: usize, w_i8: *const i8, w_len: usize, w_scales: *const f32, w_scales_len: usize, n: usize, bias: *const f32, bias_len: usize, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_sdpa_forward_masked_f32(q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f32, mask: *const f32, mask_len: usize, mask_bh_stride: usize, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_sdpa_forward_masked_f64(q: *const f64, q_len: usize, k: *const f64, k_len: usize, v: *const f64, v_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f64, mask: *const f64, mask_len: usize, mask_bh_stride: usize, out: *mut f64, out_cap: usize) -> i32;
    pub fn fth_sdpa_forward_masked_gqa_f32(q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, batch: usize, h_q: usize, h_kv: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f32, mask: *const f32, mask_len: usize, mask_bh_stride: usize, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_sdpa_forward_masked_gqa_f64(q: *const f64, q_len: usize, k: *const f64, k_len: usize, v: *const f64, v_len: usize, batch: usize, h_q: usize, h_kv: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f64, mask: *const f64, mask_len: usize, mask_bh_stride: usize, out: *mut f64, out_cap: usize) -> i32;
    pub fn fth_log_softmax_dim_tensor_contiguous_f32(input: *const f32, input_len: usize, meta: *const fth_meta, dim: usize, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_log_softmax_dim_tensor_contiguous_f64(input: *const f64, input_len: usize, meta: *const fth_meta, dim: usize, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_cross_entropy_forward_f32(logits: *const f32, logits_len: usize, target: *const u64, target_len: usize, batch: usize, classes: usize, loss: *mut f32, loss_cap: usize) -> i32;
    pub fn fth_cross_entropy_forward_f64(logits: *const f64, logits_len: usize, target: *const u64, target_len: usize, batch: usize, classes: usize, loss: *mut f64, loss_cap: usize) -> i32;
    pub fn fth_cross_entropy_backward_f32(logits: *const f32, logits_len: usize, target: *const u64, target_len: usize, dloss: *const f32, dloss_len: usize, batch: usize, classes: usize, dlogits: *mut f32, dlogits_cap: usize) -> i32;
    pub fn fth_cross_entropy_backward_f64(logits: *const f64, logits_len: usize, target: *const u64, target_len: usize, dloss: *const f64, dloss_len: usize, batch: usize, classes: usize, dlogits: *mut f64, dlogits_cap: usize) -> i32;
    pub fn fth_layer_norm_backward_f32(dy: *const f32, dy_len: usize, x: *const f32, x_len: usize, weight: *const f32, batch: usize, norm_size: usize, eps: f32, dx: *mut f32, dx_cap: usize, dweight: *mut f32, dweight_cap: usize, dbias: *mut f32, dbias_cap: usize) -> i32;
    pub fn fth_layer_norm_backward_f64(dy: *const f64, dy_len: usize, x: *const f64, x_len: usize, weight: *const f64, batch: usize, norm_size: usize, eps: f64, dx: *mut f64, dx_cap: usize, dweight: *mut f64, dweight_cap: usize, dbias: *mut f64, dbias_cap: usize) -> i32;
    pub fn fth_rms_norm_backward_f32(dy: *const f32, dy_len: usize, x: *const f32, x_len: usize, weight: *const f32, batch: usize, norm_size: usize, eps: f32, dx: *mut f32, dx_cap: usize, dweight: *mut f32, dweight_cap: usize) -> i32;
    pub fn fth_rms_norm_backward_f64(dy: *const f64, dy_len: usize, x: *const f64, x_len: usize, weight: *const f64, batch: usize, norm_size: usize, eps: f64, dx: *mut f64, dx_cap: usize, dweight: *mut f64, dweight_cap: usize) -> i32;
    pub fn fth_linear_backward_f32(dy: *const f32, dy_len: usize, x: *const f32, x_len: usize, weight: *const f32, weight_len: usize, batch: usize, in_features: usize, out_features: usize, need_bias: i32, dx: *mut f32, dx_cap: usize, dweight: *mut f32, dweight_cap: usize, dbias: *mut f32, dbias_cap: usize) -> i32;
    pub fn fth_linear_backward_f64(dy: *const f64, dy_len: usize, x: *const f64, x_len: usize, weight: *const f64, weight_len: usize, batch: usize, in_features: usize, out_features: usize, need_bias: i32, dx: *mut f64, dx_cap: usize, dweight: *mut f64, dweight_cap: usize, dbias: *mut f64, dbias_cap: usize) -> i32;
    pub fn fth_sdpa_backward_f32(q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, dout: *const f32, dout_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f32, causal: i32, dq: *mut f32, dq_cap: usize, dk: *mut f32, dk_cap: usize, dv: *mut f32, dv_cap: usize) -> i32;
    pub fn fth_sdpa_backward_f64(q: *const f64, q_len: usize, k: *const f64, k_len: usize, v: *const f64, v_len: usize, dout: *const f64, dout_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f64, causal: i32, dq: *mut f64, dq_cap: usize, dk: *mut f64, dk_cap: usize, dv: *mut f64, dv_cap: usize) -> i32;
    pub fn fth_sdpa_backward_f32_unit_dout(q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f32, causal: i32, dq: *mut f32, dq_cap: usize, dk: *mut f32, dk_cap: usize, dv: *mut f32, dv_cap: usize) -> i32;
    pub fn fth_sdpa_backward_masked_f32(q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, dout: *const f32, dout_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f32, mask: *const f32, mask_len: usize, mask_bh_stride: usize, dq: *mut f32, dq_cap: usize, dk: *mut f32, dk_cap: usize, dv: *mut f32, dv_cap: usize) -> i32;
    pub fn fth_sdpa_backward_masked_f64(q: *const f64, q_len: usize, k: *const f64, k_len: usize, v: *const f64, v_len: usize, dout: *const f64, dout_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f64, mask: *const f64, mask_len: usize, mask_bh_stride: usize, dq: *mut f64, dq_cap: usize, dk: *mut f64, dk_cap: usize, dv: *mut f64, dv_cap: usize) -> i32;
    pub fn fth_gelu_tensor_contiguous_f32(input: *const f32, input_len: usize, meta: *const fth_meta, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_gelu_tanh_tensor_contiguous_f32(input: *const f32, input_len: usize, meta: *const fth_meta, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_gelu_tanh_tensor_contiguous_f64(input: *const f64, input_len: usize, meta: *const fth_meta, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_gelu_tensor_contiguous_f64(input: *const f64, input_len: usize, meta: *const fth_meta, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_add_tensor_contiguous_f32(lhs: *const f32, lhs_len: usize, rhs: *const f32, rhs_len: usize, lhs_meta: *const fth_meta, rhs_meta: *const fth_meta, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_add_tensor_contiguous_f64(lhs: *const f64, lhs_len: usize, rhs: *const f64, rhs_len: usize, lhs_meta: *const fth_meta, rhs_meta: *const fth_meta, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_transpose_2d_into_f32(src: *const f32, src_len: usize, dst: *mut f32, dst_cap: usize, rows: usize, cols: usize) -> i32;
    pub fn fth_transpose_2d_into_f64(src: *const f64, src_len: usize, dst: *mut f64, dst_cap: usize, rows: usize, cols: usize) -> i32;
    pub fn fth_transpose_batched_materialize_f32(src: *const f32, src_len: usize, batch: usize, rows: usize, cols: usize, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_transpose_batched_materialize_f64(src: *const f64, src_len: usize, batch: usize, rows: usize, cols: usize, out: *mut f64, out_cap: usize) -> i32;
    pub fn fth_sdpa_forward_f32(q: *const f32, q_len: usize, k: *const f32, k_len: usize, v: *const f32, v_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f32, causal: i32, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_sdpa_forward_f64(q: *const f64, q_len: usize, k: *const f64, k_len: usize, v: *const f64, v_len: usize, num_bh: usize, seq_q: usize, seq_k: usize, d_k: usize, d_v: usize, scale: f64, causal: i32, out: *mut f64, out_cap: usize) -> i32;
    pub fn fth_index_select_tensor_contiguous_f32(input: *const f32, input_len: usize, meta: *const fth_meta, dim: usize, indices: *const f64, num_indices: usize, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_index_select_tensor_contiguous_f64(input: *const f64, input_len: usize, meta: *const fth_meta, dim: usize, indices: *const f64, num_indices: usize, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_argmax_dim_tensor_contiguous_f32(input: *const f32, input_len: usize, meta: *const fth_meta, dim: usize, out: *mut f32, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_argmax_dim_tensor_contiguous_f64(input: *const f64, input_len: usize, meta: *const fth_meta, dim: usize, out: *mut f64, out_cap: usize, out_len: *mut usize) -> i32;
    pub fn fth_tensor_upload(host: *const f32, rows: i64, cols: i64, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_tensor_alloc(rows: i64, cols: i64, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_tensor_download(t: *const fth_tensor, host: *mut f32, host_cap: usize) -> i32;
    pub fn fth_tensor_shape(t: *const fth_tensor, rows: *mut i64, cols: *mut i64) -> i32;
    pub fn fth_tensor_data(t: *const fth_tensor) -> *mut c_void;
    pub fn fth_tensor_free(t: *mut fth_tensor) -> i32;
    pub fn fth_pool_stats(bytes_in_use: *mut u64, bytes_cached: *mut u64) -> i32;
    pub fn fth_pool_trim() -> i32;
    pub fn fth_batch_new(out: *mut *mut fth_batch) -> i32;
    pub fn fth_batch_free(b: *mut fth_batch) -> i32;
    pub fn fth_batch_finish(b: *mut fth_batch) -> i32;
    pub fn fth_batch_linear(b: *mut fth_batch, a: *const fth_tensor, w: *const fth_tensor, bias: *const fth_tensor, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_matmul(b: *mut fth_batch, a: *const fth_tensor, rhs: *const fth_tensor, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_layernorm(b: *mut fth_batch, x: *const fth_tensor, gamma: *const fth_tensor, beta: *const fth_tensor, eps: f32, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_rmsnorm(b: *mut fth_batch, x: *const fth_tensor, gamma: *const fth_tensor, eps: f32, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_gelu(b: *mut fth_batch, x: *const fth_tensor, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_gelu_tanh(b: *mut fth_batch, x: *const fth_tensor, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_add(b: *mut fth_batch, x: *const fth_tensor, y: *const fth_tensor, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_softmax(b: *mut fth_batch, x: *const fth_tensor, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_batch_mha(b: *mut fth_batch, q: *const fth_tensor, k: *const fth_tensor, v: *const fth_tensor, n_heads: i64, batch: i64, causal: i32, out: *mut *mut fth_tensor) -> i32;
    pub fn fth_encoder_new(d_model: i64, n_heads: i64, d_ff: i64, ln_eps: f32, causal: i32, layers: *const fth_layer_weights, n_layers: i64, out: *mut *mut fth_encoder) -> i32;
    pub fn fth_encoder_free(e: *mut fth_encoder) -> i32;
    pub fn fth_encoder_set_activation(e: *mut fth_encoder, activation: i32) -> i32;
    pub fn fth_encoder_forward(e: *mut fth_encoder, input: *const f32, batch: i64, seq: i64, out: *mut f32, out_cap: usize) -> i32;
    pub fn fth_encoder_forward_dev(e: *mut fth_encoder, x_dev: *const f32, batch: i64, seq: i64, out_dev: *mut f32, s: fth_stream) -> i32;
    pub fn fth_encoder_forward_graph(e: *mut fth_encoder, x_dev: *const f32, batch: i64, seq: i64, out_dev: *mut f32, s: fth_stream) -> i32;
    pub fn fth_safetensors_open(path: *const c_char, out: *mut *mut fth_safetensors) -> i32;
    pub fn fth_safetensors_open_bytes(data: *const c_void, len: usize, out: *mut *mut fth_safetensors) -> i32;
    pub fn fth_safetensors_close(f: *mut fth_safetensors) -> i32;
    pub fn fth_safetensors_count(f: *const fth_safetensors) -> i64;
    pub fn fth_safetensors_name(f: *const fth_safetensors, index: i64) -> *const c_char;
    pub fn fth_safetensors_info(f: *const fth_safetensors, name: *const c_char, info: *mut fth_safetensors_tensor) -> i32;
    pub fn fth_safetensors_read(f: *const fth_safetensors, name: *const c_char, dst: *mut c_void, dst_bytes: usize) -> i32;
    pub fn fth_safetensors_read_f32_dev(f: *const fth_safetensors, name: *const c_char, transpose_2d: i32, dst_dev: *mut f32, dst_elems: usize, s: fth_stream) -> i32;
    pub fn fth_safetensors_read_f64_dev(f: *const fth_safetensors, name: *const c_char, transpose_2d: i32, dst_dev: *mut f64, dst_elems: usize, s: fth_stream) -> i32;
    pub fn fth_safetensors_metadata_count(f: *const fth_safetensors) -> i32;
    pub fn fth_safetensors_metadata(f: *const fth_safetensors, key: *const c_char) -> *const c_char;
    pub fn fth_statedict_open(path: *const c_char, out: *mut *mut fth_statedict) -> i32;
    pub fn fth_statedict_open_bytes(data: *const c_void, len: usize, out: *mut *mut fth_statedict) -> i32;
    pub fn fth_statedict_close(f: *mut fth_statedict) -> i32;
    pub fn fth_statedict_count(f: *const fth_statedict) -> i64;
    pub fn fth_statedict_name(f: *const fth_statedict, index: i64) -> *const c_char;
    pub fn fth_statedict_info(f: *const fth_statedict, name: *const c_char, info: *mut fth_safetensors_tensor) -> i32;
    pub fn fth_statedict_read(f: *const fth_statedict, name: *const c_char, dst: *mut c_void, dst_bytes: usize) -> i32;
    pub fn fth_statedict_read_f32_dev(f: *const fth_statedict, name: *const c_char, transpose_2d: i32, dst_dev: *mut f32, dst_elems: usize, s: fth_stream) -> i32;
    pub fn fth_statedict_read_f64_dev(f: *const fth_statedict, name: *const c_char, transpose_2d: i32, dst_dev: *mut f64, dst_elems: usize, s: fth_stream) -> i32;
    pub fn fth_gpt2_new(vocab: i64, max_pos: i64, d_model: i64, n_heads: i64, d_ff: i64, ln_eps: f32, wte: *const f32, wpe: *const f32, layers: *const fth_layer_weights, n_layers: i64, lnf_w: *const f32, lnf_b: *const f32, out: *mut *mut fth_gpt2) -> i32;
    pub fn fth_gpt2_from_safetensors(f: *const fth_safetensors, n_heads: i64, ln_eps: f32, activation: i32, out: *mut *mut fth_gpt2) -> i32;
    pub fn fth_gpt2_from_statedict(f: *const fth_statedict, n_heads: i64, ln_eps: f32, activation: i32, out: *mut *mut fth_gpt2) -> i32;
    pub fn fth_gpt2_dims(g: *const fth_gpt2, vocab: *mut i64, max_pos: *mut i64, d_model: *mut i64, n_heads: *mut i64, d_ff: *mut i64, n_layers: *mut i64) -> i32;
    pub fn fth_gpt2_free(g: *mut fth_gpt2) -> i32;
    pub fn fth_gpt2_set_activation(g: *mut fth_gpt2, activation: i32) -> i32;
    pub fn fth_gpt2_forward_dev(g: *mut fth_gpt2, ids_dev: *const f64, batch: i64, seq: i64, logits_dev: *mut f32, argmax_dev: *mut f32, s: fth_stream) -> i32;
    pub fn fth_gpt2_hidden_dev(g: *const fth_gpt2) -> *const f32;
    pub fn fth_gpt2_bad_index(g: *const fth_gpt2, position: *mut i64) -> i32;
}
