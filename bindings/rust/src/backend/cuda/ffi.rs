// GENERATED by bindings/rust/gen_ffi.py from include/sage_cuda.h — do not edit by hand.
//
// The raw C ABI of libsagecuda.so.  Safe wrappers live in backend/cuda/mod.rs.
#![allow(non_camel_case_types)]
use std::os::raw::{c_char, c_void};

#[repr(C)] pub struct sage_ctx { _p: [u8; 0] }
#[repr(C)] pub struct sage_buf { _p: [u8; 0] }
#[repr(C)] pub struct sage_module { _p: [u8; 0] }

pub const SAGE_MAX_DIMS: usize = 8;
pub const SAGE_OK: i32 = 0;
pub const SAGE_ERR_INVALID: i32 = 1;
pub const SAGE_ERR_OOM: i32 = 2;
pub const SAGE_ERR_DEVICE: i32 = 3;
pub const SAGE_ERR_COMPILE: i32 = 4;
pub const SAGE_ERR_NO_DEVICE: i32 = 5;
pub const SAGE_ERR_TIMEOUT: i32 = 6;
pub const SAGE_ERR_UNSUPPORTED: i32 = 7;
pub const SAGE_F32: i32 = 0;
pub const SAGE_I32: i32 = 1;
pub const SAGE_U32: i32 = 2;
// storage types of the language-model operators alone
pub const SAGE_F16: i32 = 3;
pub const SAGE_BF16: i32 = 4;
pub const SAGE_I8: i32 = 5;
pub const SAGE_U8: i32 = 6;

/// Tensor = buffer + Shape{extents, strides, offset} in elements (src/tensor.rs:106-110, src/shape.rs:37-43).
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_tensor {
    pub buf: *mut sage_buf, pub dtype: i32, pub ndim: i32,
    pub extents: [i64; SAGE_MAX_DIMS], pub strides: [i64; SAGE_MAX_DIMS], pub offset: i64,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_ctx_opts {
    pub mem_capacity_bytes: u64, pub use_cache: i32, pub ref_compat: i32, pub pattern_fusion: i32, pub gemm_backend: i32,
}
#[repr(C)] #[derive(Clone, Copy, Default)]
pub struct sage_mem_stats_t { pub capacity: u64, pub mem_total: u64, pub mem_used: u64, pub mem_peak: u64, pub num_device_allocs: u64 }
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_arg { pub kind: i32, pub buf: *mut sage_buf, pub i: i64, pub f: f32, pub bytes: *const c_void, pub nbytes: usize }
/// Every pair is ordered [w, h] like SizedExtent<2> (src/ops/conv.rs:83).
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_window { pub ker: [i32; 2], pub stride: [i32; 2], pub pad: [i32; 2], pub dil: [i32; 2] }
/// One tensor of an AdamW step; absent operands have a null `buf`.
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_adamw_tensor {
    pub param: sage_tensor, pub grad: sage_tensor, pub m: sage_tensor, pub v: sage_tensor, pub m_scale: sage_tensor, pub v_scale: sage_tensor, pub copy: sage_tensor,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_adamw_opts { pub lr: f64, pub beta1: f64, pub beta2: f64, pub eps: f64, pub weight_decay: f64, pub grad_scale: f64, pub step: i64 }
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_block_norms_opts {
    pub after_weight: sage_tensor, pub after_bias: sage_tensor, pub before_weight: sage_tensor, pub before_bias: sage_tensor, pub gate: sage_tensor, pub seed: sage_tensor,
    pub after: i32, pub before: i32, pub residual_scale: f32, pub eps: f32, pub p: f32, pub site: u64,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_block_norms_sums { pub after_weight: sage_tensor, pub after_bias: sage_tensor, pub before_weight: sage_tensor, pub before_bias: sage_tensor, pub gate: sage_tensor }

#[link(name = "sagecuda")]
extern "C" {
    pub fn sage_device_count(count: *mut i32) -> i32;
    pub fn sage_device_name(index: i32, name: *mut c_char, name_len: usize) -> i32;
    pub fn sage_ctx_opts_default(opts: *mut sage_ctx_opts);
    pub fn sage_ctx_create(device: i32, opts: *const sage_ctx_opts, ctx: *mut *mut sage_ctx) -> i32;
    pub fn sage_ctx_destroy(ctx: *mut sage_ctx) -> i32;
    pub fn sage_sync(ctx: *mut sage_ctx) -> i32;
    pub fn sage_last_error(ctx: *mut sage_ctx) -> *const c_char;
    pub fn sage_status_word(ctx: *mut sage_ctx, word: *mut u32) -> i32;
    pub fn sage_selftest_bounded_wait(ctx: *mut sage_ctx) -> i32;
    pub fn sage_ctx_stream(ctx: *mut sage_ctx) -> *mut c_void;
    pub fn sage_ctx_use_stream(ctx: *mut sage_ctx, stream: *mut c_void) -> i32;
    pub fn sage_ctx_use_own_stream(ctx: *mut sage_ctx) -> i32;
    pub fn sage_alloc(ctx: *mut sage_ctx, bytes: usize, buf: *mut *mut sage_buf) -> i32;
    pub fn sage_free(ctx: *mut sage_ctx, buf: *mut sage_buf) -> i32;
    pub fn sage_buf_wrap(ctx: *mut sage_ctx, device_ptr: *mut c_void, bytes: usize, buf: *mut *mut sage_buf) -> i32;
    pub fn sage_last_oom(ctx: *mut sage_ctx, needed_bytes: *mut u64, total_bytes: *mut u64) -> i32;
    pub fn sage_mem_stats(ctx: *mut sage_ctx, stats: *mut sage_mem_stats_t) -> i32;
    pub fn sage_release_cached(ctx: *mut sage_ctx) -> i32;
    pub fn sage_garbage_collect(ctx: *mut sage_ctx, reclaimed: *mut u64, runs_total: *mut u64, reclaimed_total: *mut u64) -> i32;
    pub fn sage_upload(ctx: *mut sage_ctx, dst: *mut sage_buf, dst_offset: usize, src: *const c_void, bytes: usize) -> i32;
    pub fn sage_download(ctx: *mut sage_ctx, src: *const sage_buf, src_offset: usize, dst: *mut c_void, bytes: usize) -> i32;
    pub fn sage_upload_async(ctx: *mut sage_ctx, dst: *mut sage_buf, dst_offset: usize, src: *const c_void, bytes: usize) -> i32;
    pub fn sage_memset(ctx: *mut sage_ctx, buf: *mut sage_buf, offset: usize, byte_value: i32, bytes: usize) -> i32;
    pub fn sage_buf_ptr(buf: *const sage_buf) -> *mut c_void;
    pub fn sage_buf_size(buf: *const sage_buf) -> usize;
    pub fn sage_host_alloc(bytes: usize, ptr: *mut *mut c_void) -> i32;
    pub fn sage_host_free(ptr: *mut c_void) -> i32;
    pub fn sage_module_get(ctx: *mut sage_ctx, cuda_src: *const c_char, module: *mut *mut sage_module) -> i32;
    pub fn sage_launch(ctx: *mut sage_ctx, module: *mut sage_module, kernel_name: *const c_char, grid: *const u32, block: *const u32, smem_bytes: u32, args: *const sage_arg, nargs: i32) -> i32;
    pub fn sage_map(ctx: *mut sage_ctx, expr: *const c_char, x: *const sage_tensor, nx: i32, y: *const sage_tensor) -> i32;
    pub fn sage_reduce(ctx: *mut sage_ctx, kind: i32, x: *const sage_tensor, axes: *const i32, naxes: i32, y: *const sage_tensor) -> i32;
    pub fn sage_reduce_arg(ctx: *mut sage_ctx, is_max: i32, x: *const sage_tensor, axis: i32, y: *const sage_tensor) -> i32;
    pub fn sage_softmax(ctx: *mut sage_ctx, x: *const sage_tensor, rows: i64, inner: i64, y: *const sage_tensor) -> i32;
    pub fn sage_log_sum_exp(ctx: *mut sage_ctx, x: *const sage_tensor, rows: i64, inner: i64, y: *const sage_tensor) -> i32;
    pub fn sage_layer_norm(ctx: *mut sage_ctx, x: *const sage_tensor, rows: i64, inner: i64, gamma: *const sage_tensor, beta: *const sage_tensor, eps: f32, y: *const sage_tensor) -> i32;
    pub fn sage_gather(ctx: *mut sage_ctx, x: *const sage_tensor, ind: *const sage_tensor, axis: i32, y: *const sage_tensor) -> i32;
    pub fn sage_scatter(ctx: *mut sage_ctx, x: *const sage_tensor, ind: *const sage_tensor, axis: i32, y: *const sage_tensor) -> i32;
    pub fn sage_unslice(ctx: *mut sage_ctx, x: *const sage_tensor, axis: i32, start: i64, y: *const sage_tensor) -> i32;
    pub fn sage_concat(ctx: *mut sage_ctx, xs: *const sage_tensor, nx: i32, axis: i32, y: *const sage_tensor) -> i32;
    pub fn sage_gemm(ctx: *mut sage_ctx, trans_a: i32, trans_b: i32, m: i64, n: i64, k: i64, a: *const sage_buf, a_off: i64, lda: i64, b: *const sage_buf, b_off: i64, ldb: i64, c: *mut sage_buf, c_off: i64, ldc: i64) -> i32;
    pub fn sage_gemm_strided_batched(ctx: *mut sage_ctx, trans_a: i32, trans_b: i32, m: i64, n: i64, k: i64, a: *const sage_buf, a_off: i64, lda: i64, stride_a: i64, b: *const sage_buf, b_off: i64, ldb: i64, stride_b: i64, c: *mut sage_buf, c_off: i64, ldc: i64, stride_c: i64, batch: i64) -> i32;
    pub fn sage_gemm_noalloc(ctx: *mut sage_ctx, trans_a: i32, trans_b: i32, m: i64, n: i64, k: i64, a: *const sage_buf, a_off: i64, lda: i64, b: *const sage_buf, b_off: i64, ldb: i64, c: *mut sage_buf, c_off: i64, ldc: i64) -> i32;
    pub fn sage_im2col(ctx: *mut sage_ctx, x: *const sage_tensor, w: *const sage_window, y: *const sage_tensor) -> i32;
    pub fn sage_col2im(ctx: *mut sage_ctx, x: *const sage_tensor, w: *const sage_window, y: *const sage_tensor) -> i32;
    pub fn sage_pool2d(ctx: *mut sage_ctx, is_max: i32, x: *const sage_tensor, w: *const sage_window, y: *const sage_tensor) -> i32;
    pub fn sage_conv2d_nhwc(ctx: *mut sage_ctx, x: *const sage_tensor, filter: *const sage_tensor, w: *const sage_window, y: *const sage_tensor) -> i32;
    pub fn sage_embedding(ctx: *mut sage_ctx, table: *const sage_tensor, ids: *const sage_tensor, scale: f32, y: *const sage_tensor) -> i32;
    pub fn sage_embedding_grad(ctx: *mut sage_ctx, g: *const sage_tensor, ids: *const sage_tensor, scale: f32, add: i32, dtable: *const sage_tensor) -> i32;
    pub fn sage_token_log_probs(ctx: *mut sage_ctx, logits: *const sage_tensor, ids: *const sage_tensor, scale: f32, log_probs: *const sage_tensor, entropy: *const sage_tensor, stats: *const sage_tensor, top_ids: *const sage_tensor, top_log_probs: *const sage_tensor) -> i32;
    pub fn sage_token_log_probs_grad(ctx: *mut sage_ctx, logits: *const sage_tensor, ids: *const sage_tensor, scale: f32, stats: *const sage_tensor, entropy: *const sage_tensor, g_log_probs: *const sage_tensor, g_entropy: *const sage_tensor, dlogits: *const sage_tensor) -> i32;
    pub fn sage_token_log_probs_and_grad(ctx: *mut sage_ctx, logits: *const sage_tensor, ids: *const sage_tensor, scale: f32, g_log_probs: *const sage_tensor, g_entropy: *const sage_tensor, log_probs: *const sage_tensor, entropy: *const sage_tensor, dlogits: *const sage_tensor) -> i32;
    pub fn sage_head_log_probs(ctx: *mut sage_ctx, hidden: *const sage_tensor, weight: *const sage_tensor, ids: *const sage_tensor, scale: f32, log_probs: *const sage_tensor, entropy: *const sage_tensor, stats: *const sage_tensor) -> i32;
    pub fn sage_head_log_probs_grad(ctx: *mut sage_ctx, hidden: *const sage_tensor, weight: *const sage_tensor, ids: *const sage_tensor, scale: f32, stats: *const sage_tensor, entropy: *const sage_tensor, g_log_probs: *const sage_tensor, g_entropy: *const sage_tensor, dhidden: *const sage_tensor, dweight: *const sage_tensor) -> i32;
    pub fn sage_dropout(ctx: *mut sage_ctx, x: *const sage_tensor, y: *const sage_tensor, seed: *const sage_tensor, p: f32, site: u64) -> i32;
    pub fn sage_block_norms(ctx: *mut sage_ctx, opts: *const sage_block_norms_opts, x: *const sage_tensor, y: *const sage_tensor, out: *const sage_tensor, h: *const sage_tensor, stats: *const sage_tensor) -> i32;
    pub fn sage_block_norms_grad(ctx: *mut sage_ctx, opts: *const sage_block_norms_opts, out: *const sage_tensor, y: *const sage_tensor, stats: *const sage_tensor, g_out: *const sage_tensor, g_h: *const sage_tensor, dx: *const sage_tensor, dy: *const sage_tensor, sums: *const sage_block_norms_sums) -> i32;
    pub fn sage_adamw_step(ctx: *mut sage_ctx, tensors: *const sage_adamw_tensor, count: i32, opts: *const sage_adamw_opts) -> i32;
    pub fn sage_adamw_states(ctx: *mut sage_ctx, m: *const sage_tensor, m_scale: *const sage_tensor, v: *const sage_tensor, v_scale: *const sage_tensor, m_out: *const sage_tensor, v_out: *const sage_tensor) -> i32;
    pub fn sage_ipc_export(ctx: *mut sage_ctx, buf: *mut sage_buf, handle: *mut u8, offset: *mut u64) -> i32;
    pub fn sage_ipc_open(ctx: *mut sage_ctx, handle: *const u8, peer_ptr: *mut *mut c_void) -> i32;
    pub fn sage_ipc_close(ctx: *mut sage_ctx, peer_ptr: *mut c_void) -> i32;
    pub fn sage_peer_write(ctx: *mut sage_ctx, peer_ptr: *mut c_void, peer_offset: usize, src: *const sage_buf, src_offset: usize, bytes: usize) -> i32;
    pub fn sage_peer_write_ptr(ctx: *mut sage_ctx, peer_ptr: *mut c_void, peer_offset: usize, src_dev: *const c_void, bytes: usize) -> i32;
    pub fn sage_launch_count(ctx: *mut sage_ctx, kernels: *mut u64, memsets: *mut u64) -> i32;
    pub fn sage_trace_begin(ctx: *mut sage_ctx) -> i32;
    pub fn sage_trace_get(ctx: *mut sage_ctx, out: *mut c_char, out_len: usize, needed: *mut usize) -> i32;
    pub fn sage_timer_start(ctx: *mut sage_ctx) -> i32;
    pub fn sage_timer_stop(ctx: *mut sage_ctx, milliseconds: *mut f32) -> i32;
    pub fn sage_profile_begin(ctx: *mut sage_ctx) -> i32;
    pub fn sage_profile_end(ctx: *mut sage_ctx, out: *mut c_char, out_len: usize, needed: *mut usize) -> i32;
}
