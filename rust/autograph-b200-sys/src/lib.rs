//! Raw bindings of `libautograph_b200.so` (include/autograph_b200.h), generated by
//! rust/gen_sys.py.  NOT COMPILED where this repository is developed (no Rust toolchain on
//! those machines): it is the crate a maintainer of autograph would add behind a `b200`
//! cargo feature.  Every function returns an ag_status (0 = ok); `check` turns it into the
//! `anyhow::Result` the reference uses everywhere.
#![allow(non_camel_case_types)]
use std::os::raw::{c_char, c_int, c_void};

#[repr(C)] pub struct ag_device { _private: [u8; 0] }
#[repr(C)] pub struct ag_model { _private: [u8; 0] }
#[repr(C)] pub struct ag_comm { _private: [u8; 0] }

pub const AG_F32: c_int = 0;
pub const AG_BF16: c_int = 1;
pub const AG_U8: c_int = 2;
pub const AG_U16: c_int = 3;
pub const AG_U32: c_int = 4;

pub const AG_OK: c_int = 0;
pub const AG_ERR_INVALID: c_int = -1;
pub const AG_ERR_SHAPE: c_int = -2;
pub const AG_ERR_DTYPE: c_int = -3;
pub const AG_ERR_CUDA: c_int = -4;
pub const AG_ERR_OOM: c_int = -5;
pub const AG_ERR_DEVICE_TIMEOUT: c_int = -6;
pub const AG_ERR_UNSUPPORTED: c_int = -7;
pub const AG_ERR_LIMIT: c_int = -8;

#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct ag_conv2_options {
    pub filter: [i32; 2],
    pub padding: [i32; 2],
    pub stride: [i32; 2],
    pub dilation: [i32; 2],
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ag_conv_stage {
    pub w: *const c_void,
    pub bias: *const c_void,
    pub oc: i64,
    pub options: ag_conv2_options,
    pub relu: i32,
    pub pool: [i32; 2],
}

#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct ag_layer_spec {
    pub kind: i32,
    pub a: i32,
    pub b: i32,
    pub c: i32,
    pub d: i32,
    pub bias: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ag_polar_matrix {
    pub g: *const c_void,
    pub o: *mut c_void,
    pub rows: i64,
    pub cols: i64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ag_muon_matrix {
    pub w: *mut c_void,
    pub g: *const c_void,
    pub v: *mut f32,
    pub rows: i64,
    pub cols: i64,
    pub scale: f32,
}

#[link(name = "autograph_b200")]
extern "C" {
    pub fn ag_last_error() -> *const c_char;
    pub fn ag_version() -> *const c_char;
    pub fn ag_kernel_launch_count(count: *mut u64) -> c_int;
    pub fn ag_device_count(count: *mut c_int) -> c_int;
    pub fn ag_device_create(ordinal: c_int, out: *mut *mut ag_device) -> c_int;
    pub fn ag_device_create_on_stream(ordinal: c_int, cuda_stream: *mut c_void, out: *mut *mut ag_device) -> c_int;
    pub fn ag_device_destroy(dev: *mut ag_device) -> c_int;
    pub fn ag_device_wait(dev: *mut ag_device) -> c_int;
    pub fn ag_debug_expiring_wait(dev: *mut ag_device, limit_ns: u64) -> c_int;
    pub fn ag_device_stream(dev: *mut ag_device) -> *mut c_void;
    pub fn ag_device_ordinal(dev: *mut ag_device) -> c_int;
    pub fn ag_alloc(dev: *mut ag_device, bytes: usize, dptr: *mut *mut c_void) -> c_int;
    pub fn ag_free(dev: *mut ag_device, dptr: *mut c_void) -> c_int;
    pub fn ag_host_alloc(bytes: usize, hptr: *mut *mut c_void) -> c_int;
    pub fn ag_host_free(hptr: *mut c_void) -> c_int;
    pub fn ag_upload(dev: *mut ag_device, dptr: *mut c_void, host: *const c_void, bytes: usize) -> c_int;
    pub fn ag_download(dev: *mut ag_device, host: *mut c_void, dptr: *const c_void, bytes: usize) -> c_int;
    pub fn ag_copy(dev: *mut ag_device, dst: *mut c_void, src: *const c_void, bytes: usize) -> c_int;
    pub fn ag_fill_zero(dev: *mut ag_device, dptr: *mut c_void, bytes: usize) -> c_int;
    pub fn ag_gemm(dev: *mut ag_device, dtype: c_int, m: i64, k: i64, n: i64, alpha: f32, a: *const c_void, off_a: i64, rsa: i64, csa: i64, b: *const c_void, off_b: i64, rsb: i64, csb: i64, beta: f32, c: *mut c_void, off_c: i64, rsc: i64, csc: i64) -> c_int;
    pub fn ag_gemm_static_scratch(ordinal: c_int, cuda_stream: *mut c_void, dtype: c_int, m: i64, k: i64, n: i64, alpha: f32, a: *const c_void, off_a: i64, rsa: i64, csa: i64, b: *const c_void, off_b: i64, rsb: i64, csb: i64, beta: f32, c: *mut c_void, off_c: i64, rsc: i64, csc: i64) -> c_int;
    pub fn ag_dense_forward(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, inputs: i64, w: *const c_void, outputs: i64, bias: *const c_void, fuse_relu: c_int, y: *mut c_void) -> c_int;
    pub fn ag_dense_chain_forward(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, n_layers: i32, dims: *const i64, weights: *const *const c_void, biases: *const *const c_void, relu: *const i32, y: *mut c_void) -> c_int;
    pub fn ag_dense_chain_forward_keep(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, n_layers: i32, dims: *const i64, weights: *const *const c_void, biases: *const *const c_void, relu: *const i32, pre_out: *const *mut c_void, act_out: *const *mut c_void) -> c_int;
    pub fn ag_dense_chain_backward(dev: *mut ag_device, dtype: c_int, bs: i64, n_layers: i32, dims: *const i64, layer_in: *const *const c_void, weights: *const *const c_void, gate: *const *const c_void, dy: *const c_void, g: *const *mut c_void, dx: *mut c_void, dw: *const *mut c_void, db: *const *mut c_void) -> c_int;
    pub fn ag_conv2_forward(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, ic: i64, ih: i64, iw: i64, w: *const c_void, oc: i64, bias: *const c_void, opt: *const ag_conv2_options, fuse_relu: c_int, y: *mut c_void) -> c_int;
    pub fn ag_conv2_relu_max_pool2_forward(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, ic: i64, ih: i64, iw: i64, w: *const c_void, oc: i64, bias: *const c_void, opt: *const ag_conv2_options, fuse_relu: c_int, pool_h: i32, pool_w: i32, y: *mut c_void) -> c_int;
    pub fn ag_conv2_relu_max_pool2_forward_keep(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, ic: i64, ih: i64, iw: i64, w: *const c_void, oc: i64, bias: *const c_void, opt: *const ag_conv2_options, pre: *mut c_void, y: *mut c_void) -> c_int;
    pub fn ag_conv_dense_chain_forward(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, ic: i64, ih: i64, iw: i64, n_conv: i32, stages: *const ag_conv_stage, n_dense: i32, dims: *const i64, weights: *const *const c_void, biases: *const *const c_void, relu: *const i32, y: *mut c_void) -> c_int;
    pub fn ag_conv_dense_chain_forward_u8(dev: *mut ag_device, dtype: c_int, x: *const u8, alpha: f32, bs: i64, ic: i64, ih: i64, iw: i64, n_conv: i32, stages: *const ag_conv_stage, n_dense: i32, dims: *const i64, weights: *const *const c_void, biases: *const *const c_void, relu: *const i32, y: *mut c_void) -> c_int;
    pub fn ag_conv2_backward_input(dev: *mut ag_device, dtype: c_int, w: *const c_void, oc: i64, ic: i64, dy: *const c_void, bs: i64, ih: i64, iw: i64, opt: *const ag_conv2_options, dx: *mut c_void) -> c_int;
    pub fn ag_conv2_backward_weight(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, ic: i64, ih: i64, iw: i64, dy: *const c_void, oc: i64, opt: *const ag_conv2_options, beta: f32, dw: *mut c_void) -> c_int;
    pub fn ag_conv2_output_shape(ih: i64, iw: i64, opt: *const ag_conv2_options, oh: *mut i64, ow: *mut i64) -> c_int;
    pub fn ag_im2col_conv2(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, c: i64, ih: i64, iw: i64, opt: *const ag_conv2_options, y: *mut c_void) -> c_int;
    pub fn ag_col2im_conv2(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, c: i64, gh: i64, gw: i64, opt: *const ag_conv2_options, y: *mut c_void) -> c_int;
    pub fn ag_max_pool2(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, c: i64, ih: i64, iw: i64, h: i32, w: i32, sh: i32, sw: i32, y: *mut c_void) -> c_int;
    pub fn ag_max_pool2_backward(dev: *mut ag_device, dtype: c_int, dx: *mut c_void, bs: i64, c: i64, ih: i64, iw: i64, h: i32, w: i32, sh: i32, sw: i32, dy: *const c_void) -> c_int;
    pub fn ag_max_pool2_backward_from_input(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, c: i64, ih: i64, iw: i64, h: i32, w: i32, sh: i32, sw: i32, dy: *const c_void, dx: *mut c_void) -> c_int;
    pub fn ag_relu_max_pool2_forward(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, c: i64, ih: i64, iw: i64, y: *mut c_void) -> c_int;
    pub fn ag_relu_max_pool2_backward(dev: *mut ag_device, dtype: c_int, x: *const c_void, bs: i64, c: i64, ih: i64, iw: i64, dy: *const c_void, dx: *mut c_void) -> c_int;
    pub fn ag_scaled_cast_u8(dev: *mut ag_device, dtype: c_int, alpha: f32, x: *const u8, y: *mut c_void, n: i64) -> c_int;
    pub fn ag_relu(dev: *mut ag_device, dtype: c_int, x: *const c_void, y: *mut c_void, n: i64) -> c_int;
    pub fn ag_relu_backward(dev: *mut ag_device, dtype: c_int, x: *const c_void, dy: *const c_void, dx: *mut c_void, n: i64) -> c_int;
    pub fn ag_scaled_add(dev: *mut ag_device, dtype: c_int, alpha: f32, x: *const c_void, y: *mut c_void, n: i64) -> c_int;
    pub fn ag_bias_add(dev: *mut ag_device, dtype: c_int, y: *mut c_void, bias: *const c_void, rows: i64, cols: i64, inner: i64) -> c_int;
    pub fn ag_bias_grad(dev: *mut ag_device, dtype: c_int, x: *const c_void, rows: i64, cols: i64, inner: i64, beta: f32, y: *mut c_void) -> c_int;
    pub fn ag_layer_norm_forward(dev: *mut ag_device, dtype: c_int, x: *const c_void, weight: *const c_void, bias: *const c_void, rows: i64, cols: i64, eps: f32, y: *mut c_void, mean: *mut f32, rstd: *mut f32) -> c_int;
    pub fn ag_layer_norm_backward(dev: *mut ag_device, dtype: c_int, x: *const c_void, weight: *const c_void, mean: *const f32, rstd: *const f32, dy: *const c_void, rows: i64, cols: i64, dx: *mut c_void, beta: f32, dweight: *mut c_void, dbias: *mut c_void) -> c_int;
    pub fn ag_cross_entropy_loss(dev: *mut ag_device, dtype: c_int, label_dtype: c_int, x: *const c_void, t: *const c_void, bs: i64, classes: i64, loss_host: *mut f32) -> c_int;
    pub fn ag_cross_entropy_loss_device(dev: *mut ag_device, dtype: c_int, label_dtype: c_int, x: *const c_void, t: *const c_void, bs: i64, classes: i64, loss_dev: *mut f32) -> c_int;
    pub fn ag_cross_entropy_loss_device_grad(dev: *mut ag_device, dtype: c_int, label_dtype: c_int, x: *const c_void, t: *const c_void, bs: i64, classes: i64, loss_dev: *mut f32, dy: f32, dx: *mut c_void) -> c_int;
    pub fn ag_cross_entropy_loss_backward(dev: *mut ag_device, dtype: c_int, label_dtype: c_int, x: *const c_void, t: *const c_void, bs: i64, classes: i64, dy: f32, dx: *mut c_void) -> c_int;
    pub fn ag_accuracy(dev: *mut ag_device, dtype: c_int, label_dtype: c_int, x: *const c_void, t: *const c_void, bs: i64, classes: i64, correct_host: *mut u64) -> c_int;
    pub fn ag_sgd_update(dev: *mut ag_device, dtype: c_int, w: *mut c_void, g: *const c_void, n: i64, lr: f32) -> c_int;
    pub fn ag_sgd_update_momentum(dev: *mut ag_device, dtype: c_int, w: *mut c_void, g: *const c_void, v: *mut c_void, n: i64, lr: f32, momentum: f32) -> c_int;
    pub fn ag_newton_schulz(dev: *mut ag_device, dtype: c_int, n: i32, matrices: *const ag_polar_matrix, steps: i32) -> c_int;
    pub fn ag_muon_update(dev: *mut ag_device, dtype: c_int, n: i32, matrices: *const ag_muon_matrix, lr: f32, momentum: f32, nesterov: c_int, weight_decay: f32, steps: i32) -> c_int;
    pub fn ag_model_create(dev: *mut ag_device, dtype: c_int, layers: *const ag_layer_spec, n_layers: i32, seed: u64, out: *mut *mut ag_model) -> c_int;
    pub fn ag_model_create_lenet5(dev: *mut ag_device, dtype: c_int, seed: u64, out: *mut *mut ag_model) -> c_int;
    pub fn ag_model_destroy(model: *mut ag_model) -> c_int;
    pub fn ag_model_parameter_count(model: *mut ag_model, count: *mut i32) -> c_int;
    pub fn ag_model_parameter_len(model: *mut ag_model, index: i32, len: *mut i64) -> c_int;
    pub fn ag_model_set_parameter(model: *mut ag_model, index: i32, host: *const c_void) -> c_int;
    pub fn ag_model_get_parameter(model: *mut ag_model, index: i32, host: *mut c_void) -> c_int;
    pub fn ag_model_get_gradient(model: *mut ag_model, index: i32, host: *mut c_void) -> c_int;
    pub fn ag_model_set_sgd(model: *mut ag_model, momentum: f32) -> c_int;
    pub fn ag_model_get_velocity(model: *mut ag_model, index: i32, host: *mut c_void) -> c_int;
    pub fn ag_model_set_velocity(model: *mut ag_model, index: i32, host: *const c_void) -> c_int;
    pub fn ag_model_set_muon(model: *mut ag_model, momentum: f32, nesterov: c_int, weight_decay: f32, steps: i32, vector_scale: f32) -> c_int;
    pub fn ag_model_get_momentum(model: *mut ag_model, index: i32, host: *mut f32) -> c_int;
    pub fn ag_model_set_momentum(model: *mut ag_model, index: i32, host: *const f32) -> c_int;
    pub fn ag_model_set_grad_scale(model: *mut ag_model, scale: f32) -> c_int;
    pub fn ag_model_infer(model: *mut ag_model, x_host: *const c_void, bs: i64, c: i64, h: i64, w: i64, logits_host: *mut c_void) -> c_int;
    pub fn ag_model_infer_enqueue(model: *mut ag_model, x_host: *const c_void, bs: i64, c: i64, h: i64, w: i64, logits_host: *mut c_void, ticket: *mut i32) -> c_int;
    pub fn ag_model_infer_wait(model: *mut ag_model, ticket: i32) -> c_int;
    pub fn ag_model_infer_u8(model: *mut ag_model, x_host: *const u8, bs: i64, c: i64, h: i64, w: i64, alpha: f32, logits_host: *mut c_void) -> c_int;
    pub fn ag_model_forward_device(model: *mut ag_model, x_dev: *const c_void, bs: i64, c: i64, h: i64, w: i64, logits_dev: *mut c_void) -> c_int;
    pub fn ag_model_train_step(model: *mut ag_model, x_host: *const c_void, t_host: *const u8, bs: i64, c: i64, h: i64, w: i64, lr: f32, loss_host: *mut f32) -> c_int;
    pub fn ag_model_train_forward_backward(model: *mut ag_model, x_dev: *const c_void, t_dev: *const u8, bs: i64, c: i64, h: i64, w: i64, loss_host: *mut f32, grad_bucket: *mut *mut c_void, grad_len: *mut i64) -> c_int;
    pub fn ag_model_apply_update(model: *mut ag_model, lr: f32) -> c_int;
    pub fn ag_model_last_loss(model: *mut ag_model, loss_host: *mut f32) -> c_int;
    pub fn ag_comm_create(devs: *const *mut ag_device, n: c_int, out: *mut *mut ag_comm) -> c_int;
    pub fn ag_comm_unique_id(id_out: *mut c_void, bytes: usize) -> c_int;
    pub fn ag_comm_create_rank(dev: *mut ag_device, world: c_int, rank: c_int, unique_id: *const c_void, id_bytes: usize, out: *mut *mut ag_comm) -> c_int;
    pub fn ag_comm_destroy(comm: *mut ag_comm) -> c_int;
    pub fn ag_comm_world(comm: *mut ag_comm, world: *mut c_int, fused_available: *mut c_int) -> c_int;
    pub fn ag_comm_set_timeout(comm: *mut ag_comm, seconds: f64) -> c_int;
    pub fn ag_allreduce_sum(comm: *mut ag_comm, rank: c_int, dtype: c_int, buf: *mut c_void, n: i64) -> c_int;
    pub fn ag_allreduce_sum_all(comm: *mut ag_comm, dtype: c_int, bufs: *const *mut c_void, n: i64) -> c_int;
    pub fn ag_comm_wait(comm: *mut ag_comm, rank: c_int) -> c_int;
    pub fn ag_model_allreduce_update(model: *mut ag_model, comm: *mut ag_comm, rank: c_int, lr: f32) -> c_int;
}

/// status -> anyhow::Error with the library's message (the reference returns
/// `anyhow::Result` everywhere and `bail!`s on shape and type mismatches).
pub fn check(status: c_int) -> anyhow::Result<()> {
    if status == AG_OK {
        return Ok(());
    }
    let msg = unsafe { std::ffi::CStr::from_ptr(ag_last_error()) }.to_string_lossy().into_owned();
    Err(anyhow::anyhow!("autograph_b200 ({status}): {msg}"))
}
