// Raw bindings of libullm_cuda.so.  GENERATED by gen_ffi.py from include/*.h - do not edit by hand.
#![allow(non_camel_case_types, non_upper_case_globals, dead_code)]

use std::os::raw::{c_char, c_int, c_uint, c_void};

#[repr(C)]
pub struct ullm_cuda_ctx {
    _private: [u8; 0],
}
#[repr(C)]
pub struct ullm_cuda_buf {
    _private: [u8; 0],
}
#[repr(C)]
pub struct ullm_cuda_fwd {
    _private: [u8; 0],
}
#[repr(C)]
pub struct ullm_cuda_experts {
    _private: [u8; 0],
}
#[repr(C)]
pub struct ullm_cuda_weight {
    _private: [u8; 0],
}
#[repr(C)]
pub struct ullm_cuda_shard {
    _private: [u8; 0],
}
#[repr(C)]
pub struct ullm_st {
    _private: [u8; 0],
}
#[repr(C)]
pub struct ullm_gguf {
    _private: [u8; 0],
}

pub const ULLM_SHARD_HANDLE_BYTES: usize = 64;
pub const ULLM_SHARD_MAX_RANKS: usize = 8;
pub const ULLM_SHARD_NCCL_ID_BYTES: usize = 128;
pub const ULLM_CUDA_MOE_NOALLOC_SCRATCH_BYTES: usize = 4194304;
pub const ULLM_FORWARD_VERIFY_MAX: c_int = 64;
pub const ULLM_OK: c_int = 0;
pub const ULLM_ERR_UNSUPPORTED: c_int = 1;
pub const ULLM_ERR_FORMAT: c_int = 2;
pub const ULLM_ERR_CUDA: c_int = 3;
pub const ULLM_ERR_TIMEOUT: c_int = 4;
pub const ULLM_ERR_OOM: c_int = 5;
pub const ULLM_ERR_INVALID: c_int = 6;
pub const ULLM_DTYPE_F32: c_int = 0;
pub const ULLM_DTYPE_F16: c_int = 1;
pub const ULLM_DTYPE_Q4_K: c_int = 12;
pub const ULLM_DTYPE_Q6_K: c_int = 14;
pub const ULLM_DTYPE_BF16: c_int = 30;
pub const ULLM_DTYPE_MLX_U32: c_int = 1000;
pub const ULLM_OPT_PDL: c_int = 1;
pub const ULLM_OPT_SHARD_TIMEOUT_MS: c_int = 2;
pub const ULLM_EPI_STORE: c_int = 0;
pub const ULLM_EPI_RESIDUAL: c_int = 1;
pub const ULLM_EPI_SWIGLU: c_int = 2;
pub const ULLM_SHARD_NO_WAIT: c_int = 1;
pub const ULLM_SHARD_FUSED_STORES: c_int = 2;
pub const ULLM_SHARD_SM_PUSH: c_int = 4;
pub const ULLM_KV_FAULT_NO_PAGES: c_int = 1;
pub const ULLM_KV_FAULT_SEQ: c_int = 2;
pub const ULLM_KV_FAULT_LEN: c_int = 4;
pub const ULLM_KV_FAULT_PAGE: c_int = 8;
pub const ULLM_KV_FAULT_PATH: c_int = 16;
pub const ULLM_KV_FAULT_SHARED: c_int = 32;
pub const ULLM_KV_FAULT_POS: c_int = 64;
pub const ULLM_GGUF_OK: c_int = 0;
pub const ULLM_GGUF_ERR_UNSUPPORTED: c_int = 1;
pub const ULLM_GGUF_ERR_FORMAT: c_int = 2;
pub const ULLM_GGUF_ERR_IO: c_int = 6;
pub const ULLM_GGUF_ERR_INVALID: c_int = 7;
pub const ULLM_GGUF_ERR_MISSING: c_int = 8;
pub const ULLM_ST_OK: c_int = 0;
pub const ULLM_ST_ERR_UNSUPPORTED: c_int = 1;
pub const ULLM_ST_ERR_FORMAT: c_int = 2;
pub const ULLM_ST_ERR_IO: c_int = 6;
pub const ULLM_ST_ERR_INVALID: c_int = 7;
pub const ULLM_ST_ERR_MISSING: c_int = 8;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_chain_op {
    pub w: *const ullm_cuda_weight,
    pub d_x: *const f32,
    pub d_y: *mut f32,
    pub d_norm_w: *const f32,
    pub eps: f32,
    pub epi: c_int,
    pub d_res: *const f32,
    pub dep: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_shard_op {
    pub w: *const ullm_cuda_weight,
    pub d_x: *const f32,
    pub y_offset: usize,
    pub row0: usize,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_moe_experts_input {
    pub gate_w: *const c_void,
    pub gate_scales: *const c_void,
    pub gate_biases: *const c_void,
    pub up_w: *const c_void,
    pub up_scales: *const c_void,
    pub up_biases: *const c_void,
    pub down_w: *const c_void,
    pub down_scales: *const c_void,
    pub down_biases: *const c_void,
    pub table_dtype: c_int,
    pub n_experts: usize,
    pub hidden: usize,
    pub inter: usize,
    pub group: usize,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_pages {
    pub dtype: c_int,
    pub n_layer: usize,
    pub n_pages: usize,
    pub page_size: usize,
    pub n_kv_head: usize,
    pub head_dim: usize,
    pub d_k: *mut c_void,
    pub d_v: *mut c_void,
    pub layer_stride: usize,
    pub page_stride: usize,
    pub slot_stride: usize,
    pub head_stride: usize,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_table {
    pub d_blocks: *mut i32,
    pub d_len: *mut i32,
    pub d_refs: *mut i32,
    pub d_fault: *mut i32,
    pub n_seq: usize,
    pub max_blocks: usize,
    pub d_work: *mut c_void,
    pub work_bytes: usize,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_qk_norm_rope {
    pub kv: *const ullm_kv_pages,
    pub layer: usize,
    pub x_dtype: c_int,
    pub q_dtype: c_int,
    pub n_rows: usize,
    pub n_head: usize,
    pub d_q: *const c_void,
    pub d_k: *const c_void,
    pub d_v: *const c_void,
    pub q_stride: usize,
    pub k_stride: usize,
    pub v_stride: usize,
    pub d_q_out: *mut c_void,
    pub q_out_stride: usize,
    pub d_q_norm: *const f32,
    pub d_k_norm: *const f32,
    pub d_q_bias: *const f32,
    pub d_k_bias: *const f32,
    pub d_v_bias: *const f32,
    pub eps: f32,
    pub d_rope: *const f32,
    pub n_pos: usize,
    pub rot_dim: usize,
    pub neox: c_int,
    pub d_row_seq: *const i32,
    pub d_row_slot: *const i32,
    pub d_row_pos: *const i32,
    pub d_blocks: *const i32,
    pub n_table: usize,
    pub max_blocks: usize,
    pub d_fault: *mut i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_tree_attn {
    pub kv: *const ullm_kv_pages,
    pub layer: usize,
    pub dtype: c_int,
    pub n_rows: usize,
    pub n_seq: usize,
    pub n_head: usize,
    pub d_q: *const c_void,
    pub q_stride: usize,
    pub d_out: *mut c_void,
    pub out_stride: usize,
    pub d_cu: *const i32,
    pub d_len: *const i32,
    pub d_ids: *const i32,
    pub d_blocks: *const i32,
    pub n_table: usize,
    pub max_blocks: usize,
    pub d_mask: *const u32,
    pub mask_words: usize,
    pub scale: f32,
    pub d_work: *mut c_void,
    pub work_bytes: usize,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_gpu_params {
    pub n_embd: usize,
    pub n_layer: usize,
    pub n_head: usize,
    pub n_kv_head: usize,
    pub head_dim: usize,
    pub n_ff: usize,
    pub n_ctx: usize,
    pub vocab: usize,
    pub rope_theta: f32,
    pub eps: f32,
    pub rope_neox: c_int,
    pub qk_norm: c_int,
    pub sandwich_norm: c_int,
    pub geglu: c_int,
    pub n_experts: usize,
    pub n_experts_used: usize,
    pub moe_inter: usize,
    pub sliding_window: usize,
    pub kv_f16: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_gpu_weight {
    pub dtype: c_int,
    pub bytes: *const c_void,
    pub len: usize,
    pub out: usize,
    pub cols: usize,
    pub mlx_scales: *const f32,
    pub mlx_biases: *const f32,
    pub mlx_group: usize,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_gpu_layer_input {
    pub attn_norm: *const f32,
    pub ffn_norm: *const f32,
    pub wq: ullm_gpu_weight,
    pub wk: ullm_gpu_weight,
    pub wv: ullm_gpu_weight,
    pub wo: ullm_gpu_weight,
    pub w_gate: ullm_gpu_weight,
    pub w_up: ullm_gpu_weight,
    pub w_down: ullm_gpu_weight,
    pub q_bias: *const f32,
    pub k_bias: *const f32,
    pub v_bias: *const f32,
    pub q_norm: *const f32,
    pub k_norm: *const f32,
    pub moe_gate: ullm_gpu_weight,
    pub experts: *const ullm_moe_experts_input,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_gpu_model_input {
    pub params: ullm_gpu_params,
    pub output: ullm_gpu_weight,
    pub final_norm: *const f32,
    pub layers: *const ullm_gpu_layer_input,
    pub mlx_table_dtype: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_debug_stat {
    pub label: [c_char; 16],
    pub nan: u64,
    pub inf: u64,
    pub maxabs: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_gguf_tensor {
    pub name: *const c_char,
    pub dtype: c_int,
    pub n_dims: u32,
    pub shape: [u64; 8],
    pub offset: u64,
    pub nbytes: u64,
    pub data: *const c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_gguf_llama_params {
    pub n_embd: u64,
    pub n_layer: u64,
    pub n_head: u64,
    pub n_kv_head: u64,
    pub head_dim: u64,
    pub n_ff: u64,
    pub n_ctx: u64,
    pub vocab: u64,
    pub rope_theta: f32,
    pub eps: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_st_tensor {
    pub name: *const c_char,
    pub dtype: c_int,
    pub n_dims: u32,
    pub shape: [u64; 8],
    pub shard: u32,
    pub offset: u64,
    pub nbytes: u64,
    pub data: *const c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_st_mlx_weight {
    pub weight: *const u32,
    pub scales: *const u16,
    pub biases: *const u16,
    pub out: u64,
    pub r#in: u64,
    pub group: u64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_st_mlx_params {
    pub n_embd: u64,
    pub n_layer: u64,
    pub n_head: u64,
    pub n_kv_head: u64,
    pub head_dim: u64,
    pub n_experts: u64,
    pub n_experts_used: u64,
    pub moe_inter: u64,
    pub n_ctx: u64,
    pub vocab: u64,
    pub group: u64,
    pub rope_theta: f32,
    pub eps: f32,
}

#[link(name = "ullm_cuda")]
extern "C" {
    pub fn ullm_cuda_ctx_create(device: c_int, out: *mut *mut ullm_cuda_ctx) -> c_int;
    pub fn ullm_cuda_ctx_destroy(ctx: *mut ullm_cuda_ctx);
    pub fn ullm_cuda_last_error(ctx: *const ullm_cuda_ctx) -> *const c_char;
    pub fn ullm_cuda_ctx_set_option(ctx: *mut ullm_cuda_ctx, option: c_int, value: c_int) -> c_int;
    pub fn ullm_cuda_device_name(ctx: *const ullm_cuda_ctx, name: *mut c_char, cap: usize) -> c_int;
    pub fn ullm_cuda_sm_count(ctx: *const ullm_cuda_ctx) -> c_int;
    pub fn ullm_cuda_synchronize(ctx: *mut ullm_cuda_ctx) -> c_int;
    pub fn ullm_cuda_upload(ctx: *mut ullm_cuda_ctx, bytes: *const c_void, len: usize, out: *mut *mut ullm_cuda_buf) -> c_int;
    pub fn ullm_cuda_alloc(ctx: *mut ullm_cuda_ctx, len: usize, out: *mut *mut ullm_cuda_buf) -> c_int;
    pub fn ullm_cuda_download(ctx: *mut ullm_cuda_ctx, buf: *const ullm_cuda_buf, offset: usize, host: *mut c_void, len: usize) -> c_int;
    pub fn ullm_cuda_buf_ptr(buf: *const ullm_cuda_buf) -> *mut c_void;
    pub fn ullm_cuda_buf_len(buf: *const ullm_cuda_buf) -> usize;
    pub fn ullm_cuda_buf_free(ctx: *mut ullm_cuda_ctx, buf: *mut ullm_cuda_buf);
    pub fn ullm_cuda_dequantize(ctx: *mut ullm_cuda_ctx, dtype: c_int, data: *const c_void, data_len: usize, out: *mut f32, n: usize) -> c_int;
    pub fn ullm_cuda_dequantize_mlx4(ctx: *mut ullm_cuda_ctx, weight: *const u32, scales: *const f32, biases: *const f32, out_dim: usize, in_dim: usize, group: usize, y: *mut f32) -> c_int;
    pub fn ullm_cuda_matvec_quant(ctx: *mut ullm_cuda_ctx, dtype: c_int, w_bytes: *const c_void, w_len: usize, x: *const f32, y: *mut f32, out_dim: usize, in_dim: usize) -> c_int;
    pub fn ullm_cuda_matvec_resident(ctx: *mut ullm_cuda_ctx, dtype: c_int, w: *const ullm_cuda_buf, x: *const f32, y: *mut f32, out_dim: usize, in_dim: usize) -> c_int;
    pub fn ullm_cuda_matvec_mlx4(ctx: *mut ullm_cuda_ctx, w: *const c_void, scales: *const f32, biases: *const f32, x: *const f32, y: *mut f32, out_dim: usize, in_dim: usize, group: usize) -> c_int;
    pub fn ullm_cuda_matvec_dev(ctx: *mut ullm_cuda_ctx, dtype: c_int, d_w: *const c_void, d_scales: *const c_void, d_biases: *const c_void, table_dtype: c_int, group: usize, d_x: *const f32, d_y: *mut f32, out_dim: usize, in_dim: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_weight_create(ctx: *mut ullm_cuda_ctx, w: *const ullm_gpu_weight, mlx_table_dtype: c_int, out: *mut *mut ullm_cuda_weight) -> c_int;
    pub fn ullm_cuda_weight_destroy(ctx: *mut ullm_cuda_ctx, w: *mut ullm_cuda_weight);
    pub fn ullm_cuda_weight_matvec(ctx: *mut ullm_cuda_ctx, w: *const ullm_cuda_weight, x: *const f32, y: *mut f32) -> c_int;
    pub fn ullm_cuda_weight_matvec_dev(ctx: *mut ullm_cuda_ctx, w: *const ullm_cuda_weight, d_x: *const f32, d_y: *mut f32, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_weight_matvec_batch_dev(ctx: *mut ullm_cuda_ctx, n: usize, w: *const *const ullm_cuda_weight, d_x: *const *const f32, d_y: *const *mut f32, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_weight_matvec_batch(ctx: *mut ullm_cuda_ctx, n: usize, w: *const *const ullm_cuda_weight, x: *const *const f32, y: *const *mut f32) -> c_int;
    pub fn ullm_cuda_weight_matvec_chain_dev(ctx: *mut ullm_cuda_ctx, n: usize, ops: *const ullm_chain_op, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_weight_matmul(ctx: *mut ullm_cuda_ctx, w: *const ullm_cuda_weight, x: *const f32, y: *mut f32, s: usize) -> c_int;
    pub fn ullm_cuda_weight_matmul_dev(ctx: *mut ullm_cuda_ctx, w: *const ullm_cuda_weight, d_x: *const f32, d_y: *mut f32, s: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_weight_export(ctx: *mut ullm_cuda_ctx, w: *const ullm_cuda_weight, bytes: *mut c_void, len: usize) -> c_int;
    pub fn ullm_cuda_weight_bytes(w: *const ullm_cuda_weight) -> usize;
    pub fn ullm_cuda_weight_create_st(ctx: *mut ullm_cuda_ctx, st: *const ullm_st, name: *const c_char, group: usize, out: *mut *mut ullm_cuda_weight) -> c_int;
    pub fn ullm_cuda_matmul_quant(ctx: *mut ullm_cuda_ctx, dtype: c_int, w_bytes: *const c_void, w_len: usize, x: *const f32, y: *mut f32, out_dim: usize, in_dim: usize, s: usize) -> c_int;
    pub fn ullm_cuda_matmul_mlx4(ctx: *mut ullm_cuda_ctx, w: *const c_void, scales: *const f32, biases: *const f32, x: *const f32, y: *mut f32, out_dim: usize, in_dim: usize, group: usize, s: usize) -> c_int;
    pub fn ullm_cuda_matmul_dev(ctx: *mut ullm_cuda_ctx, dtype: c_int, d_w: *const c_void, d_scales: *const c_void, d_biases: *const c_void, table_dtype: c_int, group: usize, d_x: *const f32, d_y: *mut f32, out_dim: usize, in_dim: usize, s: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_shard_create(ctx: *mut ullm_cuda_ctx, world: c_int, rank: c_int, y_floats: usize, out: *mut *mut ullm_cuda_shard) -> c_int;
    pub fn ullm_cuda_shard_destroy(s: *mut ullm_cuda_shard);
    pub fn ullm_cuda_shard_export(s: *const ullm_cuda_shard, handle: *mut c_void) -> c_int;
    pub fn ullm_cuda_shard_connect(s: *mut ullm_cuda_shard, handles: *const c_void) -> c_int;
    pub fn ullm_cuda_shard_connect_local(shards: *const *mut ullm_cuda_shard, world: c_int) -> c_int;
    pub fn ullm_cuda_shard_reset(s: *mut ullm_cuda_shard) -> c_int;
    pub fn ullm_cuda_shard_y(s: *const ullm_cuda_shard) -> *mut f32;
    pub fn ullm_cuda_shard_read(s: *mut ullm_cuda_shard, offset: usize, host: *mut f32, n: usize) -> c_int;
    pub fn ullm_cuda_shard_row_range(out: usize, world: c_int, rank: c_int, row0: *mut usize, rows: *mut usize) -> c_int;
    pub fn ullm_cuda_shard_weight_create(s: *mut ullm_cuda_shard, full: *const ullm_gpu_weight, mlx_table_dtype: c_int, out: *mut *mut ullm_cuda_weight) -> c_int;
    pub fn ullm_cuda_shard_matvec_dev(s: *mut ullm_cuda_shard, n: usize, ops: *const ullm_shard_op, flags: c_int, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_shard_matvec(s: *mut ullm_cuda_shard, n: usize, ops: *const ullm_shard_op, x_host: *const *const f32, y_host: *mut f32, y_offset: usize, y_count: usize) -> c_int;
    pub fn ullm_cuda_shard_wait_dev(s: *mut ullm_cuda_shard, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_shard_matmul_dev(s: *mut ullm_cuda_shard, w: *const ullm_cuda_weight, d_x: *const f32, tokens: usize, y_offset: usize, row0: usize, out_total: usize, flags: c_int, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_shard_nccl_id(id: *mut c_void) -> c_int;
    pub fn ullm_cuda_shard_nccl_init(s: *mut ullm_cuda_shard, id: *const c_void) -> c_int;
    pub fn ullm_cuda_shard_allgather_nccl_dev(s: *mut ullm_cuda_shard, d_send: *const f32, d_recv: *mut f32, count: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_shard_nccl_check(s: *mut ullm_cuda_shard) -> c_int;
    pub fn ullm_cuda_experts_create(ctx: *mut ullm_cuda_ctx, r#in: *const ullm_moe_experts_input, out: *mut *mut ullm_cuda_experts) -> c_int;
    pub fn ullm_cuda_experts_create_st(ctx: *mut ullm_cuda_ctx, st: *const ullm_st, prefix: *const c_char, n_experts: usize, hidden: usize, inter: usize, group: usize, out: *mut *mut ullm_cuda_experts) -> c_int;
    pub fn ullm_cuda_experts_destroy(ctx: *mut ullm_cuda_ctx, e: *mut ullm_cuda_experts);
    pub fn ullm_cuda_moe_ffn(ctx: *mut ullm_cuda_ctx, e: *const ullm_cuda_experts, x: *const f32, logits: *const f32, n_tok: usize, k: usize, y: *mut f32, idx: *mut u32, wts: *mut f32) -> c_int;
    pub fn ullm_cuda_moe_ffn_dev(ctx: *mut ullm_cuda_ctx, e: *const ullm_cuda_experts, d_x: *const f32, d_logits: *const f32, n_tok: usize, k: usize, d_y: *mut f32, d_idx: *mut u32, d_wts: *mut f32, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_moe_ffn_noalloc(device: c_int, dev_experts: *const ullm_moe_experts_input, d_x: *const f32, d_logits: *const f32, n_tok: usize, k: usize, d_y: *mut f32, stream: *mut c_void, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_cuda_kv_work_bytes(n_pages: usize, n_seq: usize) -> usize;
    pub fn ullm_cuda_kv_fork_dev(ctx: *mut ullm_cuda_ctx, kv: *const ullm_kv_pages, t: *const ullm_kv_table, d_src: *const i32, d_dst: *const i32, n: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_kv_grow_dev(ctx: *mut ullm_cuda_ctx, kv: *const ullm_kv_pages, t: *const ullm_kv_table, d_seq: *const i32, d_add: *const i32, n: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_kv_accept_dev(ctx: *mut ullm_cuda_ctx, kv: *const ullm_kv_pages, t: *const ullm_kv_table, d_seq: *const i32, d_draft: *const i32, d_path: *const i32, d_kept: *const i32, n: usize, max_path: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_kv_trim_dev(ctx: *mut ullm_cuda_ctx, kv: *const ullm_kv_pages, t: *const ullm_kv_table, d_seq: *const i32, d_new_len: *const i32, n: usize, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_kv_copy_pages_dev(ctx: *mut ullm_cuda_ctx, kv: *const ullm_kv_pages, d_src: *const i32, d_dst: *const i32, n: usize, d_fault: *mut i32, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_tree_plan_dev(ctx: *mut ullm_cuda_ctx, n_rows: usize, n_seq: usize, d_cu: *const i32, d_len: *const i32, d_ids: *const i32, n_table: usize, d_parent: *const i32, d_row_seq: *mut i32, d_row_slot: *mut i32, d_row_pos: *mut i32, d_mask: *mut u32, mask_words: usize, d_fault: *mut i32, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_qk_norm_rope_dev(ctx: *mut ullm_cuda_ctx, a: *const ullm_qk_norm_rope, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_tree_attn_work_bytes(ctx: *const ullm_cuda_ctx, kv: *const ullm_kv_pages, dtype: c_int) -> usize;
    pub fn ullm_cuda_tree_attn_dev(ctx: *mut ullm_cuda_ctx, a: *const ullm_tree_attn, stream: *mut c_void) -> c_int;
    pub fn ullm_cuda_forward_create(ctx: *mut ullm_cuda_ctx, r#in: *const ullm_gpu_model_input, out: *mut *mut ullm_cuda_fwd) -> c_int;
    pub fn ullm_cuda_forward_create_gguf(ctx: *mut ullm_cuda_ctx, g: *const ullm_gguf, kv_f16: c_int, out: *mut *mut ullm_cuda_fwd) -> c_int;
    pub fn ullm_cuda_forward_create_st(ctx: *mut ullm_cuda_ctx, st: *const ullm_st, kv_f16: c_int, out: *mut *mut ullm_cuda_fwd) -> c_int;
    pub fn ullm_cuda_forward_destroy(f: *mut ullm_cuda_fwd);
    pub fn ullm_cuda_forward(f: *mut ullm_cuda_fwd, x_init: *const f32, pos: usize, logits: *mut f32) -> c_int;
    pub fn ullm_cuda_forward_debug(f: *mut ullm_cuda_fwd, x_init: *const f32, pos: usize, out: *mut ullm_debug_stat, cap: usize, n_out: *mut usize) -> c_int;
    pub fn ullm_cuda_forward_set_kv(f: *mut ullm_cuda_fwd, pos0: usize, n: usize, k: *const f32, v: *const f32) -> c_int;
    pub fn ullm_cuda_forward_supports_batched_prefill(f: *const ullm_cuda_fwd) -> c_int;
    pub fn ullm_cuda_forward_batch(f: *mut ullm_cuda_fwd, embeds: *const f32, s: usize, logits: *mut f32) -> c_int;
    pub fn ullm_cuda_forward_verify(f: *mut ullm_cuda_fwd, embeds: *const f32, parents: *const i32, n: usize, pos: usize, logits: *mut f32) -> c_int;
    pub fn ullm_cuda_forward_accept(f: *mut ullm_cuda_fwd, pos: usize, n: usize, path: *const i32, kept: usize) -> c_int;
    pub fn ullm_cuda_forward_greedy(f: *mut ullm_cuda_fwd, embd_table: *const ullm_cuda_buf, embd_dtype: c_int, first_token: u32, pos: usize, n: usize, tokens_out: *mut u32) -> c_int;
    pub fn ullm_cuda_forward_greedy_weight(f: *mut ullm_cuda_fwd, embd_table: *const ullm_cuda_weight, first_token: u32, pos: usize, n: usize, tokens_out: *mut u32) -> c_int;
    pub fn ullm_gguf_open(path: *const c_char, out: *mut *mut ullm_gguf, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_gguf_from_bytes(bytes: *const c_void, len: usize, out: *mut *mut ullm_gguf, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_gguf_close(g: *mut ullm_gguf);
    pub fn ullm_gguf_version(g: *const ullm_gguf) -> u32;
    pub fn ullm_gguf_architecture(g: *const ullm_gguf) -> *const c_char;
    pub fn ullm_gguf_alignment(g: *const ullm_gguf) -> u64;
    pub fn ullm_gguf_data_start(g: *const ullm_gguf) -> u64;
    pub fn ullm_gguf_tensor_count(g: *const ullm_gguf) -> usize;
    pub fn ullm_gguf_tensor_at(g: *const ullm_gguf, i: usize, out: *mut ullm_gguf_tensor) -> c_int;
    pub fn ullm_gguf_tensor_find(g: *const ullm_gguf, name: *const c_char, out: *mut ullm_gguf_tensor) -> c_int;
    pub fn ullm_gguf_meta_count(g: *const ullm_gguf) -> usize;
    pub fn ullm_gguf_meta_key_at(g: *const ullm_gguf, i: usize) -> *const c_char;
    pub fn ullm_gguf_meta_type(g: *const ullm_gguf, key: *const c_char, type_id: *mut c_int, elem_type_id: *mut c_int, array_len: *mut u64) -> c_int;
    pub fn ullm_gguf_meta_u64(g: *const ullm_gguf, key: *const c_char, out: *mut u64) -> c_int;
    pub fn ullm_gguf_meta_f32(g: *const ullm_gguf, key: *const c_char, out: *mut f32) -> c_int;
    pub fn ullm_gguf_meta_str(g: *const ullm_gguf, key: *const c_char, s: *mut *const c_char, len: *mut usize) -> c_int;
    pub fn ullm_gguf_meta_array_u64(g: *const ullm_gguf, key: *const c_char, i: usize, out: *mut u64) -> c_int;
    pub fn ullm_gguf_meta_array_f32(g: *const ullm_gguf, key: *const c_char, i: usize, out: *mut f32) -> c_int;
    pub fn ullm_gguf_meta_array_str(g: *const ullm_gguf, key: *const c_char, i: usize, s: *mut *const c_char, len: *mut usize) -> c_int;
    pub fn ullm_gguf_llama_params_get(g: *const ullm_gguf, out: *mut ullm_gguf_llama_params, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_st_open(path: *const c_char, out: *mut *mut ullm_st, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_st_from_bytes(bytes: *const c_void, len: usize, out: *mut *mut ullm_st, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_st_close(m: *mut ullm_st);
    pub fn ullm_st_shard_count(m: *const ullm_st) -> usize;
    pub fn ullm_st_tensor_count(m: *const ullm_st) -> usize;
    pub fn ullm_st_tensor_at(m: *const ullm_st, i: usize, out: *mut ullm_st_tensor) -> c_int;
    pub fn ullm_st_tensor_find(m: *const ullm_st, name: *const c_char, out: *mut ullm_st_tensor) -> c_int;
    pub fn ullm_st_has_tensor(m: *const ullm_st, name: *const c_char) -> c_int;
    pub fn ullm_st_config_u64(m: *const ullm_st, path: *const c_char, out: *mut u64) -> c_int;
    pub fn ullm_st_config_f32(m: *const ullm_st, path: *const c_char, out: *mut f32) -> c_int;
    pub fn ullm_st_config_str(m: *const ullm_st, path: *const c_char, s: *mut *const c_char, len: *mut usize) -> c_int;
    pub fn ullm_st_has_text_config(m: *const ullm_st) -> c_int;
    pub fn ullm_st_has_tokenizer_json(m: *const ullm_st) -> c_int;
    pub fn ullm_st_mlx_weight_get(m: *const ullm_st, name: *const c_char, group: u64, out: *mut ullm_st_mlx_weight, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_st_mlx_experts_get(m: *const ullm_st, name: *const c_char, n_experts: u64, out_dim: u64, in_dim: u64, group: u64, expert: u64, out: *mut ullm_st_mlx_weight, err: *mut c_char, err_cap: usize) -> c_int;
    pub fn ullm_st_mlx_params_get(m: *const ullm_st, out: *mut ullm_st_mlx_params, err: *mut c_char, err_cap: usize) -> c_int;
}
