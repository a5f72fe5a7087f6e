//! Raw declarations of the C ABI in `include/krikil_cuda.h`, one for one (same
//! names, argument order and C types).  Handles are opaque; every function
//! returns a `krk_status` (`KRK_OK` = 0) unless noted, with the message of the
//! last failure on the calling thread in `krk_last_error()`.  Device pointers
//! are passed as raw pointers; `stream` is a `cudaStream_t` (null = the
//! default stream).
#![allow(non_camel_case_types, dead_code)]

use std::ffi::{c_char, c_double, c_float, c_int, c_void};

pub const KRK_ABI_VERSION: c_int = 1;

pub const KRK_HIDDEN: usize = 608;
pub const KRK_VOCAB: usize = 2048;
pub const KRK_INTERMEDIATE: usize = 2432;
pub const KRK_LAYERS: usize = 8;
pub const KRK_ATTN_HEADS: usize = 8;
pub const KRK_ATTN_HEAD_DIM: usize = 76;
pub const KRK_MAMBA_D_STATE: usize = 128;
pub const KRK_MAMBA_D_CONV: usize = 4;
pub const KRK_MAMBA_D_INNER: usize = 1216;
pub const KRK_MAMBA_HEAD_DIM: usize = 64;
pub const KRK_MAMBA_HEADS: usize = 19;
pub const KRK_MAMBA_D_IN_PROJ: usize = 2707;
pub const KRK_MAMBA_D_XBC: usize = 1472;
pub const KRK_EOS_TOKEN: u32 = 0;

// enum krk_status
pub const KRK_OK: c_int = 0;
pub const KRK_BAD_TOKEN: c_int = 1;
pub const KRK_CONTEXT_OVERFLOW: c_int = 2;
pub const KRK_EMPTY: c_int = 3;
pub const KRK_IO: c_int = 4;
pub const KRK_NOT_FOUND: c_int = 5;
pub const KRK_INVALID: c_int = 6;
pub const KRK_CUDA: c_int = 7;
pub const KRK_CHECK_FAILED: c_int = 8;

// krk_state_profile classes
pub const KRK_PROF_DEVICE_TOTAL: c_int = 0;
pub const KRK_PROF_GEMM: c_int = 1;
pub const KRK_PROF_SSD_STEP: c_int = 2;
pub const KRK_PROF_ATTN_DECODE: c_int = 3;
pub const KRK_PROF_NORM: c_int = 4;
pub const KRK_PROF_CONV: c_int = 5;
pub const KRK_PROF_SSD_SCAN: c_int = 6;
pub const KRK_PROF_ATTN_PREFILL: c_int = 7;
pub const KRK_PROF_OTHER: c_int = 8;
pub const KRK_PROF_CLASSES: c_int = 9;

pub const KRK_ATTN_NOALLOC_MAX_FLOATS: usize = 1 << 20;

// krk_check_status bits (checked builds)
pub const KRK_CHECK_TOKEN: u32 = 1;
pub const KRK_CHECK_POSITION: u32 = 2;
pub const KRK_CHECK_TABLE: u32 = 4;
pub const KRK_CHECK_COLUMN: u32 = 8;

// element types of the paged key-value cache
pub const KRK_TYPE_F32: c_int = 0;
pub const KRK_TYPE_F16: c_int = 1;
pub const KRK_TYPE_BF16: c_int = 2;

// status bits of krk_k_kv_page_plan and krk_k_kv_page_release
pub const KRK_PAGES_EXHAUSTED: i32 = 1;
pub const KRK_PAGES_ROW_FULL: i32 = 2;
pub const KRK_PAGES_ROWS: i32 = 4;
pub const KRK_PAGES_BAD_LENGTH: i32 = 8;
pub const KRK_PAGES_OVERFLOW: i32 = 16;

#[repr(C)]
pub struct krk_model {
    _private: [u8; 0],
}
#[repr(C)]
pub struct krk_state {
    _private: [u8; 0],
}

extern "C" {
    pub fn krk_last_error() -> *const c_char;
    pub fn krk_status_string(status: c_int) -> *const c_char;
    pub fn krk_abi_version() -> c_int;

    pub fn krk_model_load(path: *const c_char, device: c_int, out: *mut *mut krk_model) -> c_int;
    pub fn krk_model_free(model: *mut krk_model) -> c_int;
    pub fn krk_model_device(model: *const krk_model, device: *mut c_int) -> c_int;
    pub fn krk_model_stream(model: *const krk_model, stream: *mut *mut c_void) -> c_int;

    pub fn krk_state_create(model: *const krk_model, batch: c_int, max_ctx: c_int, out: *mut *mut krk_state) -> c_int;
    pub fn krk_state_free(state: *mut krk_state) -> c_int;
    pub fn krk_state_reset(state: *mut krk_state, mask: *const u8) -> c_int;
    pub fn krk_state_batch(state: *const krk_state, batch: *mut c_int) -> c_int;
    pub fn krk_state_context_limit(state: *const krk_state, max_ctx: *mut c_int) -> c_int;
    pub fn krk_state_positions(state: *const krk_state, pos_out: *mut i64) -> c_int;

    pub fn krk_prefill(model: *const krk_model, state: *mut krk_state, tokens: *const u32, lens: *const i32,
                       logits_out: *mut c_float) -> c_int;
    pub fn krk_step(model: *const krk_model, state: *mut krk_state, tokens: *const u32, logits_out: *mut c_float)
                    -> c_int;
    pub fn krk_generate_greedy(model: *const krk_model, state: *mut krk_state, prompts: *const u32,
                               lens: *const i32, max_new_tokens: c_int, repetition_penalty: c_float,
                               stop_at_eos: c_int, tokens_out: *mut u32, n_out: *mut i32) -> c_int;
    pub fn krk_generate_sample(model: *const krk_model, state: *mut krk_state, prompts: *const u32,
                               lens: *const i32, max_new_tokens: c_int, temperature: c_float, top_p: c_float,
                               top_k: c_int, repetition_penalty: c_float, seeds: *const u64, stop_at_eos: c_int,
                               tokens_out: *mut u32, n_out: *mut i32) -> c_int;
    pub fn krk_state_export(state: *const krk_state, seq: c_int, layer: c_int, what: c_int, out: *mut c_float,
                            n: i64) -> c_int;
    pub fn krk_launch_count(count: *mut u64) -> c_int;
    pub fn krk_checked_build() -> c_int;
    pub fn krk_check_status(bits: *mut u32, clear: c_int) -> c_int;
    pub fn krk_state_set_decode_streams(state: *mut krk_state, n: c_int) -> c_int;
    pub fn krk_state_set_step_graphs(state: *mut krk_state, enable: c_int) -> c_int;
    pub fn krk_state_profile(state: *mut krk_state, enable: c_int) -> c_int;
    pub fn krk_state_profile_read(state: *const krk_state, cls: c_int, total_ms: *mut c_double,
                                  launches: *mut i64) -> c_int;
    pub fn krk_state_profile_units(state: *const krk_state, cls: c_int, units: *mut i64) -> c_int;

    // per-kernel entry points (device pointers, asynchronous on `stream`)
    pub fn krk_k_rmsnorm_rows(x: *const c_float, w: *const c_float, eps: c_float, rows: i64, dim: c_int,
                              y: *mut c_float, stream: *mut c_void) -> c_int;
    pub fn krk_k_rmsnorm_fm(x: *const c_float, ldx: c_int, w: *const c_float, eps: c_float, k: c_int, m: c_int,
                            out: *mut c_float, ldo: c_int, stream: *mut c_void) -> c_int;
    pub fn krk_k_gated_rmsnorm_residual(x: *const c_float, z: *const c_float, res: *const c_float,
                                        w: *const c_float, eps: c_float, rows: i64, dim: c_int, y: *mut c_float,
                                        stream: *mut c_void) -> c_int;
    pub fn krk_k_gemm(at: *const c_float, lda: c_int, wt: *const c_float, ldw: c_int, c: *mut c_float, ldc: c_int,
                      m: c_int, n: c_int, k: c_int, epilogue: c_int, out_fm: c_int, stream: *mut c_void) -> c_int;
    pub fn krk_k_gemm_tiled(at: *const c_float, lda: c_int, wt: *const c_float, ldw: c_int, c: *mut c_float,
                            ldc: c_int, m: c_int, n: c_int, k: c_int, epilogue: c_int, out_fm: c_int,
                            tile_rows: c_int, stream: *mut c_void) -> c_int;
    pub fn krk_k_gemm_tile_rows(m: c_int, n: c_int) -> c_int;
    pub fn krk_k_embed(tok: *const u32, wte: *const c_float, vocab: c_int, k: c_int, m: c_int, out: *mut c_float,
                       ldo: c_int, stream: *mut c_void) -> c_int;
    pub fn krk_k_pointwise(op: c_int, x: *const c_float, y: *mut c_float, n: i64, stream: *mut c_void) -> c_int;
    pub fn krk_k_conv_ssd_step(x: *const c_float, bm: *const c_float, cm: *const c_float, dt: *const c_float,
                               conv_state: *mut c_float, conv_w: *const c_float, conv_b: *const c_float,
                               ssm: *mut c_float, dt_bias: *const c_float, a_neg: *const c_float,
                               dsk: *const c_float, y: *mut c_float, b: c_int, h: c_int, p: c_int, n: c_int,
                               stream: *mut c_void) -> c_int;
    pub fn krk_k_conv_ssd_scan(x: *const c_float, bm: *const c_float, cm: *const c_float, dt: *const c_float,
                               conv_state: *mut c_float, conv_w: *const c_float, conv_b: *const c_float,
                               ssm: *mut c_float, dt_bias: *const c_float, a_neg: *const c_float,
                               dsk: *const c_float, y: *mut c_float, b: c_int, t: c_int, h: c_int, p: c_int,
                               n: c_int, stream: *mut c_void) -> c_int;
    /// Returns a size, not a status.
    pub fn krk_attn_work_floats(b: c_int, h: c_int, dh: c_int, ctx: c_int, split: c_int) -> usize;
    pub fn krk_k_rope_kv_attn_decode(q: *const c_float, k: *const c_float, v: *const c_float, kc: *mut c_float,
                                     vc: *mut c_float, pos: *const i32, out: *mut c_float, work: *mut c_float,
                                     b: c_int, h: c_int, dh: c_int, ctx: c_int, split: c_int, theta: c_float,
                                     stream: *mut c_void) -> c_int;
    pub fn krk_k_gemm_sgemm_order(at: *const c_float, lda: c_int, wt: *const c_float, ldw: c_int, c: *mut c_float,
                                  ldc: c_int, m: c_int, n: c_int, k: c_int, stream: *mut c_void) -> c_int;
    pub fn krk_k_attn_prefill_rows(kmax: c_int, dh: c_int) -> c_int;
    pub fn krk_k_rope_kv_attn_prefill(qkv: *mut c_float, q_rs: i64, kc: *mut c_float, vc: *mut c_float, c_sb: i64,
                                      c_sh: i64, c_st: i64, cu_seqlens: *const i32, start: *const i32, s: c_int,
                                      total_rows: c_int, h: c_int, dh: c_int, theta: c_float, blocks: *const i32,
                                      nblocks: c_int, rows_per_block: c_int, kmax: c_int, out: *mut c_float,
                                      o_rs: i64, o_cs: i64, stream: *mut c_void) -> c_int;
    pub fn krk_k_rope_kv_attn_decode_noalloc(q: *const c_float, k: *const c_float, v: *const c_float,
                                             kc: *mut c_float, vc: *mut c_float, pos: *const i32,
                                             out: *mut c_float, b: c_int, h: c_int, dh: c_int, ctx: c_int,
                                             split: c_int, theta: c_float, stream: *mut c_void) -> c_int;
    pub fn krk_k_kv_page_plan(new_tokens: *const i32, lens: *const i32, table: *mut i32, table_ld: i64, b: c_int,
                              width: c_int, free_pages: *const i32, free_count: *const i32, num_pages: c_int,
                              page_size: c_int, lens_out: *mut i32, free_count_out: *mut i32, cu_new: *mut i32,
                              positions: *mut i32, slots: *mut i32, rows: c_int, status: *mut i32,
                              stream: *mut c_void) -> c_int;
    pub fn krk_k_kv_page_release(done_mask: *const u8, lens: *const i32, table: *const i32, table_ld: i64,
                                 b: c_int, width: c_int, free_pages: *mut i32, free_count: *const i32,
                                 num_pages: c_int, page_size: c_int, lens_out: *mut i32, free_count_out: *mut i32,
                                 status: *mut i32, stream: *mut c_void) -> c_int;
    pub fn krk_k_rope_kv_append_paged(q: *mut c_void, q_st: i64, q_sh: i64, k: *mut c_void, k_st: i64, k_sh: i64,
                                      v: *mut c_void, v_st: i64, v_sh: i64, dtype: c_int, q_out: *mut c_void,
                                      qo_st: i64, qo_sh: i64, kc: *mut c_void, vc: *mut c_void, c_sp: i64,
                                      c_st: i64, c_sh: i64, cache_type: c_int, slots: *const i32,
                                      positions: *const i32, t: c_int, hq: c_int, hkv: c_int, dh: c_int,
                                      rot_dim: c_int, num_pages: c_int, page_size: c_int, theta: c_float,
                                      stream: *mut c_void) -> c_int;
    /// Returns a size, not a status.
    pub fn krk_attn_paged_work_floats(b: c_int, hq: c_int, hkv: c_int, dh: c_int, max_len: c_int, window: c_int)
                                      -> usize;
    pub fn krk_k_attn_decode_paged(q: *mut c_void, q_sb: i64, q_sh: i64, dtype: c_int, kc: *mut c_void,
                                   vc: *mut c_void, c_sp: i64, c_st: i64, c_sh: i64, cache_type: c_int,
                                   table: *const i32, table_ld: i64, width: c_int, num_pages: c_int,
                                   page_size: c_int, lens: *const i32, b: c_int, hq: c_int, hkv: c_int, dh: c_int,
                                   scale: c_float, window: c_int, max_len: c_int, out: *mut c_void, o_sb: i64,
                                   o_sh: i64, lse: *mut c_float, work: *mut c_float, work_floats: usize,
                                   stream: *mut c_void) -> c_int;
    pub fn krk_k_causal_conv(x: *mut c_void, x_st: i64, weight: *const c_float, bias: *const c_float,
                             out: *mut c_void, o_st: i64, dtype: c_int, state: *mut c_void, state_stride: i64,
                             num_slots: c_int, slots: *const i32, init: *const i32, cu: *const i32, rows: c_int,
                             requests: c_int, channels: c_int, width: c_int, silu: c_int,
                             stream: *mut c_void) -> c_int;
    pub fn krk_k_causal_conv_step(x: *mut c_void, x_st: i64, weight: *const c_float, bias: *const c_float,
                                  out: *mut c_void, o_st: i64, dtype: c_int, state: *mut c_void, state_stride: i64,
                                  num_slots: c_int, slots: *const i32, init: *const i32, rows: c_int,
                                  channels: c_int, width: c_int, silu: c_int, stream: *mut c_void) -> c_int;
    /// Returns a size, not a status.
    pub fn krk_selective_scan_work_floats(rows: c_int, channels: c_int, states: c_int, groups: c_int, max_len: c_int)
                                          -> usize;
    pub fn krk_k_selective_scan(x: *mut c_void, x_st: i64, dt: *mut c_void, dt_st: i64, z: *mut c_void, z_st: i64,
                                b: *mut c_void, b_st: i64, b_sg: i64, c: *mut c_void, c_st: i64, c_sg: i64,
                                out: *mut c_void, o_st: i64, dtype: c_int, a: *const c_float, d: *const c_float,
                                dt_bias: *const c_float, state: *mut c_float, state_stride: i64, num_slots: c_int,
                                slots: *const i32, init: *const i32, cu: *const i32, rows: c_int, requests: c_int,
                                channels: c_int, states: c_int, groups: c_int, max_len: c_int, work: *mut c_float,
                                work_floats: usize, stream: *mut c_void) -> c_int;
    pub fn krk_k_selective_step(x: *mut c_void, x_st: i64, dt: *mut c_void, dt_st: i64, z: *mut c_void, z_st: i64,
                                b: *mut c_void, b_st: i64, b_sg: i64, c: *mut c_void, c_st: i64, c_sg: i64,
                                out: *mut c_void, o_st: i64, dtype: c_int, a: *const c_float, d: *const c_float,
                                dt_bias: *const c_float, state: *mut c_float, state_stride: i64, num_slots: c_int,
                                slots: *const i32, init: *const i32, rows: c_int, channels: c_int, states: c_int,
                                groups: c_int, stream: *mut c_void) -> c_int;
    pub fn krk_k_token_logprobs(logits: *mut c_void, ld: i64, dtype: c_int, rows: c_int, vocab: c_int,
                                tokens: *const i32, asked: c_int, logprobs: *mut c_float, entropy: *mut c_float,
                                top: c_int, top_ids: *mut i32, top_logprobs: *mut c_float,
                                stream: *mut c_void) -> c_int;
    pub fn krk_k_wait_probe(src16: *const c_float, polls: c_int, copy: c_int, status: *mut i32,
                            stream: *mut c_void) -> c_int;
    pub fn krk_k_greedy(logits: *const c_float, ld: i64, vocab: c_int, b: c_int, seen: *mut u32, penalty: c_float,
                        tok: *mut u32, stream: *mut c_void) -> c_int;
    pub fn krk_k_sample(logits: *const c_float, ld: i64, vocab: c_int, b: c_int, seen: *mut u32,
                        temperature: c_float, top_p: c_float, top_k: c_int, penalty: c_float, rng_state: *mut u32,
                        tok: *mut u32, stream: *mut c_void) -> c_int;
    pub fn krk_rng_seed_state(seed: u64, state10: *mut u32) -> c_int;
}
