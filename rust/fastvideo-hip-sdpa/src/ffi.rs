// @generated by gen_ffi.py from include/fv_sdpa_hip.h. Do not edit: edit the header and re-run.
//
// Raw C ABI of libfv_sdpa_hip.so. Return convention of the `c_int` entries: FV_OK launched,
// FV_DECLINED the kernel does not take the call (the reference's `Ok(None)`), negative =
// -(hipError_t) with a per-thread message behind fv_sdpa_last_error().
#![allow(clippy::too_many_arguments)]
use std::ffi::{c_char, c_int, c_longlong, c_void};

pub const FV_OK: c_int = 0;
pub const FV_DECLINED: c_int = 1;

pub const FV_PLAN_DENSE: c_int = 0;
pub const FV_PLAN_COMPOSED: c_int = 1;
pub const FV_PLAN_BLOCK_CAUSAL: c_int = 2;
pub const FV_PLAN_VDN_WINDOW: c_int = 3;
pub const FV_PLAN_KV_WINDOW: c_int = 4;
pub const FV_KV_ROPE_ABSOLUTE: c_int = 0;
pub const FV_KV_ROPE_RELATIVISTIC: c_int = 1;
pub const FV_KV_ROPE_REBASED_SINK: c_int = 2;
pub const FV_SDPA_SCALE_LOG2_DOMAIN: f32 = 0.6931471805599453;

/// `fv_tensor`: a device tensor descriptor (rt/tensor.rs:196-210 `CudaTensor`, device side).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct FvTensor {
    pub data: *mut c_void,
    /// 0 = f32, 1 = bf16 bits
    pub dtype: c_int,
    pub rank: c_int,
    pub shape: [usize; 8],
    /// 0 = contiguous; else (rank 4) the rows per (batch, head) plane of the storage
    pub plane_rows: usize,
}

/// `fv_plan`: rt/sdpa.rs:29-137 `Plan`, flattened.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct FvPlan {
    pub kind: c_int,
    pub has_scale: c_int,
    pub scale: f32,
    pub mask: *const FvTensor,
    pub fp8_first: c_int,
    pub block_tokens: usize,
    pub window: usize,
    pub sink: usize,
    pub video_start: usize,
    pub frame_tokens: usize,
    pub frames: usize,
    pub chunk: usize,
    pub radius: usize,
    /// -1 = FASTVIDEO_WAN_CAUSAL_FLASH, 0 composed f32, 1 dense route
    pub kv_flash: c_int,
}

/// `fv_kv_cache`: opaque.
#[repr(C)]
pub struct FvKvCache {
    _private: [u8; 0],
}

#[link(name = "fv_sdpa_hip")]
extern "C" {
    pub fn fv_sdpa_last_error() -> *const c_char;
    pub fn fv_sdpa_arch() -> *const c_char;
    pub fn fv_sdpa_init() -> c_int;
    pub fn fv_sdpa_supported(b: usize, h: usize, sq: usize, sk: usize, d: usize) -> c_int;
    pub fn fv_sdpa_is_log2_domain_scale(scale: f32) -> c_int;
    pub fn fv_sdpa_log2_domain_launches() -> u64;
    pub fn fv_sdpa_exact_pass_reruns() -> u64;
    pub fn fv_sdpa_dense_bf16(q: *const u16, k: *const u16, v: *const u16, out: *mut c_void, out_is_bf16: c_int, bh: usize, sq: usize, sk: usize, d: usize, scale: f32, stream: *mut c_void) -> c_int;
    pub fn fv_sdpa_dense_bf16_strided(q: *const u16, k: *const u16, v: *const u16, out: *mut c_void, out_is_bf16: c_int, bh: usize, sq: usize, sk: usize, d: usize, scale: f32, q_rows: usize, k_rows: usize, v_rows: usize, stream: *mut c_void) -> c_int;
    pub fn fv_sdpa_splitkv_choose(bh: usize, sq: usize, sk: usize) -> usize;
    pub fn fv_sdpa_splitkv_workspace_bytes(bh: usize, sq: usize, d: usize, splits: usize) -> usize;
    pub fn fv_sdpa_dense_bf16_splitkv(q: *const u16, k: *const u16, v: *const u16, out: *mut c_void, out_is_bf16: c_int, bh: usize, sq: usize, sk: usize, d: usize, scale: f32, q_rows: usize, k_rows: usize, v_rows: usize, splits: usize, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn fv_sdpa_splitkv_static_bytes() -> usize;
    pub fn fv_sdpa_splitkv_static_splits(bh: usize, sq: usize, sk: usize, d: usize, splits: usize) -> usize;
    pub fn fv_sdpa_dense_bf16_splitkv_static(q: *const u16, k: *const u16, v: *const u16, out: *mut c_void, out_is_bf16: c_int, bh: usize, sq: usize, sk: usize, d: usize, scale: f32, q_rows: usize, k_rows: usize, v_rows: usize, splits: usize, stream: *mut c_void) -> c_int;
    pub fn fv_sdpa_block_causal_bf16(q: *const u16, k: *const u16, v: *const u16, out: *mut c_void, out_is_bf16: c_int, bh: usize, sq: usize, sk: usize, d: usize, scale: f32, block_tokens: usize, window: usize, sink: usize, stream: *mut c_void) -> c_int;
    pub fn fv_sdpa_vdn_window_bf16(q: *const u16, k: *const u16, v: *const u16, out: *mut c_void, out_is_bf16: c_int, bh: usize, sq: usize, sk: usize, d: usize, scale: f32, video_start: usize, frame_tokens: usize, frames: usize, chunk: usize, radius: usize, stream: *mut c_void) -> c_int;
    pub fn fv_cast_f32_bf16(x: *const f32, y: *mut u16, n: usize, stream: *mut c_void) -> c_int;
    pub fn fv_cast_f32_bf16_scaled(x: *const f32, y: *mut u16, n: usize, mul: f32, stream: *mut c_void) -> c_int;
    pub fn fv_cast_bf16_f32(x: *const u16, y: *mut f32, n: usize, stream: *mut c_void) -> c_int;
    pub fn fv_softmax_last(x: *const f32, out: *mut c_void, out_is_bf16: c_int, rows: usize, width: usize, stream: *mut c_void) -> c_int;
    pub fn fv_sdpa_composed_f32(q: *const f32, k: *const f32, v: *const f32, mask: *const f32, mask_per_bh: c_int, out: *mut f32, bh: usize, sq: usize, sk: usize, d: usize, scale: f32, stream: *mut c_void) -> c_int;
    pub fn fv_rt_sdpa(q: *const FvTensor, k: *const FvTensor, v: *const FvTensor, plan: *const FvPlan, out: *mut FvTensor, stream: *mut c_void) -> c_int;
    pub fn fv_rt_free(p: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn fv_rt_sdpa_need(q: *const FvTensor, k: *const FvTensor, v: *const FvTensor, plan: *const FvPlan, need_out: *mut usize) -> c_int;
    pub fn fv_rt_sdpa_into(q: *const FvTensor, k: *const FvTensor, v: *const FvTensor, plan: *const FvPlan, out: *mut c_void, out_bytes: usize, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn fv_rt_set_bf16_activations(v: c_int);
    pub fn fv_rt_bf16_activations() -> c_int;
    pub fn fv_rt_set_fold_scale(v: c_int);
    pub fn fv_rt_fold_scale() -> c_int;
    pub fn fv_rt_log_level() -> c_int;
    pub fn fv_rt_parse_log_level(v: *const c_char) -> c_int;
    pub fn fv_rt_parse_backend(v: *const c_char) -> c_int;
    pub fn fv_rt_backend() -> c_int;
    pub fn fv_rt_set_backend(v: c_int);
    pub fn fv_rt_dense_route(q_shape: *const usize, k_shape: *const usize, v_shape: *const usize, masked: c_int, backend: c_int, steps_out: *mut c_int, dims_out: *mut usize) -> c_int;
    pub fn fv_rt_stats(out5: *mut u64);
    pub fn fv_kv_plan(capacity: usize, sink: usize, max_attention: usize, frame_tokens: usize, rolling: c_int, global_end: usize, local_end_prev: usize, current_start: usize, n: usize, move_out: *mut usize) -> c_int;
    pub fn fv_kv_copy_tokens(dst: *mut c_void, dst_rows: usize, dst_off: usize, src: *const c_void, src_rows: usize, src_off: usize, len: usize, bh: usize, d: usize, is_bf16: c_int, stream: *mut c_void) -> c_int;
    pub fn fv_kv_shift_tokens_down(t: *mut c_void, rows: usize, from: usize, to: usize, len: usize, bh: usize, d: usize, is_bf16: c_int, stream: *mut c_void) -> c_int;
    pub fn fv_kv_cache_new(capacity: usize, sink: usize, max_attention: usize, frame_tokens: usize, rolling: c_int, rope_policy: c_int, layers: usize) -> *mut FvKvCache;
    pub fn fv_kv_cache_new_dynamic(capacity: usize, sink: usize, max_attention: usize, frame_tokens: usize, rolling: c_int, rope_policy: c_int, layers: usize) -> *mut FvKvCache;
    pub fn fv_kv_cache_is_static(c: *const FvKvCache) -> c_int;
    pub fn fv_kv_cache_free(c: *mut FvKvCache);
    pub fn fv_kv_cache_reset(c: *mut FvKvCache);
    pub fn fv_kv_cache_set_sink_guard(c: *mut FvKvCache, on: c_int);
    pub fn fv_kv_cache_pointers(c: *const FvKvCache, layer: usize, out4: *mut usize) -> c_int;
    pub fn fv_kv_cache_set_pointers(c: *mut FvKvCache, in4: *const usize, layers: usize) -> c_int;
    pub fn fv_kv_cache_advance(c: *mut FvKvCache, current_start: usize, n: usize, sink_target: usize) -> c_int;
    pub fn fv_kv_cache_block_key(c: *const FvKvCache, current_start: usize, n: usize, sink_target: usize, out5: *mut usize) -> c_int;
    pub fn fv_kv_cache_rebase_sink(c: *mut FvKvCache, target: usize, orig_cos: *const f32, orig_sin: *const f32, new_cos: *const f32, new_sin: *const f32, stream: *mut c_void) -> c_int;
    pub fn fv_rope_bhsd(x: *const c_void, x_is_bf16: c_int, x_rows: usize, cos_t: *const f32, sin_t: *const f32, negate_sin: c_int, out: *mut c_void, out_is_bf16: c_int, out_rows: usize, bh: usize, s: usize, d: usize, stream: *mut c_void) -> c_int;
    pub fn fv_kv_cache_bytes(c: *const FvKvCache) -> usize;
    pub fn fv_kv_cache_update(c: *mut FvKvCache, layer: usize, k: *const FvTensor, v: *const FvTensor, current_start: usize, k_window: *mut FvTensor, v_window: *mut FvTensor, stream: *mut c_void) -> c_int;
    pub fn fv_paged_append(k: *const c_void, k_stride: usize, v: *const c_void, v_stride: usize, q: *const c_void, q_stride: usize, q_out: *mut u16, in_is_bf16: c_int, heads: usize, cos_t: *const f32, sin_t: *const f32, rope_rows: usize, rope_at: *const i32, halves: c_int, k_pages: *mut c_void, v_pages: *mut c_void, k_scales: *mut c_void, v_scales: *mut c_void, pages: usize, page_tokens: usize, kv_heads: usize, d: usize, q_start: *const i32, lens: *const i32, table: *const i32, table_stride: usize, table_pages: usize, seqs: usize, tokens: usize, stream: *mut c_void) -> c_int;
    pub fn fv_paged_read(k_out: *mut c_void, v_out: *mut c_void, out_is_bf16: c_int, k_pages: *const c_void, v_pages: *const c_void, k_scales: *const c_void, v_scales: *const c_void, pages: usize, page_tokens: usize, kv_heads: usize, d: usize, q_start: *const i32, lens: *const i32, table: *const i32, table_stride: usize, table_pages: usize, seqs: usize, tokens: usize, stream: *mut c_void) -> c_int;
    pub fn fv_paged_attention_workspace_bytes_for(four_bits: c_int, heads: usize, kv_heads: usize, d: usize, seqs: usize, tokens: usize, max_q: usize, max_len: usize, block_tokens: usize, window: usize, sink: usize) -> usize;
    pub fn fv_paged_attention_workspace_bytes(heads: usize, kv_heads: usize, d: usize, seqs: usize, tokens: usize, max_q: usize, max_len: usize, block_tokens: usize, window: usize, sink: usize) -> usize;
    pub fn fv_paged_attention(q: *const u16, q_stride: usize, out: *mut c_void, out_is_bf16: c_int, heads: usize, k_pages: *const c_void, v_pages: *const c_void, k_scales: *const c_void, v_scales: *const c_void, pages: usize, page_tokens: usize, kv_heads: usize, d: usize, q_start: *const i32, lens: *const i32, table: *const i32, table_stride: usize, table_pages: usize, seqs: usize, tokens: usize, max_q: usize, max_len: usize, scale: f32, block_tokens: usize, window: usize, sink: usize, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn fv_packed_attention_workspace_bytes(heads: usize, kv_heads: usize, d: usize, seqs: usize, q_tokens: usize, k_tokens: usize, max_q: usize, max_k: usize, causal: c_int, block_tokens: usize, window: usize, sink: usize) -> usize;
    pub fn fv_packed_attention(q: *const u16, q_stride: usize, k: *const u16, k_stride: usize, v: *const u16, v_stride: usize, out: *mut c_void, out_is_bf16: c_int, lse: *mut f32, heads: usize, kv_heads: usize, d: usize, q_start: *const i32, k_start: *const i32, seqs: usize, q_tokens: usize, k_tokens: usize, max_q: usize, max_k: usize, scale: f32, causal: c_int, block_tokens: usize, window: usize, sink: usize, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn fv_packed_attention_backward_workspace_bytes(dout_is_bf16: c_int, heads: usize, kv_heads: usize, d: usize, seqs: usize, q_tokens: usize, k_tokens: usize, max_q: usize, max_k: usize, causal: c_int, block_tokens: usize, window: usize, sink: usize) -> usize;
    pub fn fv_packed_attention_backward(dout: *const c_void, dout_is_bf16: c_int, q: *const u16, q_stride: usize, k: *const u16, k_stride: usize, v: *const u16, v_stride: usize, out: *const c_void, out_is_bf16: c_int, lse: *const f32, dq: *mut c_void, dk: *mut c_void, dv: *mut c_void, grads_are_bf16: c_int, heads: usize, kv_heads: usize, d: usize, q_start: *const i32, k_start: *const i32, seqs: usize, q_tokens: usize, k_tokens: usize, max_q: usize, max_k: usize, scale: f32, causal: c_int, block_tokens: usize, window: usize, sink: usize, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn fv_rope_frequencies(pairs: usize, base: f64, scaling: c_int, factor: f64, original: f64, low: f64, high: f64, out: *mut u64) -> c_int;
    pub fn fv_rope_tokens(q: *const c_void, q_stride: usize, q_out: *mut c_void, q_out_stride: usize, heads: usize, k: *const c_void, k_stride: usize, k_out: *mut c_void, k_out_stride: usize, kv_heads: usize, d: usize, in_is_bf16: c_int, out_is_bf16: c_int, freq: *const u64, pair_axis: *const i32, pairs: usize, positions: *const i32, axes: usize, tokens: usize, amplitude: f32, halves: c_int, inverse: c_int, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_topk_for(sparsity: f64, num_tiles: usize) -> usize;
    pub fn fv_vsa_default_sparsity() -> f64;
    pub fn fv_vsa_tile_plan(t: usize, h: usize, w: usize, dims_out: *mut usize, slot_src: *mut i32, token_slot: *mut u32, block_sizes: *mut i32) -> c_int;
    pub fn fv_vsa_tile_mean(x: *const c_void, x_is_bf16: c_int, slot_src: *const i32, block_sizes: *const i32, out: *mut f32, bh: usize, seq: usize, dim: usize, num_tiles: usize, round16: c_int, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_coarse(qc: *const f32, kc: *const f32, vc: *const f32, scores: *mut f32, coarse: *mut f32, bh: usize, num_tiles: usize, dim: usize, scale: f32, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_topk(scores: *const f32, out: *mut u32, rows: usize, n: usize, k: usize, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_tile_qkv(x: *const c_void, x_is_bf16: c_int, slot_src: *const i32, xt: *mut u16, bh: usize, seq: usize, padded: usize, dim: usize, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_fine(qt: *const u16, kt: *const u16, vt: *const u16, selected: *const u32, block_sizes: *const i32, out: *mut f32, bh: usize, num_tiles: usize, topk: usize, dim: usize, scale: f32, q_base: usize, q_tiles: usize, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_combine(sparse: *const f32, coarse: *const f32, gate: *const c_void, gate_is_bf16: c_int, slot_src: *const i32, out: *mut f32, bh: usize, seq: usize, dim: usize, num_tiles: usize, q_base: usize, q_tiles: usize, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_combine_round16(sparse: *const f32, coarse: *const f32, gate: *const c_void, gate_is_bf16: c_int, slot_src: *const i32, out: *mut f32, bh: usize, seq: usize, dim: usize, num_tiles: usize, q_base: usize, q_tiles: usize, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_workspace_bytes(bh: usize, num_tiles: usize, topk: usize, dim: usize) -> usize;
    pub fn fv_vsa_attention(q: *const c_void, k: *const c_void, v: *const c_void, qkv_is_bf16: c_int, gate: *const c_void, gate_is_bf16: c_int, slot_src: *const i32, block_sizes: *const i32, out: *mut f32, workspace: *mut c_void, workspace_bytes: usize, selected_out: *mut u32, bh: usize, seq: usize, num_tiles: usize, topk: usize, dim: usize, scale: f32, stream: *mut c_void) -> c_int;
    pub fn fv_vsa_attention_tiled(qt: *const u16, kt: *const u16, vt: *const u16, gate: *const c_void, gate_is_bf16: c_int, slot_src: *const i32, block_sizes: *const i32, out: *mut f32, workspace: *mut c_void, workspace_bytes: usize, selected_out: *mut u32, bh: usize, seq: usize, num_tiles: usize, topk: usize, dim: usize, scale: f32, stream: *mut c_void) -> c_int;
    pub fn fv_qk_norm_rope_bhsd(src: *const c_void, src_is_bf16: c_int, w: *const c_void, w_is_bf16: c_int, cos_t: *const f32, sin_t: *const f32, out: *mut c_void, out_is_bf16: c_int, batch: usize, seq: usize, heads: usize, d: usize, src_width: usize, col_off: usize, eps: f32, out_mul: f32, stream: *mut c_void) -> c_int;
    pub fn fv_qk_norm_rope_tiles(src: *const c_void, src_is_bf16: c_int, w: *const c_void, w_is_bf16: c_int, cos_t: *const f32, sin_t: *const f32, out: *mut c_void, out_is_bf16: c_int, batch: usize, seq: usize, heads: usize, d: usize, src_width: usize, col_off: usize, eps: f32, out_mul: f32, token_slot: *const u32, padded: usize, stream: *mut c_void) -> c_int;
    pub fn fv_split_heads_bhsd(src: *const c_void, out: *mut c_void, is_bf16: c_int, batch: usize, seq: usize, heads: usize, d: usize, src_width: usize, col_off: usize, stream: *mut c_void) -> c_int;
    pub fn fv_split_heads_tiles(src: *const c_void, out: *mut c_void, is_bf16: c_int, batch: usize, seq: usize, heads: usize, d: usize, src_width: usize, col_off: usize, token_slot: *const u32, padded: usize, stream: *mut c_void) -> c_int;
    pub fn fv_merge_heads(src: *const c_void, out: *mut c_void, is_bf16: c_int, batch: usize, heads: usize, seq: usize, d: usize, stream: *mut c_void) -> c_int;
    pub fn fv_block_causal_allows(block_tokens: usize, window: usize, sink: usize, q: usize, k: usize) -> c_int;
    pub fn fv_block_causal_dense_mask(block_tokens: usize, window: usize, sink: usize, sq: usize, sk: usize, mask: *mut f32);
    pub fn fv_vdn_window_allows(video_start: usize, frame_tokens: usize, frames: usize, chunk: usize, radius: usize, q: usize, k: usize) -> c_int;
    pub fn fv_vdn_window_dense_mask(video_start: usize, frame_tokens: usize, frames: usize, chunk: usize, radius: usize, sq: usize, sk: usize, mask: *mut f32);
    pub fn fv_block_causal_for(num_frames_per_block: usize, local_attn_size: c_longlong, frame_tokens: usize, out3: *mut usize) -> c_int;
    pub fn fv_block_causal_tile_walk(block_tokens: usize, window: usize, sink: usize, sq: usize, sk: usize, q0: usize, out4: *mut c_int) -> c_int;
    pub fn fv_sp_shard_ranges(seq: usize, world: usize, out: *mut usize);
}
