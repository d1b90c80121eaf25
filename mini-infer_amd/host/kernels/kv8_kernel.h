// kv8_kernel.h -- launchers of the paged KV cache held in 8 bits: rotary
// positions into it, its writes, the attention over it and its pages.  The
// reference has no counterpart (its cache is fp16,
// src/kernels/model_utils_kernel.cuh:53-67).  All forward to the C ABI
// (include/mi_kernels.h, which has the formulas and limits) and throw
// std::runtime_error if a launch is rejected.
#pragma once

#include <cstdint>

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "mi_kernels.h"

namespace mini_infer {
namespace kernels {

// In place: rotary positions of q [T, Hq, hd] and k [T, Hkv, hd], tokens
// q_stride / k_stride elements apart (slices of a fused QKV product), over the
// first rotary_dim elements of a head, NeoX halves or neighbouring pairs; cos
// and sin times mscale.  positions_d [T] on the device, inv_freq_h
// [rotary_dim / 2] on the host.
void launch_rope_partial_qk(__half* q, __half* k, const int64_t* positions_d,
                            const float* inv_freq_h, int T, int Hq, int Hkv, int head_dim,
                            int rotary_dim, int64_t q_stride, int64_t k_stride, bool interleaved,
                            float mscale, hipStream_t stream);

// K and V [B*S, Hkv, hd] into layer `layer` of an 8-bit cache k_cache /
// v_cache [L, num_blocks, Hkv, block_size, hd] with one exponent byte per page
// and head in k_scale / v_scale [L, num_blocks, Hkv], where
// launch_paged_kv_scatter_kv places them.
void launch_kv8_scatter(const __half* k, const __half* v, uint8_t* k_cache, uint8_t* v_cache,
                        uint8_t* k_scale, uint8_t* v_scale, const int* block_table,
                        const int* seq_len, const int* start_pos, int B, int S, int layer,
                        int num_blocks, int Hkv, int head_dim, int block_size,
                        int max_blocks_per_seq, hipStream_t stream);

// Workspace of launch_kv8_attention for a [B, S] batch: zeros before its first
// use, then for this function alone.
int64_t kv8_attention_workspace_bytes(int B, int S, int Hq, int Hkv, int head_dim,
                                      int max_blocks_per_seq);

// Causal attention of q [B*S, Hq, hd] over layer `layer` of an 8-bit cache that
// holds the tokens' own K and V; window > 0: over each token's last `window`
// keys.  out [B*S, Hq, hd].
void launch_kv8_attention(const __half* q, const uint8_t* k_cache, const uint8_t* v_cache,
                          const uint8_t* k_scale, const uint8_t* v_scale, __half* out,
                          const int* block_table, const int* seq_len, const int* start_pos, int B,
                          int S, int Hq, int Hkv, int head_dim, float scale, int window, int layer,
                          int num_blocks, int block_size, int max_blocks_per_seq, void* workspace,
                          int64_t workspace_bytes, hipStream_t stream);

// The pages of a cache, kept on the device (mi_kv_pages_*): status [n] gets
// MI_KV_DONE, MI_KV_FULL or MI_KV_REFUSED per row or pair.
void launch_kv_copy_pages(const mi_kv_pages* caches, int num_caches, int num_blocks, const int* src,
                          const int* dst, int n, int* status, hipStream_t stream);
void launch_kv_free(int* block_table, int* seq_len, int* ref_count, int B, int max_blocks_per_seq,
                    int num_blocks, const int* rows, int n, hipStream_t stream);
void launch_kv_fork(int* block_table, int* seq_len, int* ref_count, int B, int max_blocks_per_seq,
                    int num_blocks, const int* parents, const int* children, int n, int* status,
                    hipStream_t stream);
int64_t kv_pages_workspace_bytes(int num_blocks, int n);
void launch_kv_reserve(const mi_kv_pages* caches, int num_caches, int* block_table, int* seq_len,
                       int* ref_count, int B, int max_blocks_per_seq, int num_blocks,
                       int block_size, const int* rows, const int* lengths, int n, int* status,
                       void* workspace, int64_t workspace_bytes, hipStream_t stream);
void launch_kv_compact(const mi_kv_pages* caches, int num_caches, int* block_table, int* ref_count,
                       int B, int max_blocks_per_seq, int num_blocks, int* moved, void* workspace,
                       int64_t workspace_bytes, hipStream_t stream);

}  // namespace kernels
}  // namespace mini_infer
