// Host-callable launchers of the attention operators (attention_kernels.cu, paged_attention.cu). All pointers are
// device addresses on the current device; every call is stream-ordered and returns 0 or a CUDA error. Element types
// are AttnType codes.
#pragma once

#include <cstddef>
#include <cstdint>

namespace rocshmem {
namespace kernels {

enum AttnType : int { ATTN_BF16 = 0, ATTN_F16 = 1, ATTN_F32 = 2, ATTN_E4M3 = 3 };

// Queries and keys of one call of the norm + rotation: rows of `dim` elements at base + t * token + h * head (strides
// in elements); outputs are contiguous [tokens, heads, dim].
struct NormRopeArgs {
  const void *q, *k;
  long long q_token, q_head, k_token, k_head;
  const void *q_weight, *k_weight;
  const void *positions;  // [tokens], 32- or 64-bit
  const float *table;  // [table_rows, rotary]: cosines, then sines
  int tokens, q_heads, k_heads, dim, rotary, table_rows;
  float eps;
  int interleaved, type, weight_type, wide_positions;
};
int qk_norm_rope(const NormRopeArgs &a, void *q_out, void *k_out, void *stream);
// Floats of workspace that the backward pass needs.
size_t qk_norm_rope_workspace(int dim);
// gq, gk: contiguous gradients of the outputs. dq, dk contiguous; dq_weight, dk_weight of the weights' type.
int qk_norm_rope_backward(const NormRopeArgs &a, const void *gq, const void *gk, void *dq, void *dk, void *dq_weight,
                          void *dk_weight, float *workspace, void *stream);

// A paged cache: k, v [pages, kv_heads, page_size, dim], scales [pages, kv_heads, page_size] for e4m3 (else null).
struct KvCacheArgs {
  void *k, *v;
  float *k_scale, *v_scale;
  int pages, kv_heads, page_shift, dim, type;
};
// Rows k[t, h, :], v[t, h, :] (strides in elements) go to slots[t] (32- or 64-bit); slots outside the cache are
// skipped.
int kv_cache_write(const KvCacheArgs &c, const void *k, const void *v, long long k_token, long long k_head,
                   long long v_token, long long v_head, const void *slots, int wide_slots, int tokens, int type,
                   void *stream);
// k_out, v_out [tokens, kv_heads, dim] contiguous; rows of slots outside the cache become zeros.
int kv_cache_read(const KvCacheArgs &c, void *k_out, void *v_out, const void *slots, int wide_slots, int tokens,
                  int type, void *stream);

struct PagedAttentionArgs {
  const void *q;
  long long q_token, q_head;
  const int *block_table;  // [batch, max_pages]
  long long table_stride;
  const int *lengths;
  int batch, heads, max_pages, window;
  float scale, softcap;
  int q_type, out_type;
  void *out;   // [batch, heads, dim]
  float *lse;  // [batch, heads] or null
};
// Bytes of workspace that a call needs (which may be none); 0 when the sizes are refused.
size_t paged_attention_workspace(const KvCacheArgs &c, const PagedAttentionArgs &a);
int paged_attention(const KvCacheArgs &c, const PagedAttentionArgs &a, void *workspace, size_t workspace_bytes,
                    void *stream);

// outs [parts, rows, dim] (part stride in elements), lses [parts, rows] (part stride in elements) -> out [rows, dim],
// lse [rows].
int attention_join(const void *outs, const float *lses, long long out_part, long long lse_part, int parts,
                   long long rows, int dim, int in_type, int out_type, void *out, float *lse, void *stream);

}  // namespace kernels
}  // namespace rocshmem
