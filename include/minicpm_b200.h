/*
 * minicpm_b200.h -- C ABI of the sm_100a paged prefill attention and the
 * fused RoPE + paged KV-cache write.
 *
 * Plain C: device pointers, element strides and sizes; no framework types.
 * Every entry point returns a status code (B200_OK on success) and never
 * throws; b200_last_error() gives the message of the last failure on the
 * calling thread.  All work is enqueued on the given CUDA stream
 * (a cudaStream_t passed as void*; NULL is the legacy default stream) and
 * no entry point synchronises the host, allocates device memory or
 * launches anything on another stream.
 *
 * Reference interfaces replaced (paths inside the reference project):
 *   b200_paged_attn_fwd    -> the two launches of paged_split_kv_attention,
 *                             kernels/triton_split_kv_paged.py:283-360
 *                             (_split_kv_forward :18-155, _split_kv_reduce
 *                             :158-228), including the q-block compaction
 *                             (:283-293) that the reference does on the host.
 *   b200_split_combine     -> the _split_kv_reduce launch on its own,
 *                             kernels/triton_split_kv_paged.py:342-360.
 *   b200_rope_kv_write     -> the _rope_and_cache_kernel launch of
 *                             fused_rope_and_cache,
 *                             kernels/triton_rope_kv_cache.py:261-286.
 *   b200_choose_num_splits -> the fixed split count of
 *                             kernels/attention.py:166 and
 *                             kernels/triton_unified_attention_optimized.py:216-218
 *                             (the reference has no automatic choice).
 *   b200_attn_workspace_bytes -> the per-call scratch allocation of
 *                             kernels/triton_split_kv_paged.py:295-306.
 *   b200_kv_cache_write    -> the service's plain KV-cache update,
 *                             IluvatarAttentionImpl.do_kv_cache_update
 *                             (integration/vllm-plugin-FL-split-kv.patch:815-858),
 *                             i.e. vLLM's triton_reshape_and_cache_flash and
 *                             triton_reshape_and_cache_flash_per_token_head_quant.
 *   b200_rope_kv_write with key_out / an fp8 cache
 *                          -> the service RoPE ABI,
 *                             IluvatarAttentionImpl.do_rope_and_kv_cache_update
 *                             (integration/vllm-plugin-FL-split-kv.patch:865-899).
 */
#ifndef MINICPM_B200_H_
#define MINICPM_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B200_ABI_VERSION 2

#if defined(__GNUC__)
#define B200_API __attribute__((visibility("default")))
#else
#define B200_API
#endif

/* Status codes. */
#define B200_OK 0
#define B200_ERR_INVALID 1     /* bad shape, stride, dtype or argument value  */
#define B200_ERR_UNSUPPORTED 2 /* valid for the reference, not for this build */
#define B200_ERR_CUDA 3        /* a CUDA runtime / driver call failed          */
#define B200_ERR_WORKSPACE 4   /* workspace missing or too small               */

/* Element types. */
#define B200_DTYPE_F16 0
#define B200_DTYPE_BF16 1
#define B200_DTYPE_F32 2
#define B200_DTYPE_I32 3
#define B200_DTYPE_I64 4
#define B200_DTYPE_FP8_E4M3 5 /* cache element types of the quantised KV-cache writes */
#define B200_DTYPE_FP8_E5M2 6
#define B200_DTYPE_I8 7

/* KV-cache quantisation modes (same numbering as vLLM's KVQuantMode). */
#define B200_KVQ_NONE 0               /* cache dtype == key dtype: bit copy                */
#define B200_KVQ_FP8_PER_TENSOR 1     /* fp8(x / scale), one device float per cache        */
#define B200_KVQ_INT8_PER_TOKEN_HEAD 2 /* int8 with a dynamic scale per (token, head)      */
#define B200_KVQ_FP8_PER_TOKEN_HEAD 3  /* fp8 e4m3 with a dynamic scale per (token, head)  */

/* Device-side error codes (b200_device_error). */
#define B200_DEVERR_NONE 0u
#define B200_DEVERR_WAIT_TIMEOUT 1u /* an in-kernel wait ran past its limit     */
#define B200_DEVERR_SLOT_RANGE 2u   /* slot_mapping entry >= num_blocks*bs      */
#define B200_DEVERR_POS_RANGE 3u    /* position outside the cos/sin table        */
#define B200_DEVERR_DECODE_QLEN 4u  /* max_seqlen_q = 1 but a sequence has more query tokens */
#define B200_DEVERR_SEQ_ROW 5u      /* a table row out of range, named twice, in use, or with a bad length */
#define B200_DEVERR_NO_PAGE 6u      /* no free page was left                     */
#define B200_DEVERR_PAGE_RANGE 7u   /* a page id out of range, a missing page, or a release of a free page */
#define B200_DEVERR_PAGE_SHARED 8u  /* a row would be written into a page that other sequences share */
#define B200_DEVERR_ACCEPT 9u       /* an accepted path that does not rise, or a bad count */

/*
 * Paged causal varlen attention (prefill / chunked prefill), GQA, Split-KV.
 *
 * q          [total_q, num_q_heads, head_dim], element strides q_stride_t/h, d contiguous
 * k, v       paged caches [num_blocks, block_size, num_kv_heads, head_dim], strides
 *            *_stride_block/_tok/_head, d contiguous (the cache[:, 0] / cache[:, 1]
 *            views of a [num_blocks, 2, block_size, KH, D] cache are accepted)
 * out        [total_q, num_q_heads, head_dim], written in place
 * block_table [num_seqs, block_table_cols], int32 or int64, row stride in elements
 * cu_seqlens_q [num_seqs + 1], seqused_k [num_seqs]: int32 or int64
 * num_splits  0 = choose automatically, else 1..16.  A decode batch (max_seqlen_q == 1)
 *             runs the decode kernel, which splits the keys of each sequence into
 *             chunks of its own choosing; num_splits does not change the result.
 * workspace   device buffer of at least b200_attn_workspace_bytes(...) bytes,
 *             owned by the caller; must not be shared by calls that overlap.
 * All pointers: 16-byte aligned; all strides except d: multiples of 8 elements.
 */
typedef struct B200AttnParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const void* block_table;
  const void* cu_seqlens_q;
  const void* seqused_k;
  int64_t q_stride_t, q_stride_h;
  int64_t k_stride_block, k_stride_tok, k_stride_head;
  int64_t v_stride_block, v_stride_tok, v_stride_head;
  int64_t out_stride_t, out_stride_h;
  int64_t block_table_stride;
  int32_t block_table_cols;
  int32_t block_table_dtype; /* B200_DTYPE_I32 / I64 */
  int32_t seqlen_dtype;      /* dtype of cu_seqlens_q and seqused_k: I32 / I64 */
  int32_t dtype;             /* q / k / v / out element type: F16 / BF16 */
  int32_t num_seqs;
  int32_t total_q;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t block_size;
  int32_t num_blocks;
  int32_t max_seqlen_q;
  int32_t max_seqlen_k;
  int32_t num_splits;
  float softmax_scale;
  void* workspace;
  size_t workspace_bytes;
} B200AttnParams;

/* Workspace bytes b200_paged_attn_fwd needs for these sizes (num_splits 0 = auto). */
B200_API size_t b200_attn_workspace_bytes(int32_t total_q, int32_t num_seqs, int32_t num_q_heads,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t num_splits,
                                 int32_t max_seqlen_k, int32_t dtype);

/* The split count b200_paged_attn_fwd uses for num_splits = 0. */
B200_API int32_t b200_choose_num_splits(int32_t total_q, int32_t num_seqs, int32_t num_q_heads,
                               int32_t num_kv_heads, int32_t max_seqlen_k);

B200_API int b200_paged_attn_fwd(const B200AttnParams* params, void* stream);

/*
 * 1 if b200_paged_attn_fwd runs this head shape and element type, else 0:
 * q/k/v/out F16 or BF16, head_dim 64, 128 or 256, num_q_heads a multiple of
 * num_kv_heads with at most 128 query heads per KV head.  The dispatcher and
 * the service route other shapes to their baseline kernel before calling in,
 * as they route the unsupported features of kernels/attention.py:99-110 and
 * integration/vllm-plugin-FL-split-kv.patch:88-141 (the reference's Triton
 * kernel takes head_dim 64/128/256 and any ratio,
 * kernels/triton_split_kv_paged.py:270-279).
 */
B200_API int32_t b200_attn_shape_supported(int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                           int32_t dtype);

/*
 * b200_paged_attn_fwd without a caller-supplied workspace: no counterpart in
 * the reference.  For callers that cannot allocate device memory at call time
 * (an engine that reserved HBM for its KV cache up front, a foreign-language
 * host without a device allocator, a path where cudaMalloc's implicit device
 * synchronisation is not acceptable).  params->workspace and
 * params->workspace_bytes are ignored; the scratch is one file-scope device
 * array of B200_STATIC_SCRATCH_BYTES, held by every GPU that loads this
 * library until the process exits.  Calls whose scratch need
 * (b200_attn_workspace_bytes) exceeds it fail with B200_ERR_INVALID.  The
 * first call on a device looks up the array's device address (make it before
 * any stream capture) and keeps it for the life of the process: after a
 * cudaDeviceReset (or anything else that destroys the device's primary
 * context) that address is stale, so do not use this entry point across a
 * device reset.  All calls on a device share the array: calls that
 * overlap on the GPU (other streams, other threads) race and must not be
 * issued.  No scratch byte needs to start at zero; every byte a call reads
 * it wrote first.  Allocates nothing.
 */
#define B200_STATIC_SCRATCH_BYTES (32u << 20)
B200_API int b200_paged_attn_fwd_noalloc(const B200AttnParams* params, void* stream);

/*
 * Cross-split combine: out[t,h,:] = sum_s w_s O_s[t,h,:] / max(sum_s w_s, 1e-20),
 * w_s = exp(m_s - max_s m_s) * l_s for l_s > 0, else 0.
 * o_splits [num_splits, total_q, num_heads, head_dim] (F16 / BF16 / F32), m, l
 * [num_splits, total_q, num_heads] F32, out [total_q, num_heads, head_dim]
 * (F16 / BF16 / F32); d contiguous everywhere.
 */
typedef struct B200CombineParams {
  const void* o_splits;
  const float* m_splits;
  const float* l_splits;
  void* out;
  int64_t o_stride_s, o_stride_t, o_stride_h;
  int64_t m_stride_s, m_stride_t, m_stride_h;
  int64_t l_stride_s, l_stride_t, l_stride_h;
  int64_t out_stride_t, out_stride_h;
  int32_t o_dtype;
  int32_t out_dtype;
  int32_t num_splits;
  int32_t total_q;
  int32_t num_heads;
  int32_t head_dim;
} B200CombineParams;

B200_API int b200_split_combine(const B200CombineParams* params, void* stream);

/*
 * Fused RoPE + paged KV-cache write.  query [T, Hq, D] rotated in place;
 * rotate(key) -> key_cache[slot / bs, slot % bs, h, :]; value -> value_cache[...];
 * tokens with slot < 0 skip both cache writes.  cos_sin_cache [max_position,
 * rotary_dim] = [cos(0..rd/2) | sin(0..rd/2)].  Caches [num_blocks, bs, Hkv, D].
 */
typedef struct B200RopeParams {
  void* query;
  const void* key;
  const void* value;
  const void* positions;
  const void* cos_sin_cache;
  void* key_cache;
  void* value_cache;
  const void* slot_mapping;
  int64_t q_stride_t, q_stride_h, q_stride_d;
  int64_t k_stride_t, k_stride_h, k_stride_d;
  int64_t v_stride_t, v_stride_h, v_stride_d;
  int64_t cos_sin_stride_t;
  int64_t cache_stride_block, cache_stride_tok, cache_stride_head, cache_stride_d;
  int32_t num_tokens;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t rotary_dim;
  int32_t block_size;
  int32_t num_blocks;
  int32_t max_position;
  int32_t is_neox;
  int32_t dtype;          /* query / key / value / caches: F16 / BF16 */
  int32_t cos_sin_dtype;  /* F16 / BF16 / F32 */
  int32_t position_dtype; /* I32 / I64 */
  int32_t slot_dtype;     /* I32 / I64 */
  /* Service ABI (vLLM's rope-and-cache call with k_out = key):            */
  void* key_out;          /* NULL: key untouched; else rotated key [T, Hkv, D] stored here
                             for every token (may alias key)                             */
  int64_t ko_stride_t, ko_stride_h;
  int32_t cache_dtype;    /* == dtype, or FP8_E4M3 / FP8_E5M2: caches hold
                             fp8(round_to_dtype(x) / scale), RNE, saturating             */
  const float* k_scale;   /* fp8 caches: one device float each                           */
  const float* v_scale;
} B200RopeParams;

B200_API int b200_rope_kv_write(const B200RopeParams* params, void* stream);

/*
 * Paged KV-cache write (vLLM "flash" layout): for every token t with
 * slot_mapping[t] >= 0, key[t, h, :] -> key_cache[slot / bs, slot % bs, h, :]
 * and value[t, h, :] -> value_cache[...], as
 *   B200_KVQ_NONE                bit copy (cache_dtype == dtype);
 *   B200_KVQ_FP8_PER_TENSOR      fp8(x / *k_scale) (resp. *v_scale), x / s rounded to
 *                                nearest, fp8 round-to-nearest-even, saturating to the
 *                                largest finite value;
 *   B200_KVQ_*_PER_TOKEN_HEAD    s = max(max_d |x| / QMAX, 1e-6) per (token, head),
 *                                q = clamp(x * (1 / s), QMIN, QMAX) -> int8 by truncation
 *                                toward zero (QMAX 127, QMIN -128) or fp8 e4m3 RNE (±448);
 *                                s stored to k_scale_cache / v_scale_cache
 *                                [num_blocks, block_size, num_kv_heads] (float strides).
 * key, value [num_tokens, num_kv_heads, head_dim] (F16 / BF16 / F32), d contiguous;
 * caches [num_blocks, block_size, num_kv_heads, >= head_dim], d contiguous (the
 * per-token-head caches may carry the scale inline after head_dim).  Slots
 * >= num_blocks * block_size are skipped and recorded (B200_DEVERR_SLOT_RANGE).
 * Alignment: key / value rows 16 bytes; cache rows 16 bytes (NONE), 4 bytes (1-byte types).
 */
typedef struct B200KvWriteParams {
  const void* key;
  const void* value;
  void* key_cache;
  void* value_cache;
  const void* slot_mapping;
  const float* k_scale;  /* FP8_PER_TENSOR */
  const float* v_scale;
  float* k_scale_cache;  /* *_PER_TOKEN_HEAD */
  float* v_scale_cache;
  int64_t k_stride_t, k_stride_h;
  int64_t v_stride_t, v_stride_h;
  int64_t kc_stride_block, kc_stride_tok, kc_stride_head;
  int64_t vc_stride_block, vc_stride_tok, vc_stride_head;
  int64_t ks_stride_block, ks_stride_tok, ks_stride_head;
  int64_t vs_stride_block, vs_stride_tok, vs_stride_head;
  int32_t num_tokens;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t block_size;
  int32_t num_blocks;
  int32_t dtype;       /* key / value: F16 / BF16 / F32 */
  int32_t cache_dtype; /* NONE: == dtype; FP8_PER_TENSOR: FP8_E4M3 / FP8_E5M2;
                          INT8_PER_TOKEN_HEAD: I8; FP8_PER_TOKEN_HEAD: FP8_E4M3 */
  int32_t quant_mode;  /* B200_KVQ_* */
  int32_t slot_dtype;  /* I32 / I64 */
} B200KvWriteParams;

B200_API int b200_kv_cache_write(const B200KvWriteParams* params, void* stream);

/*
 * Dequantise the pages a batch references, for attention over a quantised KV
 * cache (the service's fp8 / int8 caches; the reference sends those calls to
 * vLLM's unified_attention, integration/vllm-plugin-FL-split-kv.patch:473-523).
 * For sequence b and page p < ceil(seqused_k[b] / block_size), the cache rows
 * of block_table[b, p] go to dense page b * max_pages + p of out_cache
 * [num_seqs * max_pages, 2 (K, V), block_size, num_kv_heads, head_dim] in
 * out_dtype, and out_block_table[b, p] = b * max_pages + p for every p <
 * max_pages; b200_paged_attn_fwd then runs on out_cache[:, 0] / [:, 1] with
 * out_block_table.  Element values: FP8_PER_TENSOR fp8(x) * *k_scale (resp.
 * *v_scale); *_PER_TOKEN_HEAD x * scale_cache[block, slot, head]; both rounded
 * to nearest in out_dtype.  Cache element types: FP8_E4M3 / FP8_E5M2
 * (per-tensor), I8 / FP8_E4M3 (per-token-head).  Cache strides in elements
 * (bytes), multiples of 4; head_dim a multiple of 4.  A block id outside
 * [0, num_blocks) gives a zero page.
 */
typedef struct B200KvDequantParams {
  const void* key_cache;
  const void* value_cache;
  int64_t kc_stride_block, kc_stride_tok, kc_stride_head;
  int64_t vc_stride_block, vc_stride_tok, vc_stride_head;
  const float* k_scale;        /* FP8_PER_TENSOR */
  const float* v_scale;
  const float* k_scale_cache;  /* *_PER_TOKEN_HEAD, float element strides below */
  const float* v_scale_cache;
  int64_t ks_stride_block, ks_stride_tok, ks_stride_head;
  int64_t vs_stride_block, vs_stride_tok, vs_stride_head;
  const void* block_table;
  int64_t block_table_stride;
  int32_t block_table_cols;
  int32_t block_table_dtype; /* I32 / I64 */
  const void* seqused_k;
  int32_t seqlen_dtype;      /* I32 / I64 */
  void* out_cache;
  int32_t* out_block_table;  /* [num_seqs, max_pages] */
  int32_t num_seqs;
  int32_t max_pages;
  int32_t block_size;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t num_blocks;
  int32_t cache_dtype;       /* FP8_E4M3 / FP8_E5M2 / I8 */
  int32_t quant_mode;        /* B200_KVQ_FP8_PER_TENSOR / _INT8_PER_TOKEN_HEAD / _FP8_PER_TOKEN_HEAD */
  int32_t out_dtype;         /* BF16 / F16 */
} B200KvDequantParams;

B200_API int b200_kv_dequant_pages(const B200KvDequantParams* params, void* stream);

/*
 * The attention operators below and the page operators have no counterpart in
 * the reference.  Device-side lengths, indices and page ids that disagree with
 * the sizes given here never lead outside the caller's buffers.
 */

/* Workspace bytes of b200_prompt_attn_fwd and b200_tree_attn_fwd for these sizes. */
B200_API size_t b200_varlen_attn_workspace_bytes(int32_t total_q, int32_t num_seqs, int32_t num_q_heads,
                                                 int32_t num_kv_heads, int32_t head_dim, int32_t max_seqlen_k);

/*
 * Attention of packed sequences over plain K/V rows (no cache), GQA: query row i
 * of sequence b (rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1]) sees its keys j
 * (rows cu_seqlens_k[b] + j) with j <= Lk - Lq + i (causal), or all Lk of them;
 * a row that sees no key is 0.  Rows of out outside every sequence are left as
 * they were.
 * q, out [total_q, num_q_heads, head_dim]; k, v [total_k, num_kv_heads, head_dim];
 * d contiguous, other strides multiples of 8 elements, pointers 16-byte aligned.
 * F16 / BF16, head_dim 64, 128 or 256, up to 128 query heads per KV head.
 * softmax_scale must be positive and at most 2e38.  max_seqlen_k bounds the longest
 * sequence and only decides how far the keys may be split.
 * Keys and values that some row of the tile sees must be finite; rows of k and v
 * outside every sequence may hold anything.
 * workspace: device buffer of b200_varlen_attn_workspace_bytes(...), 16-byte
 * aligned, not shared by calls that overlap.
 */
typedef struct B200PromptAttnParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const void* cu_seqlens_q; /* [num_seqs + 1] */
  const void* cu_seqlens_k; /* [num_seqs + 1]; may be cu_seqlens_q */
  int64_t q_stride_t, q_stride_h;
  int64_t k_stride_t, k_stride_h;
  int64_t v_stride_t, v_stride_h;
  int64_t out_stride_t, out_stride_h;
  int32_t seqlen_dtype; /* I32 / I64 */
  int32_t dtype;
  int32_t num_seqs;
  int32_t total_q;
  int32_t total_k;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t max_seqlen_k;
  int32_t causal;
  float softmax_scale;
  void* workspace;
  size_t workspace_bytes;
} B200PromptAttnParams;

B200_API int b200_prompt_attn_fwd(const B200PromptAttnParams* params, void* stream);

/*
 * Attention of drafted token trees over a paged cache (speculative decoding).
 * The last n = cu_seqlens_q[b + 1] - cu_seqlens_q[b] keys of sequence b are its
 * drafted tokens (their K/V rows are in the cache already); query row i sees the
 * context, keys [0, seqused_k[b] - n), and drafted key j iff
 * tree_mask[cu_seqlens_q[b] + i, j] is nonzero (columns at or past mask_cols are
 * not seen).  A row that sees no key is 0.  tree_mask: one byte per entry,
 * [total_q, mask_cols], row stride mask_stride.  Everything else as in
 * b200_paged_attn_fwd (the cache layout and its limits) and
 * b200_prompt_attn_fwd (scale, workspace).  Keys and values that some row sees
 * must be finite; drafted tokens that no row sees may hold anything.
 * The batch's units of work (query tile pairs x KV heads, one per sequence and KV
 * head at least) times the KV tiles of a full table row stay below 2^30, or the
 * call is refused: 256 sequences of 8 KV heads with tables of 2^24 keys each pass.
 */
typedef struct B200TreeAttnParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const void* tree_mask;
  const void* block_table;
  const void* cu_seqlens_q;
  const void* seqused_k;
  int64_t q_stride_t, q_stride_h;
  int64_t k_stride_block, k_stride_tok, k_stride_head;
  int64_t v_stride_block, v_stride_tok, v_stride_head;
  int64_t out_stride_t, out_stride_h;
  int64_t mask_stride;
  int64_t block_table_stride;
  int32_t mask_cols;
  int32_t block_table_cols;
  int32_t block_table_dtype; /* I32 / I64 */
  int32_t seqlen_dtype;      /* I32 / I64 */
  int32_t dtype;
  int32_t num_seqs;
  int32_t total_q;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t block_size;
  int32_t num_blocks;
  int32_t max_seqlen_k;
  float softmax_scale;
  void* workspace;
  size_t workspace_bytes;
} B200TreeAttnParams;

B200_API int b200_tree_attn_fwd(const B200TreeAttnParams* params, void* stream);

/*
 * The caches that a page operator works on: the K and V tensors of every layer,
 * [num_blocks, block_size, num_kv_heads, row], of any element type (bytes are
 * moved as they are; rows may carry their scale inline).  All share the shape and
 * the strides (bytes); a page is one dense run, tokens or heads outermost.
 * Pointers, strides and rows are multiples of 4 bytes.  The caches are distinct.
 */
typedef struct B200PageCaches {
  const void* const* base; /* host array of num_caches device pointers, 1 .. 256 */
  int32_t num_caches;
  int32_t num_blocks;
  int32_t block_size;
  int32_t num_kv_heads;
  int64_t row_bytes;
  int64_t stride_block, stride_tok, stride_head;
} B200PageCaches;

/* Block table, lengths and page reference counts of a pool of sequences. */
typedef struct B200SeqTable {
  void* block_table;   /* [max_seqs, cols], row stride in elements, -1 = no page */
  void* seq_lens;      /* [max_seqs] tokens */
  int32_t* ref_counts; /* [num_blocks], 0 = free */
  int64_t stride;
  int32_t cols;
  int32_t max_seqs;
  int32_t num_blocks;
  int32_t block_size;
  int32_t table_dtype;  /* I32 / I64 */
  int32_t seqlen_dtype; /* I32 / I64 */
} B200SeqTable;

/*
 * Page src_pages[i] -> page dst_pages[i] in every cache, i < num_pairs.  A pair
 * with a negative index is skipped (padding); an index past the cache is skipped
 * and recorded (B200_DEVERR_PAGE_RANGE).  A destination may be neither named
 * twice nor a source of another pair: the copies run at the same time.
 */
B200_API int b200_copy_pages(const B200PageCaches* caches, const void* src_pages, const void* dst_pages,
                             int32_t num_pairs, int32_t index_dtype, void* stream);

/*
 * Row children[i] of the table becomes a copy of row parents[i]: full pages are
 * shared (their counts rise by one), the used rows of a partial last page go to a
 * free page of the child's own -- the lowest free ones, in the order of the
 * entries -- and seq_lens[child] = seq_lens[parent].  A child's row must have
 * length 0 and is named once; pages that it names all the same (reserved ones) are
 * released, and are not given out by the same call.  Entries with a negative index
 * are padding.  An entry that cannot be served (a row out of range, in use or named before:
 * B200_DEVERR_SEQ_ROW; no page left: B200_DEVERR_NO_PAGE; a table that names no
 * page for the partial last one: B200_DEVERR_PAGE_RANGE) is recorded and leaves its
 * child as it was.  A full page that the parent's row does not name is missing in the
 * child's row too (-1), and is recorded the same way.
 * workspace: b200_fork_workspace_bytes(num_entries, max_seqs), 16-byte aligned.
 */
B200_API size_t b200_fork_workspace_bytes(int32_t num_entries, int32_t max_seqs);
B200_API int b200_fork_sequences(const B200PageCaches* caches, const B200SeqTable* table, const void* parents,
                                 const void* children, int32_t num_entries, int32_t index_dtype, void* workspace,
                                 size_t workspace_bytes, void* stream);

/*
 * Empties the rows named: every page's count falls by one, the row's entries
 * become -1 and its length 0.  A page whose count reaches 0 is free.  Naming a row
 * twice, or an empty one, releases nothing twice; negative rows are padding.
 */
B200_API int b200_free_sequences(const B200SeqTable* table, const void* rows, int32_t num_rows, int32_t index_dtype,
                                 void* stream);

/*
 * After the verification of drafts: for sequence b and i < num_accepted[b], the
 * K/V row at position context_lens[b] + accepted[b, i] moves to context_lens[b] +
 * i in every cache, and seq_lens[b] = context_lens[b] + num_accepted[b].
 * accepted[b, :num_accepted[b]] rises strictly (an ancestor path of a tree whose
 * parents come first).  With ref_counts, the pages behind the new length are
 * released, and a row is not written into a page that is shared.  A path is cut
 * before its first entry that does not rise (B200_DEVERR_ACCEPT), has no page
 * (B200_DEVERR_PAGE_RANGE) or would write a shared page (B200_DEVERR_PAGE_SHARED).
 * A context that is no length (negative, past 2^30 - 1) is recorded as
 * B200_DEVERR_ACCEPT: the row's length becomes 0 and it keeps its pages.
 * seq_lens is written for every row of the table and overlaps none of context_lens,
 * accepted and num_accepted.
 */
B200_API int b200_keep_accepted(const B200PageCaches* caches, const B200SeqTable* table, const void* context_lens,
                                const void* accepted, int64_t accepted_stride, int32_t most, const void* num_accepted,
                                int32_t index_dtype, void* stream);

/* Message of the last failed call on this host thread ("" if none). */
B200_API const char* b200_last_error(void);

/*
 * Synchronises `stream`, then returns and clears a code that this library's
 * kernels recorded on the current device (B200_DEVERR_*).  Cache writes and paged
 * attention, prompt attention, tree attention and the page operators record apart,
 * the first error of each: further ones are returned by the calls that follow,
 * until one returns B200_DEVERR_NONE.  For tests and debugging; the hot-path calls
 * never synchronise.
 */
B200_API int b200_device_error(void* stream, uint32_t* code);

/*
 * Test hook for the bounded waits (no reference counterpart): launches one
 * warp on `stream` that waits on an mbarrier nothing ever arrives on.  The
 * wait gives up after its limit (2 s of %globaltimer), records
 * B200_DEVERR_WAIT_TIMEOUT and the kernel returns, so the context stays
 * usable; b200_device_error then reports the timeout.  Never faults or hangs.
 */
B200_API int b200_wait_selftest(void* stream);

B200_API int b200_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* MINICPM_B200_H_ */
