// b200_tree.cu -- b200_tree_attn_fwd: drafted token trees over a paged cache.
#include <cudaTypedefs.h>

#include "attn_forms.cuh"
#include "minicpm_b200.h"

using namespace b200_host;

namespace b200_host {

cudaError_t tree_error_word(void** word) { return cudaGetSymbolAddress(word, b200::g_device_error); }

namespace {

// Keys per TMA box: the largest power of two, 16 to 128, that divides the page.
int slice_keys(int block_size) {
  int s = 16;
  while (s < b200::kAttnTileN && block_size % (2 * s) == 0) s *= 2;
  return s;
}

// K/V maps of a paged cache [num_blocks, block_size, KH, D]: one 5-D map per KV
// head (a slice with both halves, 4 KB a box at 16 keys) for up to kMaxHeadMaps
// heads, else one 4-D map (one half a box); the layouts are those of the paged form.
int encode_pages(const B200TreeAttnParams* p, const void* base, int64_t sb, int64_t st, int64_t sh, bool head_maps,
                 int slice, CUtensorMap* maps, const char* what) {
  if (p->num_blocks == 1) sb = (int64_t)p->block_size * st;
  if (p->num_kv_heads == 1) sh = p->head_dim;
  if (!head_maps) {
    const cuuint64_t dims[4] = {(cuuint64_t)p->head_dim, (cuuint64_t)p->block_size, (cuuint64_t)p->num_kv_heads,
                                (cuuint64_t)p->num_blocks};
    const cuuint64_t strides[3] = {(cuuint64_t)(st * 2), (cuuint64_t)(sh * 2), (cuuint64_t)(sb * 2)};
    const cuuint32_t box[4] = {64, (cuuint32_t)slice, 1, 1};
    return encode_map(&maps[0], map_type(p->dtype), 4, base, dims, strides, box, what);
  }
  const cuuint64_t dims[5] = {64, 8, (cuuint64_t)(p->head_dim / 64), (cuuint64_t)(p->block_size / 8),
                              (cuuint64_t)p->num_blocks};
  const cuuint64_t strides[4] = {(cuuint64_t)(st * 2), 128, (cuuint64_t)(8 * st * 2), (cuuint64_t)(sb * 2)};
  const cuuint32_t box[5] = {64, 8, (cuuint32_t)std::min(2, p->head_dim / 64), (cuuint32_t)(slice / 8), 1};
  for (int h = 0; h < p->num_kv_heads; ++h)
    if (int r = encode_map(&maps[h], map_type(p->dtype), 5, static_cast<const uint8_t*>(base) + (int64_t)h * sh * 2, dims,
                           strides, box, what))
      return r;
  return B200_OK;
}

}  // namespace
}  // namespace b200_host

extern "C" {

int b200_tree_attn_fwd(const B200TreeAttnParams* p, void* stream) {
  if (!p) return fail(B200_ERR_INVALID, "null params");
  const FormShape shape{p->q, p->k, p->v, p->out, p->q_stride_t, p->q_stride_h, p->out_stride_t, p->out_stride_h,
                        p->dtype, p->seqlen_dtype, p->num_seqs, p->total_q, p->num_q_heads, p->num_kv_heads,
                        p->head_dim, p->softmax_scale};
  if (int r = check_form(shape)) return r;
  if (p->block_size <= 0 || p->block_size % 16) return fail(B200_ERR_INVALID, "the page size must be a multiple of 16");
  if (p->num_blocks <= 0 || p->block_table_cols <= 0 || p->mask_cols < 0) return fail(B200_ERR_INVALID, "bad sizes");
  if (p->block_table_dtype != B200_DTYPE_I32 && p->block_table_dtype != B200_DTYPE_I64)
    return fail(B200_ERR_INVALID, "block_table must contain integer physical block ids");
  if (p->total_q == 0 || p->num_seqs == 0) return B200_OK;
  if (!p->tree_mask) return fail(B200_ERR_INVALID, "null tree_mask");
  if (((p->k_stride_block | p->k_stride_tok | p->k_stride_head | p->v_stride_block | p->v_stride_tok |
        p->v_stride_head) * 2) & 15)
    return fail(B200_ERR_UNSUPPORTED, "token/head/block strides must be multiples of 16 bytes");

  const int sms = sm_count();
  const FormLayout w = form_layout(true, p->total_q, p->num_seqs, p->num_q_heads, p->num_kv_heads, p->head_dim,
                                   p->max_seqlen_k, sms);
  const int64_t max_tiles = (int64_t)p->block_table_cols * p->block_size / b200::kAttnTileN + 1;
  if (int r = check_layout(w, max_tiles, p->workspace, p->workspace_bytes)) return r;

  FormLaunch f{};
  const int group = p->num_q_heads / p->num_kv_heads, ppt = b200::kAttnTileM / group;
  if (int r = encode_rows(&f.tm_q, p->dtype, p->q, p->head_dim, p->num_q_heads, p->total_q, p->q_stride_t,
                          p->q_stride_h, group, ppt, "q"))
    return r;
  f.head_maps = p->num_kv_heads <= b200::kMaxHeadMaps;
  const int slice = slice_keys(p->block_size);
  if (int r = encode_pages(p, p->k, p->k_stride_block, p->k_stride_tok, p->k_stride_head, f.head_maps, slice, f.maps.k, "k"))
    return r;
  if (int r = encode_pages(p, p->v, p->v_stride_block, p->v_stride_tok, p->v_stride_head, f.head_maps, slice, f.maps.v, "v"))
    return r;
  f.dtype = p->dtype;
  f.num_seqs = p->num_seqs;
  f.num_kv_heads = p->num_kv_heads;
  f.workspace = p->workspace;
  b200::AttnKernelArgs& a = f.a;
  a.block_table = p->block_table;
  a.cu_q = p->cu_seqlens_q;
  a.seqused = p->seqused_k;
  a.out = p->out;
  a.bt_stride = p->block_table_stride;
  a.out_st = p->out_stride_t;
  a.out_sh = p->out_stride_h;
  a.bt_cols = p->block_table_cols;
  a.bt_i64 = p->block_table_dtype == B200_DTYPE_I64;
  a.len_i64 = p->seqlen_dtype == B200_DTYPE_I64;
  a.total_q = p->total_q;
  a.num_q_heads = p->num_q_heads;
  a.group = group;
  a.block_size = p->block_size;
  a.slice = slice;
  a.num_blocks = p->num_blocks;
  a.head_dim = p->head_dim;
  a.tree_mask = static_cast<const uint8_t*>(p->tree_mask);
  a.mask_stride = p->mask_stride;
  a.mask_cols = p->mask_cols;
  a.full = 1;
  a.scale_log2 = static_cast<float>(static_cast<double>(p->softmax_scale) * 1.4426950408889634);
  return run_form<b200::kFormTree>(f, w, sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
