// b200_prompt.cu -- b200_prompt_attn_fwd: packed attention over plain K/V rows.
#include <cudaTypedefs.h>

#include "attn_forms.cuh"
#include "minicpm_b200.h"

using namespace b200_host;

namespace b200_host {

cudaError_t prompt_error_word(void** word) { return cudaGetSymbolAddress(word, b200::g_device_error); }

}  // namespace b200_host

extern "C" {

size_t b200_varlen_attn_workspace_bytes(int32_t total_q, int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                                        int32_t head_dim, int32_t max_seqlen_k) {
  if (total_q <= 0 || num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads > b200::kAttnTileM || head_dim <= 0)
    return 0;
  const int sms = sm_count();
  return std::max(form_layout(true, total_q, num_seqs, num_q_heads, num_kv_heads, head_dim, max_seqlen_k, sms).total,
                  form_layout(false, total_q, num_seqs, num_q_heads, num_kv_heads, head_dim, max_seqlen_k, sms).total);
}

int b200_prompt_attn_fwd(const B200PromptAttnParams* p, void* stream) {
  if (!p) return fail(B200_ERR_INVALID, "null params");
  const FormShape shape{p->q, p->k, p->v, p->out, p->q_stride_t, p->q_stride_h, p->out_stride_t, p->out_stride_h,
                        p->dtype, p->seqlen_dtype, p->num_seqs, p->total_q, p->num_q_heads, p->num_kv_heads,
                        p->head_dim, p->softmax_scale};
  if (int r = check_form(shape)) return r;
  if (p->total_k < 0) return fail(B200_ERR_INVALID, "bad sizes");
  if (p->total_q == 0 || p->num_seqs == 0) return B200_OK;
  if (((p->k_stride_t | p->k_stride_h | p->v_stride_t | p->v_stride_h) * 2) & 15)
    return fail(B200_ERR_UNSUPPORTED, "token/head strides must be multiples of 16 bytes");

  const int group = p->num_q_heads / p->num_kv_heads, ppt = b200::kAttnTileM / group;
  const int sms = sm_count();
  const int ppu = ppt * (p->head_dim == 256 ? 1 : b200::kAttnTilesPerUnit);
  const int64_t max_tiles = (int64_t)p->total_k / b200::kAttnTileN + 1;
  auto layout = [&](bool streamed) {
    return form_layout(streamed, p->total_q, p->num_seqs, p->num_q_heads, p->num_kv_heads, p->head_dim, p->max_seqlen_k, sms);
  };
  FormLayout w = layout(stream_prompt(p->total_q, p->total_k, p->num_seqs, ppu, p->num_kv_heads, p->max_seqlen_k,
                                      p->causal != 0, sms));
  if (w.streamed && !ticks_fit(w, max_tiles)) w = layout(false);
  if (int r = check_layout(w, max_tiles, p->workspace, p->workspace_bytes)) return r;

  FormLaunch f{};
  if (int r = encode_rows(&f.tm_q, p->dtype, p->q, p->head_dim, p->num_q_heads, p->total_q, p->q_stride_t,
                          p->q_stride_h, group, ppt, "q"))
    return r;
  if (p->total_k > 0) {
    if (int r = encode_rows(&f.maps.k[0], p->dtype, p->k, p->head_dim, p->num_kv_heads, p->total_k, p->k_stride_t,
                            p->k_stride_h, 1, b200::kAttnTileN, "k"))
      return r;
    if (int r = encode_rows(&f.maps.v[0], p->dtype, p->v, p->head_dim, p->num_kv_heads, p->total_k, p->v_stride_t,
                            p->v_stride_h, 1, b200::kAttnTileN, "v"))
      return r;
  } else {  // no key anywhere: no tile is loaded, but the kernel prefetches the descriptors
    f.maps.k[0] = f.maps.v[0] = f.tm_q;
  }
  f.dtype = p->dtype;
  f.num_seqs = p->num_seqs;
  f.num_kv_heads = p->num_kv_heads;
  f.workspace = p->workspace;
  b200::AttnKernelArgs& a = f.a;
  a.cu_q = p->cu_seqlens_q;
  a.cu_k = p->cu_seqlens_k;
  a.out = p->out;
  a.out_st = p->out_stride_t;
  a.out_sh = p->out_stride_h;
  a.len_i64 = p->seqlen_dtype == B200_DTYPE_I64;
  a.total_q = p->total_q;
  a.total_k = p->total_k;
  a.num_q_heads = p->num_q_heads;
  a.group = group;
  a.head_dim = p->head_dim;
  a.block_size = 1;
  a.full = p->causal ? 0 : 1;
  a.scale_log2 = static_cast<float>(static_cast<double>(p->softmax_scale) * 1.4426950408889634);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return w.streamed ? run_form<b200::kFormPromptStream>(f, w, sms, s) : run_form<b200::kFormPrompt>(f, w, sms, s);
}

}  // extern "C"
