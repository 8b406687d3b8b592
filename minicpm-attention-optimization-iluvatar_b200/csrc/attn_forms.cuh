// attn_forms.cuh -- launch of the attention kernel's bounded forms
// (kFormPrompt, kFormTree): workspace, division of the work, attention, join of
// shared units.
//
// The form runs paged_attn_fwd_kernel's pipeline; what differs from the causal
// paged call is here and in the kForm branches of that kernel.  Partial outputs
// of shared units are fp32, so sharing costs no rounding: the result is rounded
// once, when the join (or the epilogue of a whole unit) stores it.
#pragma once

#include <algorithm>
#include <atomic>
#include <cstring>

#include "b200_host.h"
#include "paged_attention.cuh"
#include "stream_combine.cuh"

namespace b200_host {

struct FormLayout {
  bool streamed, shares;  // shares: a unit may be shared by CTAs
  int ctas, ppt, ppu;
  int64_t qunits_ub, capacity;
  // streamed: the CTAs' shared units come first, then their partials
  size_t o_off, m_off, l_off;
  // listed: the unit count comes first, then the schedule kernel's arrays
  size_t tile_base_off, seq_off_off, qbase_off, qsplit_off, qslot_off, units_off;
  size_t total;
};

// Whole units that the batch is sure to have: as many as its query rows fill, and one
// for each sequence at least.
inline int64_t sure_units(int64_t total_q, int num_seqs, int ppu, int hkv) {
  return std::max<int64_t>((total_q + ppu - 1) / ppu, std::min<int64_t>(num_seqs, total_q)) * hkv;
}

// Draft trees are always streamed.  Prompts are where whole units would leave SMs
// idle: fewer units than SMs, or few rounds of long units that are all alike
// (bidirectional, or queries over longer prefixes) and fill the last round badly.
// Elsewhere the list wins, whose dynamic claims balance the unequal units of causal
// prompts and which writes no partials.  Listed / streamed, 16 query and 2 KV heads
// of 128: 2 x 8192 causal (6.9 rounds) 475 / 593 us, 1 x 4096 causal 82 / 110 us, 33
// sequences of up to 517 x 12 heads of 64 bidirectional 51 / 74 us; 8 x 512 over 8192
// (1.7 rounds) 311 / 293 us, 4 x 2048 over 14000 (3.5) 1027 / 943 us, 2 x 4096 x 12
// heads bidirectional (2.6) 206 / 196 us, but 16 x 1024 over 4096 (6.9) 552 / 599 us.
constexpr int kStreamRounds = 8;
constexpr int kStreamLongTiles = 32;

inline bool stream_prompt(int64_t total_q, int64_t total_k, int num_seqs, int ppu, int hkv, int max_seqlen_k, bool causal,
                          int sms) {
  const int64_t units = sure_units(total_q, num_seqs, ppu, hkv);
  if (units < sms) return true;
  const bool alike = !causal || total_k >= 2 * total_q;
  const int64_t rounds = (units + sms - 1) / sms;
  return alike && rounds <= kStreamRounds && max_seqlen_k >= kStreamLongTiles * b200::kAttnTileN &&
         10 * rounds * sms > 11 * units;  // the last round leaves more than a tenth idle
}

inline FormLayout form_layout(bool streamed, int64_t total_q, int num_seqs, int hq, int hkv, int head_dim,
                              int max_seqlen_k, int sms) {
  FormLayout w{};
  const int group = hq / hkv;
  w.ppt = b200::kAttnTileM / group;
  w.ppu = w.ppt * (head_dim == 256 ? 1 : b200::kAttnTilesPerUnit);
  w.qunits_ub = (total_q + w.ppu - 1) / w.ppu + num_seqs;
  w.capacity = w.qunits_ub * hkv;
  const int64_t tiles = std::max(max_seqlen_k, 0) / b200::kAttnTileN + 1;
  const int64_t ticks = w.capacity * (b200::kStreamOverhead + 2 * tiles);
  w.streamed = streamed;
  w.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(w.streamed ? ticks / b200::kStreamMinTicks : w.capacity, sms));
  // No unit as long as two pieces (by the caller's bound): none is shared, and there
  // is nothing to join.
  w.shares = w.streamed && w.ctas > 1 && tiles >= 2 * b200::kStreamMinTiles;
  if (w.streamed) {
    const size_t rows = w.shares ? (size_t)2 * w.ctas * b200::kUnitRows : 0;
    w.o_off = align_up(sizeof(int4) * (size_t)w.ctas, 256);
    w.m_off = w.o_off + rows * head_dim * sizeof(float);
    w.l_off = w.m_off + rows * sizeof(float);
    w.total = w.l_off + rows * sizeof(float);
    return w;
  }
  const size_t qn = (size_t)w.qunits_ub;
  w.tile_base_off = 256;
  w.seq_off_off = align_up(w.tile_base_off + sizeof(int) * ((size_t)num_seqs + 1), 256);
  w.qbase_off = align_up(w.seq_off_off + sizeof(int) * (size_t)num_seqs, 256);
  w.qsplit_off = align_up(w.qbase_off + sizeof(int) * (qn + 1), 256);
  w.qslot_off = align_up(w.qsplit_off + sizeof(int) * qn, 256);
  w.units_off = align_up(w.qslot_off + sizeof(int) * qn, 256);
  w.total = align_up(w.units_off + sizeof(int4) * (size_t)w.capacity, 256);
  return w;
}

// Streamed shares count ticks in 32 bits: no batch of these sizes may reach 2^31 of
// them, even if one sequence has every key (max_tiles KV tiles).  Prompts that could
// take the list, which counts units.
inline bool ticks_fit(const FormLayout& w, int64_t max_tiles) {
  return w.capacity <= 0x7fffffff / (b200::kStreamOverhead + 2 * max_tiles);
}

// The limits of a layout, before anything is done on the GPU.
inline int check_layout(const FormLayout& w, int64_t max_tiles, const void* workspace, size_t workspace_bytes) {
  if (w.capacity > 0x7fffffff) return fail(B200_ERR_UNSUPPORTED, "more than 2^31 units of work in one call");
  if (w.streamed && !ticks_fit(w, max_tiles))
    return fail(B200_ERR_UNSUPPORTED, "units of work (%lld) times their KV tiles (up to %lld) pass 2^30 in one call",
                (long long)w.capacity, (long long)max_tiles);
  if (!workspace || workspace_bytes < w.total)
    return fail(B200_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", w.total, workspace_bytes);
  if (!aligned16(workspace)) return fail(B200_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  return B200_OK;
}

// What a form's entry point hands over: maps and kernel arguments that only it
// knows, the rest is filled in here.
struct FormLaunch {
  CUtensorMap tm_q;
  b200::KvHeadMaps maps;
  b200::AttnKernelArgs a;
  bool head_maps;
  int dtype, num_seqs, num_kv_heads;
  void* workspace;  // checked (check_layout)
};

// Once per kernel and device: the register count that the kernel's setmaxnreg
// split adds up to, and its shared memory.
template <typename Kernel>
int prepare_attn_kernel(Kernel kernel, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return B200_OK;
  cudaFuncAttributes fa{};
  e = cudaFuncGetAttributes(&fa, kernel);
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "attention kernel: %s", cudaGetErrorString(e));
  if (fa.numRegs != b200::kAttnLaunchRegs)
    return fail(B200_ERR_CUDA, "attention kernel built with %d registers per thread, %d expected", fa.numRegs,
                b200::kAttnLaunchRegs);
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, b200::kAttnSmemAlloc);
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "attention kernel shared memory: %s", cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_release);
  return B200_OK;
}

template <typename T, bool kHeadMaps, bool kWide, bool kNarrow, int kForm>
int launch_attn_form(const FormLaunch& f, dim3 grid, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  auto kernel = b200::paged_attn_fwd_kernel<T, kHeadMaps, kWide, kNarrow, kForm>;
  if (int r = prepare_attn_kernel(kernel, done)) return r;
  return launch_form_kernel("attention kernel", !b200::form_streamed(kForm), kernel, grid, b200::kAttnThreads,
                            b200::kAttnSmemAlloc, s, f.tm_q, f.maps, f.a);
}

template <typename T, bool kHeadMaps, int kForm>
int launch_attn_dim(const FormLaunch& f, dim3 grid, cudaStream_t s) {
  if (f.a.head_dim == 256) return launch_attn_form<T, kHeadMaps, true, false, kForm>(f, grid, s);
  if (f.a.head_dim == 64) return launch_attn_form<T, kHeadMaps, false, true, kForm>(f, grid, s);
  return launch_attn_form<T, kHeadMaps, false, false, kForm>(f, grid, s);
}

// The work list of kFormPrompt.
template <int kForm>
int launch_schedule(const FormLaunch& f, const FormLayout& w, int sms, cudaStream_t s) {
  const b200::AttnKernelArgs& a = f.a;
  uint8_t* ws = static_cast<uint8_t*>(f.workspace);
  b200::SchedArgs sa{};
  sa.cu_q = a.cu_q;
  sa.seqused = a.seqused;
  sa.cu_k = a.cu_k;
  sa.len_i64 = a.len_i64;
  sa.num_seqs = f.num_seqs;
  sa.pos_per_unit = w.ppu;
  sa.num_kv_heads = f.num_kv_heads;
  sa.num_splits = 1;
  sa.num_sms = sms;
  sa.capacity = (int)w.capacity;
  sa.total_q = a.total_q;
  sa.total_k = a.total_k;
  sa.max_qunits = (int)w.qunits_ub;
  sa.full = a.full;
  sa.tile_base = reinterpret_cast<int*>(ws + w.tile_base_off);
  sa.seq_off = reinterpret_cast<int*>(ws + w.seq_off_off);
  sa.qunit_base = reinterpret_cast<int*>(ws + w.qbase_off);
  sa.qunit_split = reinterpret_cast<int*>(ws + w.qsplit_off);
  sa.qunit_slot = reinterpret_cast<int*>(ws + w.qslot_off);
  sa.units = reinterpret_cast<int4*>(ws + w.units_off);
  sa.unit_count = reinterpret_cast<int*>(ws);
  auto sched = b200::attn_schedule_kernel<kForm>;
  cudaError_t e = cudaFuncSetAttribute(sched, cudaFuncAttributeMaxDynamicSharedMemorySize, b200::kSchedSmemBytes);
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "schedule kernel shared memory: %s", cudaGetErrorString(e));
  sched<<<1, b200::kSchedThreads, b200::kSchedSmemBytes, s>>>(sa);
  return check_launch("attn_schedule_kernel");
}

// `w` lies in the workspace.
template <int kForm>
int run_form(FormLaunch& f, const FormLayout& w, int sms, cudaStream_t s) {
  b200::AttnKernelArgs& a = f.a;
  uint8_t* ws = static_cast<uint8_t*>(f.workspace);
  a.pos_per_tile = w.ppt;
  a.num_seqs = f.num_seqs;
  a.num_kv_heads = f.num_kv_heads;
  a.num_splits = 1;
  a.wide_out = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_st * 2) | (uintptr_t)(a.out_sh * 2)) & 31) == 0;
  a.min_piece = w.shares ? b200::kStreamMinTiles : 0x3fffffff;
  if constexpr (b200::form_streamed(kForm)) {
    a.stream_meta = reinterpret_cast<int4*>(ws);
    a.o_split = ws + w.o_off;
    a.m_split = reinterpret_cast<float*>(ws + w.m_off);
    a.l_split = reinterpret_cast<float*>(ws + w.l_off);
  } else {
    a.units = reinterpret_cast<int4*>(ws + w.units_off);
    a.unit_count = reinterpret_cast<int*>(ws);
    if (int r = launch_schedule<kForm>(f, w, sms, s)) return r;
  }
  const dim3 grid((unsigned)w.ctas);
  const bool bf16 = f.dtype == B200_DTYPE_BF16;
  int r;
  constexpr bool kMaps = !b200::form_rows(kForm);
  if (kMaps && f.head_maps)
    r = bf16 ? launch_attn_dim<__nv_bfloat16, kMaps, kForm>(f, grid, s) : launch_attn_dim<__half, kMaps, kForm>(f, grid, s);
  else
    r = bf16 ? launch_attn_dim<__nv_bfloat16, false, kForm>(f, grid, s) : launch_attn_dim<__half, false, kForm>(f, grid, s);
  if (r != B200_OK || !w.shares) return r;

  if constexpr (b200::form_streamed(kForm)) {
    b200::StreamCombineArgs c{};
    c.meta = a.stream_meta;
    c.o_part = static_cast<const float*>(a.o_split);
    c.m_part = a.m_split;
    c.l_part = a.l_split;
    c.cu_q = a.cu_q;
    c.out = a.out;
    c.out_st = a.out_st;
    c.out_sh = a.out_sh;
    c.len_i64 = a.len_i64;
    c.total_q = a.total_q;
    c.group = a.group;
    c.pos_per_tile = w.ppt;
    c.pos_per_unit = w.ppu;
    r = launch_stream_combine(c, f.dtype, a.head_dim, w.ctas, s);
  }
  return r;
}

// Checks that both forms share: element type, head shape, alignment, scale.
struct FormShape {
  const void *q, *k, *v, *out;
  int64_t q_st, q_sh, out_st, out_sh;
  int dtype, seqlen_dtype, num_seqs, total_q, hq, hkv, head_dim;
  float scale;
};

inline int check_form(const FormShape& p) {
  if (p.dtype != B200_DTYPE_BF16 && p.dtype != B200_DTYPE_F16)
    return fail(B200_ERR_UNSUPPORTED, "q/k/v/out must be bf16 or f16 for the sm_100a kernel");
  if (p.hq <= 0 || p.hkv <= 0 || p.hq % p.hkv || (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256))
    return fail(B200_ERR_INVALID, "unsupported head shape (head_dim 64, 128 or 256, query heads a multiple of KV heads)");
  if (p.hq / p.hkv > b200::kAttnTileM)
    return fail(B200_ERR_UNSUPPORTED, "query heads per KV head (%d) must be at most 128", p.hq / p.hkv);
  if (p.hkv > 65535) return fail(B200_ERR_UNSUPPORTED, "at most 65535 KV heads");
  if (p.seqlen_dtype != B200_DTYPE_I32 && p.seqlen_dtype != B200_DTYPE_I64)
    return fail(B200_ERR_INVALID, "sequence lengths must be int32 or int64");
  if (p.num_seqs < 0 || p.total_q < 0) return fail(B200_ERR_INVALID, "bad sizes");
  // The running maximum is taken over unscaled scores, so the scale keeps their order;
  // times log2(e) it is finite (2.36e38 would not be), or scores of 0 would give NaN.
  if (!(p.scale > 0.f) || p.scale > 2.0e38f) return fail(B200_ERR_INVALID, "softmax_scale must be positive and at most 2e38");
  if (p.total_q == 0 || p.num_seqs == 0) return B200_OK;
  if (!aligned16(p.q) || !aligned16(p.k) || !aligned16(p.v) || !aligned16(p.out))
    return fail(B200_ERR_UNSUPPORTED, "q, k, v and out must be 16-byte aligned");
  if (((p.q_st | p.q_sh | p.out_st | p.out_sh) * 2) & 15)
    return fail(B200_ERR_UNSUPPORTED, "token/head strides must be multiples of 16 bytes");
  return B200_OK;
}

inline CUtensorMapDataType map_type(int dtype) {
  return dtype == B200_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// [rows, heads, head_dim] with a box of 64 columns x box_heads x box_rows.  A
// dimension of one element takes any stride: the map gets a packed one.
inline int encode_rows(CUtensorMap* map, int dtype, const void* base, int head_dim, int heads, int64_t rows, int64_t st,
                       int64_t sh, int box_heads, int box_rows, const char* what) {
  if (heads == 1) sh = head_dim;
  if (rows == 1) st = (int64_t)heads * sh;
  const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)(sh * 2), (cuuint64_t)(st * 2)};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  return encode_map(map, map_type(dtype), 3, base, dims, strides, box, what);
}

}  // namespace b200_host
