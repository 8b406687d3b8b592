// attn_forms.cuh -- launch of the attention kernel's bounded forms
// (kFormPrompt, kFormTree): workspace, split bound, schedule, attention,
// combine of split units.
//
// The form runs paged_attn_fwd_kernel's pipeline; what differs from the causal
// paged call is here and in the kForm branches of that kernel.  Partial outputs
// of split units are fp32, so a split costs no rounding: the result is rounded
// once, when the combine (or the unsplit epilogue) stores it.
#pragma once

#include <algorithm>
#include <atomic>
#include <cstring>

#include "b200_host.h"
#include "paged_attention.cuh"

namespace b200 {

// The most runs one query unit's keys are split into.  A draft batch of one
// sequence has as few as KH units for 148 SMs; 64 runs of at least
// kMinSplitTiles tiles keep every SM busy from 2 KV heads x 16K keys on.
constexpr int kMaxFormSplits = 64;

struct FormCombineArgs {
  const float* o_part;    // [slots][num_splits][kUnitRows][D], normalised
  const float* m_part;    // [slots][num_splits][kUnitRows]
  const float* l_part;
  const int4* split_units;
  const int* unit_count;  // [2] = slots
  const void* cu_q;
  void* out;
  int64_t out_st, out_sh;
  int len_i64, total_q;
  int num_splits, group, pos_per_tile, pos_per_unit;
};

// out = sum_s w_s O_s / sum_s w_s, w_s = exp(m_s - max m) l_s, over the runs of a
// split unit: D / 8 threads a row, the m / l of a row loaded once per group and
// the weights passed by shuffles, four runs' O in flight per thread.  Memory
// bound; a call without split units ends at once.
template <typename T, int D, int kForm>
__global__ void __launch_bounds__(kCombineThreads) form_combine_kernel(const FormCombineArgs a) {
  constexpr int kTpr = D / 8;  // threads per row: 8, 16 or 32, so a warp's rows belong to one unit
  constexpr int kRowsPerBlock = kCombineThreads / kTpr;
  constexpr int kPer = kMaxFormSplits / kTpr;
  griddep_wait();
  const int sub = threadIdx.x % kTpr;
  const int64_t rows = static_cast<int64_t>(a.unit_count[2]) * kUnitRows;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock; base < rows;
       base += static_cast<int64_t>(gridDim.x) * kRowsPerBlock) {
    // rows is a multiple of 256, so every row of the block exists
    const int64_t row = base + threadIdx.x / kTpr;
    const int slot = static_cast<int>(row / kUnitRows);
    const int ur = static_cast<int>(row - static_cast<int64_t>(slot) * kUnitRows);
    const int4 su = a.split_units[slot];  // (seq, qunit, kvh, splits)
    const int t = ur / kAttnTileM, r = ur % kAttnTileM;
    const int q_begin = min(max(load_index(a.cu_q, su.x, a.len_i64), 0), a.total_q);
    const int q_end = min(load_index(a.cu_q, su.x + 1, a.len_i64), a.total_q);
    const int pos = su.y * a.pos_per_unit + t * a.pos_per_tile + r / a.group;
    const bool valid = r < a.group * a.pos_per_tile && t * a.pos_per_tile < a.pos_per_unit && pos < q_end - q_begin;
    if (!__any_sync(0xffffffffu, valid)) continue;
    const int n = su.w;
    const int64_t prow = static_cast<int64_t>(slot) * a.num_splits * kUnitRows + ur;
    float mk[kPer], wk[kPer], m_max = -INFINITY;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int s = sub + k * kTpr;
      const bool has = valid && s < n;
      mk[k] = has ? a.m_part[prow + static_cast<int64_t>(s) * kUnitRows] : -INFINITY;
      wk[k] = has ? a.l_part[prow + static_cast<int64_t>(s) * kUnitRows] : 0.f;
      m_max = fmaxf(m_max, mk[k]);
    }
#pragma unroll
    for (int off = kTpr / 2; off > 0; off >>= 1) m_max = fmaxf(m_max, __shfl_xor_sync(0xffffffffu, m_max, off, kTpr));
    float den = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      // A run in which the row saw no key has l = 0 and its O is left out by
      // selection.  A NaN among the row's scores makes l NaN: it is kept.
      wk[k] = wk[k] != 0.f ? expf(mk[k] - m_max) * wk[k] : -1.f;
      if (!(wk[k] < 0.f)) den += wk[k];
    }
#pragma unroll
    for (int off = kTpr / 2; off > 0; off >>= 1) den += __shfl_xor_sync(0xffffffffu, den, off, kTpr);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const float* o = a.o_part + prow * D + sub * 8;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k * kTpr >= n) break;  // the same in the whole warp
#pragma unroll 1
      for (int j = 0; j < kTpr; j += 4) {
        float w[4];
        float4 x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int s = k * kTpr + j + u;
          w[u] = __shfl_sync(0xffffffffu, wk[k], j + u, kTpr);
          x[u] = y[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (valid && s < n && !(w[u] < 0.f)) {
            const float4* p = reinterpret_cast<const float4*>(o + static_cast<int64_t>(s) * kUnitRows * D);
            x[u] = __ldcs(p);
            y[u] = __ldcs(p + 1);
          } else {
            w[u] = 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          acc[0] = fmaf(w[u], x[u].x, acc[0]);
          acc[1] = fmaf(w[u], x[u].y, acc[1]);
          acc[2] = fmaf(w[u], x[u].z, acc[2]);
          acc[3] = fmaf(w[u], x[u].w, acc[3]);
          acc[4] = fmaf(w[u], y[u].x, acc[4]);
          acc[5] = fmaf(w[u], y[u].y, acc[5]);
          acc[6] = fmaf(w[u], y[u].z, acc[6]);
          acc[7] = fmaf(w[u], y[u].w, acc[7]);
        }
      }
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= inv;
    if (valid) {
      const int64_t tok = q_begin + pos, head = static_cast<int64_t>(su.z) * a.group + r % a.group;
      store8<T>(static_cast<T*>(a.out) + tok * a.out_st + head * a.out_sh + sub * 8, acc);
    }
  }
}

}  // namespace b200

namespace b200_host {

struct FormLayout {
  size_t count_off, tile_base_off, seq_off_off, qbase_off, qsplit_off, qslot_off, units_off, split_units_off;
  size_t o_off, m_off, l_off, total;
  int ppt, ppu, splits;
  int64_t qunits_ub, capacity, slots_ub;
};

// The bound on the splits of a unit: enough runs that the units the batch is
// sure to have give every SM two, each run at least kMinSplitTiles tiles of the
// longest sequence.  The schedule kernel then splits each unit by its share.
inline FormLayout form_layout(int64_t total_q, int num_seqs, int hq, int hkv, int head_dim, int max_seqlen_k,
                              int sms) {
  FormLayout w{};
  const int group = hq / hkv;
  w.ppt = b200::kAttnTileM / group;
  w.ppu = w.ppt * (head_dim == 256 ? 1 : b200::kAttnTilesPerUnit);
  w.qunits_ub = (total_q + w.ppu - 1) / w.ppu + num_seqs;
  const int64_t units_lb =
      std::max<int64_t>((total_q + w.ppu - 1) / w.ppu, std::min<int64_t>(num_seqs, total_q)) * hkv;
  const int64_t most = std::max(max_seqlen_k, 1) / (b200::kMinSplitTiles * b200::kAttnTileN);
  const int64_t want = (2 * (int64_t)sms + units_lb - 1) / std::max<int64_t>(units_lb, 1);
  w.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, most, (int64_t)b200::kMaxFormSplits}));
  w.capacity = w.qunits_ub * hkv * w.splits;
  w.slots_ub = w.splits > 1 ? w.qunits_ub * hkv : 0;
  const size_t qn = (size_t)w.qunits_ub;
  w.count_off = 0;
  w.tile_base_off = 256;
  w.seq_off_off = align_up(w.tile_base_off + sizeof(int) * ((size_t)num_seqs + 1), 256);
  w.qbase_off = align_up(w.seq_off_off + sizeof(int) * (size_t)num_seqs, 256);
  w.qsplit_off = align_up(w.qbase_off + sizeof(int) * (qn + 1), 256);
  w.qslot_off = align_up(w.qsplit_off + sizeof(int) * qn, 256);
  w.units_off = align_up(w.qslot_off + sizeof(int) * qn, 256);
  w.split_units_off = align_up(w.units_off + sizeof(int4) * (size_t)w.capacity, 256);
  w.o_off = align_up(w.split_units_off + sizeof(int4) * (size_t)w.slots_ub, 256);
  const size_t rows = (size_t)w.slots_ub * (w.splits > 1 ? w.splits : 0) * b200::kUnitRows;
  w.m_off = align_up(w.o_off + rows * head_dim * sizeof(float), 256);
  w.l_off = align_up(w.m_off + rows * sizeof(float), 256);
  w.total = align_up(w.l_off + rows * sizeof(float), 256);
  return w;
}

// What a form's entry point hands over: maps and kernel arguments that only it
// knows, the rest is filled in here.
struct FormLaunch {
  CUtensorMap tm_q;
  b200::KvHeadMaps maps;
  b200::AttnKernelArgs a;
  bool head_maps;
  int dtype, num_seqs, num_kv_heads, max_seqlen_k;
  void* workspace;
  size_t workspace_bytes;
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

template <typename... KArgs, typename... Args>
int launch_dependent(const char* what, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                     const Args&... args) {
  // A programmatic dependent of the launch before it: its set-up overlaps that
  // kernel's end, and it waits (griddepcontrol.wait) before it reads its output.
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return check_launch(what);
}

template <typename T, bool kHeadMaps, bool kWide, bool kNarrow, int kForm>
int launch_attn_form(const FormLaunch& f, dim3 grid, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  auto kernel = b200::paged_attn_fwd_kernel<T, kHeadMaps, kWide, kNarrow, kForm>;
  if (int r = prepare_attn_kernel(kernel, done)) return r;
  return launch_dependent("attention kernel", kernel, grid, b200::kAttnThreads, b200::kAttnSmemAlloc, s, f.tm_q, f.maps,
                          f.a);
}

template <typename T, bool kHeadMaps, int kForm>
int launch_attn_dim(const FormLaunch& f, dim3 grid, cudaStream_t s) {
  if (f.a.head_dim == 256) return launch_attn_form<T, kHeadMaps, true, false, kForm>(f, grid, s);
  if (f.a.head_dim == 64) return launch_attn_form<T, kHeadMaps, false, true, kForm>(f, grid, s);
  return launch_attn_form<T, kHeadMaps, false, false, kForm>(f, grid, s);
}

template <typename T, int kForm>
int launch_combine(const b200::FormCombineArgs& c, int head_dim, int64_t rows, int sms, cudaStream_t s) {
  const int rows_per_block = b200::kCombineThreads / (head_dim / 8);
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((rows + rows_per_block - 1) / rows_per_block, (int64_t)sms * 8));
  auto kernel = head_dim == 256  ? b200::form_combine_kernel<T, 256, kForm>
                : head_dim == 64 ? b200::form_combine_kernel<T, 64, kForm>
                                 : b200::form_combine_kernel<T, 128, kForm>;
  return launch_dependent("form_combine_kernel", kernel, dim3((unsigned)blocks), b200::kCombineThreads, 0, s, c);
}

template <int kForm>
int run_form(FormLaunch& f, cudaStream_t s) {
  b200::AttnKernelArgs& a = f.a;
  const int sms = sm_count();
  const FormLayout w = form_layout(a.total_q, f.num_seqs, a.num_q_heads, f.num_kv_heads, a.head_dim, f.max_seqlen_k, sms);
  if (w.capacity > 0x7fffffff) return fail(B200_ERR_UNSUPPORTED, "more than 2^31 work units in one call");
  if (!f.workspace || f.workspace_bytes < w.total)
    return fail(B200_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", w.total, f.workspace_bytes);
  if (!aligned16(f.workspace)) return fail(B200_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(f.workspace);

  b200::SchedArgs sa{};
  sa.cu_q = a.cu_q;
  sa.seqused = a.seqused;
  sa.cu_k = a.cu_k;
  sa.len_i64 = a.len_i64;
  sa.num_seqs = f.num_seqs;
  sa.pos_per_unit = w.ppu;
  sa.num_kv_heads = f.num_kv_heads;
  sa.num_splits = w.splits;
  sa.num_sms = sms;
  sa.capacity = (int)w.capacity;
  sa.total_q = a.total_q;
  sa.total_k = a.total_k;
  sa.bt_cols = a.bt_cols;
  sa.block_size = a.block_size;
  sa.max_qunits = (int)w.qunits_ub;
  sa.full = a.full;
  sa.tile_base = reinterpret_cast<int*>(ws + w.tile_base_off);
  sa.seq_off = reinterpret_cast<int*>(ws + w.seq_off_off);
  sa.qunit_base = reinterpret_cast<int*>(ws + w.qbase_off);
  sa.qunit_split = reinterpret_cast<int*>(ws + w.qsplit_off);
  sa.qunit_slot = reinterpret_cast<int*>(ws + w.qslot_off);
  sa.units = reinterpret_cast<int4*>(ws + w.units_off);
  sa.split_units = reinterpret_cast<int4*>(ws + w.split_units_off);
  sa.unit_count = reinterpret_cast<int*>(ws + w.count_off);
  auto sched = b200::attn_schedule_kernel<kForm>;
  cudaError_t e = cudaFuncSetAttribute(sched, cudaFuncAttributeMaxDynamicSharedMemorySize, b200::kSchedSmemBytes);
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "schedule kernel shared memory: %s", cudaGetErrorString(e));
  sched<<<1, b200::kSchedThreads, b200::kSchedSmemBytes, s>>>(sa);
  if (int r = check_launch("attn_schedule_kernel")) return r;

  a.o_split = ws + w.o_off;
  a.m_split = reinterpret_cast<float*>(ws + w.m_off);
  a.l_split = reinterpret_cast<float*>(ws + w.l_off);
  a.units = sa.units;
  a.unit_count = sa.unit_count;
  a.pos_per_tile = w.ppt;
  a.num_splits = w.splits;
  const dim3 grid((unsigned)std::min<int64_t>(w.capacity, sms));
  const bool bf16 = f.dtype == B200_DTYPE_BF16;
  int r;
  if constexpr (kForm == b200::kFormPrompt) {
    r = bf16 ? launch_attn_dim<__nv_bfloat16, false, kForm>(f, grid, s) : launch_attn_dim<__half, false, kForm>(f, grid, s);
  } else if (f.head_maps) {
    r = bf16 ? launch_attn_dim<__nv_bfloat16, true, kForm>(f, grid, s) : launch_attn_dim<__half, true, kForm>(f, grid, s);
  } else {
    r = bf16 ? launch_attn_dim<__nv_bfloat16, false, kForm>(f, grid, s) : launch_attn_dim<__half, false, kForm>(f, grid, s);
  }
  if (r != B200_OK || w.splits == 1) return r;

  b200::FormCombineArgs c{};
  c.o_part = static_cast<const float*>(a.o_split);
  c.m_part = a.m_split;
  c.l_part = a.l_split;
  c.split_units = sa.split_units;
  c.unit_count = sa.unit_count;
  c.cu_q = a.cu_q;
  c.out = a.out;
  c.out_st = a.out_st;
  c.out_sh = a.out_sh;
  c.len_i64 = a.len_i64;
  c.total_q = a.total_q;
  c.num_splits = w.splits;
  c.group = a.group;
  c.pos_per_tile = w.ppt;
  c.pos_per_unit = w.ppu;
  const int64_t rows = w.slots_ub * b200::kUnitRows;
  return bf16 ? launch_combine<__nv_bfloat16, kForm>(c, a.head_dim, rows, sms, s)
              : launch_combine<__half, kForm>(c, a.head_dim, rows, sms, s);
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
  // The running maximum is taken over unscaled scores, so the scale keeps their order.
  if (!(p.scale > 0.f) || p.scale > 3.0e38f) return fail(B200_ERR_INVALID, "softmax_scale must be positive and finite");
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
