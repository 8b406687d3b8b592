// kv_pages.cuh -- page operators of a paged KV cache: copy, fork, free, and the
// accepted rows of a draft moved together.
//
// A cache set is a list of tensors [num_blocks, block_size, KH, row] (the K and
// the V tensor of every layer) with the same strides, so one launch serves a
// whole model.  All four are bandwidth kernels without arithmetic: bytes moved =
// 2 x the rows copied, and the small calls are bound by launch latency, which is
// why every layer goes in one launch and the bookkeeping of a fork is one block.
// Index order that atomics could disturb decides nothing: pages are given out
// lowest first in the order of the entries, and reference counts are sums.
#pragma once

#include "paged_attention.cuh"

namespace b200 {

constexpr int kMaxCaches = 256;  // K and V of up to 128 layers, passed as kernel parameters (2 KB)
constexpr int kPageThreads = 256;
constexpr int kForkThreads = 1024;

struct PageCacheSet {
  uint8_t* base[kMaxCaches];
};

struct PageShape {  // bytes unless said otherwise
  int64_t stride_block, stride_tok, seg_stride;
  int page_bytes;   // one page, dense
  int seg_bytes;    // contiguous bytes of a token's row
  int segs;         // such pieces per token (1 when the heads are adjacent, else KH)
  int block_size;   // tokens
  int num_blocks;   // pages
  int num_caches;
};

__device__ __forceinline__ int64_t load_index64(const void* p, int64_t i, int is_i64) {
  return is_i64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int*>(p)[i];
}
__device__ __forceinline__ void store_index(void* p, int64_t i, int is_i64, int v) {
  if (is_i64) static_cast<int64_t*>(p)[i] = v;
  else static_cast<int*>(p)[i] = v;
}
// A length that token positions held in 32 bits can start from.
__device__ __forceinline__ bool is_context(int64_t len) { return len >= 0 && len <= 0x3fffffff; }
// Takes the entry out of the table: -1 stays, the caller that gets the page owns its release.
__device__ __forceinline__ int64_t take_index(void* p, int64_t i, int is_i64) {
  if (is_i64) return static_cast<int64_t>(atomicExch(static_cast<unsigned long long*>(p) + i, ~0ull));
  return atomicExch(static_cast<int*>(p) + i, -1);
}
// One row of the table no longer names `page` (not negative): its count goes down.
__device__ __forceinline__ void release_page(int* ref_counts, int64_t page, int num_blocks) {
  if (page >= num_blocks) {
    record_device_error(B200_DEVERR_PAGE_RANGE);
  } else if (atomicSub(&ref_counts[page], 1) <= 0) {
    atomicAdd(&ref_counts[page], 1);  // was free already
    record_device_error(B200_DEVERR_PAGE_RANGE);
  }
}

// V: 16 bytes, or 4 for the caches whose rows carry a float32 scale inline.
template <typename V>
__device__ __forceinline__ V load_piece(const uint8_t* p) { return __ldcs(reinterpret_cast<const V*>(p)); }
template <typename V>
__device__ __forceinline__ void store_piece(uint8_t* p, V v) { *reinterpret_cast<V*>(p) = v; }

// ---------------------------------------------------------------- copy
struct CopyArgs {
  PageShape s;
  const void* src;
  const void* dst;
  int num_pairs, idx_i64;
};

// A warp moves one run of 32 x kCopyRun pieces of a page (4 KB with 16-byte
// pieces), all its loads issued before its first store.
constexpr int kCopyRun = 8;

template <typename V>
__global__ void __launch_bounds__(kPageThreads) copy_pages_kernel(const __grid_constant__ PageCacheSet set,
                                                                  const CopyArgs a) {
  const int lane = threadIdx.x & 31;
  const int pieces = a.s.page_bytes / static_cast<int>(sizeof(V));
  const int runs = (pieces + 32 * kCopyRun - 1) / (32 * kCopyRun);
  const int64_t per_cache = static_cast<int64_t>(a.num_pairs) * runs;
  const int64_t units = per_cache * a.s.num_caches;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kPageThreads / 32);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kPageThreads / 32) + threadIdx.x / 32; u < units; u += warps) {
    const int cache = static_cast<int>(u / per_cache);
    const int64_t rem = u - cache * per_cache;
    const int pair = static_cast<int>(rem / runs), run = static_cast<int>(rem - static_cast<int64_t>(pair) * runs);
    const int64_t from = load_index64(a.src, pair, a.idx_i64), to = load_index64(a.dst, pair, a.idx_i64);
    if (from < 0 || to < 0) continue;  // padding
    if (from >= a.s.num_blocks || to >= a.s.num_blocks) {
      if (lane == 0) record_device_error(B200_DEVERR_PAGE_RANGE);
      continue;
    }
    if (from == to) continue;
    const uint8_t* sp = set.base[cache] + from * a.s.stride_block;
    uint8_t* dp = set.base[cache] + to * a.s.stride_block;
    const int first = run * 32 * kCopyRun + lane;
    V v[kCopyRun];
#pragma unroll
    for (int k = 0; k < kCopyRun; ++k)
      if (first + 32 * k < pieces) v[k] = load_piece<V>(sp + static_cast<int64_t>(first + 32 * k) * sizeof(V));
#pragma unroll
    for (int k = 0; k < kCopyRun; ++k)
      if (first + 32 * k < pieces) store_piece<V>(dp + static_cast<int64_t>(first + 32 * k) * sizeof(V), v[k]);
  }
}

// ---------------------------------------------------------------- sequences
struct SeqTable {
  void* table;        // [max_seqs, cols], -1 = no page
  void* seq_lens;     // [max_seqs]
  int* ref_counts;    // [num_blocks], 0 = free
  int64_t stride;
  int cols, table_i64, len_i64, max_seqs, num_blocks, block_size;
};

struct ForkArgs {
  PageShape s;
  SeqTable t;
  const void* parents;
  const void* children;
  int n, idx_i64;
  int4* entries;      // [n]: parent, child (-1: nothing to do), length, page for the partial last page (-1: none)
  int* claims;        // [max_seqs]
  int* free_pages;    // [n]
};

// One block: which entries are sound, which need a page, and the lowest free
// pages for them in the order of the entries.
__global__ void __launch_bounds__(kForkThreads, 1) fork_plan_kernel(const ForkArgs a) {
  __shared__ int warp_sums[32];
  griddep_launch_dependents();
  auto entry = [&](int i, int& p, int& c) -> bool {  // in range; padding and errors are not
    const int64_t p64 = load_index64(a.parents, i, a.idx_i64), c64 = load_index64(a.children, i, a.idx_i64);
    if (p64 < 0 || c64 < 0) return false;
    if (p64 >= a.t.max_seqs || c64 >= a.t.max_seqs) {
      record_device_error(B200_DEVERR_SEQ_ROW);
      return false;
    }
    p = static_cast<int>(p64);
    c = static_cast<int>(c64);
    return true;
  };
  int p = 0, c = 0;
  for (int i = threadIdx.x; i < a.n; i += kForkThreads)
    if (entry(i, p, c)) a.claims[c] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kForkThreads)
    if (entry(i, p, c)) atomicMin(&a.claims[c], i);
  __syncthreads();
  int needed = 0;
  for (int base = 0; base < a.n; base += kForkThreads) {
    const int i = base + threadIdx.x;
    bool ok = false, need = false;
    int len = 0;
    if (i < a.n && entry(i, p, c)) {
      const int64_t len64 = load_index64(a.t.seq_lens, p, a.t.len_i64);
      ok = true;
      const bool claimed = *reinterpret_cast<volatile int*>(&a.claims[c]) == i;
      if (!claimed || load_index64(a.t.seq_lens, c, a.t.len_i64) != 0 || !is_context(len64) ||
          len64 > static_cast<int64_t>(a.t.cols) * a.t.block_size) {
        record_device_error(B200_DEVERR_SEQ_ROW);  // a row named twice, one in use, a length past the table
        ok = false;
      } else {
        len = static_cast<int>(len64);
        need = len % a.t.block_size != 0;
        if (need) {
          const int64_t last = load_index64(a.t.table, p * a.t.stride + len / a.t.block_size, a.t.table_i64);
          if (last < 0 || last >= a.t.num_blocks) {
            record_device_error(B200_DEVERR_PAGE_RANGE);
            ok = need = false;
          }
        }
      }
    }
    int total;
    const int before = block_exclusive_scan(need ? 1 : 0, warp_sums, total);
    if (i < a.n) a.entries[i] = make_int4(p, ok ? c : -1, len, need ? needed + before : -1);
    needed += total;
  }
  // Free pages, lowest first, until there are enough (four per thread and pass: a pass
  // of 4096 counts is one round of loads and one block scan, about 1.5 us).
  int found = 0;
  for (int64_t base = 0; base < a.t.num_blocks && found < needed; base += 4 * kForkThreads) {
    const int64_t first = base + 4 * threadIdx.x;
    bool zero[4];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      zero[k] = first + k < a.t.num_blocks && a.t.ref_counts[first + k] == 0;
      mine += zero[k];
    }
    int total;
    int at = found + block_exclusive_scan(mine, warp_sums, total);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (zero[k]) {
        if (at < needed) a.free_pages[at] = static_cast<int>(first + k);
        ++at;
      }
    found = min(found + total, needed);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kForkThreads) {
    int4 e = a.entries[i];
    if (e.w >= 0) {
      if (e.w < found) {
        e.w = *reinterpret_cast<volatile int*>(&a.free_pages[e.w]);
        a.t.ref_counts[e.w] = 1;
      } else {
        record_device_error(B200_DEVERR_NO_PAGE);
        e.y = e.w = -1;
      }
      a.entries[i] = e;
    }
    if (e.y >= 0) store_index(a.t.seq_lens, e.y, a.t.len_i64, e.z);
  }
}

// Table rows (grid.y = 0, 32 columns a warp) and the used rows of the partial last
// pages (grid.y - 1 = cache, kForkToks tokens a warp, loads before stores).
constexpr int kForkToks = 4;

template <typename V>
__global__ void __launch_bounds__(kPageThreads) fork_apply_kernel(const __grid_constant__ PageCacheSet set,
                                                                  const ForkArgs a) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kPageThreads / 32);
  const int64_t warp0 = static_cast<int64_t>(blockIdx.x) * (kPageThreads / 32) + threadIdx.x / 32;
  if (blockIdx.y == 0) {
    const int groups = (a.t.cols + 31) / 32;
    for (int64_t u = warp0; u < static_cast<int64_t>(a.n) * groups; u += warps) {
      const int i = static_cast<int>(u / groups), col = static_cast<int>(u - static_cast<int64_t>(i) * groups) * 32 + lane;
      const int4 e = a.entries[i];
      if (e.y < 0 || col >= a.t.cols) continue;
      const int full = e.z / a.t.block_size;
      // A row of length 0 may name pages all the same (reserved ones, those of a context
      // that was no length): they go back.  The plan was made by the counts before, so none
      // of them is given out by this call.
      const int64_t old = load_index64(a.t.table, e.y * a.t.stride + col, a.t.table_i64);
      if (old >= 0) release_page(a.t.ref_counts, old, a.t.num_blocks);
      int64_t page = -1;
      if (col < full) {
        page = load_index64(a.t.table, e.x * a.t.stride + col, a.t.table_i64);
        if (page < 0 || page >= a.t.num_blocks) {
          record_device_error(B200_DEVERR_PAGE_RANGE);
          page = -1;
        } else {
          atomicAdd(&a.t.ref_counts[page], 1);
        }
      } else if (col == full) {
        page = e.w;
      }
      store_index(a.t.table, e.y * a.t.stride + col, a.t.table_i64, static_cast<int>(page));
    }
    return;
  }
  uint8_t* base = set.base[blockIdx.y - 1];
  const int parts = (a.t.block_size + kForkToks - 1) / kForkToks;
  const int seg_pieces = a.s.seg_bytes / static_cast<int>(sizeof(V));
  const int row_pieces = seg_pieces * a.s.segs;
  for (int64_t u = warp0; u < static_cast<int64_t>(a.n) * parts; u += warps) {
    const int i = static_cast<int>(u / parts), tok0 = static_cast<int>(u - static_cast<int64_t>(i) * parts) * kForkToks;
    const int4 e = a.entries[i];
    if (e.y < 0 || e.w < 0) continue;
    const int full = e.z / a.t.block_size, toks = min(e.z - full * a.t.block_size - tok0, kForkToks);
    if (toks <= 0) continue;
    const int64_t from = load_index64(a.t.table, e.x * a.t.stride + full, a.t.table_i64);
    const uint8_t* sp = base + from * a.s.stride_block + tok0 * a.s.stride_tok;
    uint8_t* dp = base + static_cast<int64_t>(e.w) * a.s.stride_block + tok0 * a.s.stride_tok;
    for (int x = lane; x < row_pieces; x += 32) {
      const int seg = a.s.segs == 1 ? 0 : x / seg_pieces;
      const int64_t off = seg * a.s.seg_stride + static_cast<int64_t>(x - seg * seg_pieces) * sizeof(V);
      V v[kForkToks];
#pragma unroll
      for (int k = 0; k < kForkToks; ++k)
        if (k < toks) v[k] = load_piece<V>(sp + k * a.s.stride_tok + off);
#pragma unroll
      for (int k = 0; k < kForkToks; ++k)
        if (k < toks) store_piece<V>(dp + k * a.s.stride_tok + off, v[k]);
    }
  }
}

struct FreeArgs {
  SeqTable t;
  const void* rows;   // [n] rows to empty, or null: rows 0 .. n - 1 keep the pages that their length needs
  const void* context_lens;  // rows null: a row whose context is no length keeps all its pages
  int n, idx_i64;
};

// One block per row.  An entry is taken out of the table before its page's
// count goes down, so a row named twice is released once.
__global__ void __launch_bounds__(kPageThreads) free_pages_kernel(const FreeArgs a) {
  griddep_wait();
  const int64_t row = a.rows ? load_index64(a.rows, blockIdx.x, a.idx_i64) : static_cast<int64_t>(blockIdx.x);
  if (row < 0) return;  // padding
  if (row >= a.t.max_seqs) {
    if (threadIdx.x == 0) record_device_error(B200_DEVERR_SEQ_ROW);
    return;
  }
  int64_t first = 0;
  if (!a.rows) {
    if (!is_context(load_index64(a.context_lens, row, a.t.len_i64))) return;  // the keep kernel has recorded it
    const int64_t len = max(load_index64(a.t.seq_lens, row, a.t.len_i64), static_cast<int64_t>(0));
    first = (len + a.t.block_size - 1) / a.t.block_size;
  }
  for (int64_t col = first + threadIdx.x; col < a.t.cols; col += kPageThreads) {
    if (load_index64(a.t.table, row * a.t.stride + col, a.t.table_i64) < 0) continue;
    const int64_t page = take_index(a.t.table, row * a.t.stride + col, a.t.table_i64);
    if (page >= 0) release_page(a.t.ref_counts, page, a.t.num_blocks);
  }
  if (a.rows && threadIdx.x == 0) store_index(a.t.seq_lens, row, a.t.len_i64, 0);
}

// ---------------------------------------------------------------- accepted rows
struct KeepArgs {
  PageShape s;
  SeqTable t;               // seq_lens is the output; ref_counts may be null
  const void* context_lens; // [num_seqs], type of seq_lens
  const void* accepted;     // [num_seqs, most], row stride acc_stride
  const void* counts;       // [num_seqs]
  int64_t acc_stride;
  int num_seqs, most, idx_i64;
};

// Row context + accepted[i] -> context + i for i < count, in every cache.
// accepted rises strictly, so accepted[i] >= i: a row is written only after the
// rows at or before it in the path are read, and no later row's source lies at
// or before a place already written.  A lane owns its bytes of the row through
// the whole path, reads kKeepRun rows ahead and then writes them, which keeps
// that order without a barrier; the work is split over caches (grid.y), sequences
// and 32-piece columns of a row.  The chain of dependent loads (count, path, table,
// row) bounds it, so lane i looks up row i's places once and the warp passes them on
// by shuffles: 64 sequences x 32 layers 15 us with a lookup per lane and row, 8 us so.
constexpr int kKeepRun = 8;

template <typename V>
__global__ void __launch_bounds__(kPageThreads) keep_accepted_kernel(const __grid_constant__ PageCacheSet set,
                                                                     const KeepArgs a) {
  const int lane = threadIdx.x & 31;
  const int seg_pieces = a.s.seg_bytes / static_cast<int>(sizeof(V));
  const int row_pieces = seg_pieces * a.s.segs;
  const int cols = (row_pieces + 31) / 32;
  const int64_t units = static_cast<int64_t>(a.num_seqs) * cols;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kPageThreads / 32);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kPageThreads / 32) + threadIdx.x / 32; u < units; u += warps) {
    const int b = cols == 1 ? static_cast<int>(u) : static_cast<int>(u / cols);
    const int x = static_cast<int>(u - static_cast<int64_t>(b) * cols) * 32 + lane;
    const bool first_unit = blockIdx.y == 0 && x == lane;  // reports errors and stores the length
    const int64_t ctx64 = load_index64(a.context_lens, b, a.t.len_i64);
    const int64_t want = load_index64(a.counts, b, a.idx_i64);
    const bool bad_ctx = !is_context(ctx64), bad = bad_ctx || want < 0 || want > a.most;
    const int ctx = bad_ctx ? 0 : static_cast<int>(ctx64);
    int n = bad_ctx || want < 0 ? 0 : static_cast<int>(min(want, static_cast<int64_t>(a.most)));
    const int64_t trow = static_cast<int64_t>(b) * a.t.stride, arow = static_cast<int64_t>(b) * a.acc_stride;
    // Page of token position `pos`, -1 where the table has none; `in_page` its place there.
    auto page_of = [&](unsigned pos, int& in_page) -> int64_t {
      const unsigned col = pos / static_cast<unsigned>(a.t.block_size);
      in_page = static_cast<int>(pos - col * a.t.block_size);
      if (col >= static_cast<unsigned>(a.t.cols)) return -1;
      const int64_t page = load_index64(a.t.table, trow + col, a.t.table_i64);
      return page < a.t.num_blocks ? page : -1;
    };
    const int seg = a.s.segs == 1 ? 0 : x / seg_pieces;
    const int64_t own = seg * a.s.seg_stride + static_cast<int64_t>(x - seg * seg_pieces) * sizeof(V);
    int i0 = 0;
    while (i0 < n) {
      // The path ends at its first entry that does not rise, has no page, or would write a shared page.
      const int i = i0 + lane;
      int64_t from = 0, to = 0;
      bool moves = false;
      unsigned code = 0;
      if (i < n) {
        const int64_t at = load_index64(a.accepted, arow + i, a.idx_i64);
        const int64_t prev = i > 0 ? load_index64(a.accepted, arow + i - 1, a.idx_i64) : -1;
        if (at <= prev || at > 0x3fffffff) {
          code = B200_DEVERR_ACCEPT;
        } else {
          int from_in, to_in;
          const int64_t fp = page_of(static_cast<unsigned>(ctx) + static_cast<unsigned>(at), from_in);
          const int64_t tp = page_of(static_cast<unsigned>(ctx + i), to_in);
          moves = at != i;
          if (fp < 0 || tp < 0) code = B200_DEVERR_PAGE_RANGE;
          else if (a.t.ref_counts && moves && a.t.ref_counts[tp] != 1) code = B200_DEVERR_PAGE_SHARED;
          from = fp * a.s.stride_block + from_in * a.s.stride_tok;
          to = tp * a.s.stride_block + to_in * a.s.stride_tok;
        }
      }
      const unsigned wrong = __ballot_sync(0xffffffffu, code != 0);
      const int last = min(n, i0 + (wrong ? __ffs(wrong) - 1 : 32));
      if (first_unit && wrong && lane == __ffs(wrong) - 1) record_device_error(code);
      const unsigned moving = __ballot_sync(0xffffffffu, moves && i < last);
      for (int r0 = 0; r0 < last - i0; r0 += kKeepRun) {
        V v[kKeepRun];
#pragma unroll
        for (int k = 0; k < kKeepRun; ++k) {
          const int64_t src = __shfl_sync(0xffffffffu, from, r0 + k);
          if ((moving >> (r0 + k)) & 1u && x < row_pieces) v[k] = load_piece<V>(set.base[blockIdx.y] + src + own);
        }
#pragma unroll
        for (int k = 0; k < kKeepRun; ++k) {
          const int64_t dst = __shfl_sync(0xffffffffu, to, r0 + k);
          if ((moving >> (r0 + k)) & 1u && x < row_pieces) store_piece<V>(set.base[blockIdx.y] + dst + own, v[k]);
        }
      }
      i0 = last;
      if (wrong) n = last;
    }
    if (first_unit && lane == 0) {
      if (bad) record_device_error(B200_DEVERR_ACCEPT);
      store_index(a.t.seq_lens, b, a.t.len_i64, ctx + n);
    }
  }
}

}  // namespace b200
