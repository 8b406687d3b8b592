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
// Takes the entry out of the table: -1 stays, the caller that gets the page owns its release.
__device__ __forceinline__ int64_t take_index(void* p, int64_t i, int is_i64) {
  if (is_i64) return static_cast<int64_t>(atomicExch(static_cast<unsigned long long*>(p) + i, ~0ull));
  return atomicExch(static_cast<int*>(p) + i, -1);
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
template <int kUnused = 0>
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
      if (*reinterpret_cast<volatile int*>(&a.claims[c]) != i || load_index64(a.t.seq_lens, c, a.t.len_i64) != 0 || len64 < 0 ||
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
  // Free pages, lowest first, until there are enough (four per thread and pass).
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

// Table rows (32 columns a warp) and the used rows of the partial last pages
// (kForkToks tokens of one cache a warp, loads before stores).
constexpr int kForkToks = 4;

template <typename V>
__global__ void __launch_bounds__(kPageThreads) fork_apply_kernel(const __grid_constant__ PageCacheSet set,
                                                                  const ForkArgs a) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kPageThreads / 32);
  const int64_t warp0 = static_cast<int64_t>(blockIdx.x) * (kPageThreads / 32) + threadIdx.x / 32;
  const int groups = (a.t.cols + 31) / 32;
  for (int64_t u = warp0; u < static_cast<int64_t>(a.n) * groups; u += warps) {
    const int i = static_cast<int>(u / groups), col = static_cast<int>(u - static_cast<int64_t>(i) * groups) * 32 + lane;
    const int4 e = a.entries[i];
    if (e.y < 0 || col >= a.t.cols) continue;
    const int full = e.z / a.t.block_size;
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
  const int parts = (a.t.block_size + kForkToks - 1) / kForkToks;
  const int seg_pieces = a.s.seg_bytes / static_cast<int>(sizeof(V));
  const int row_pieces = seg_pieces * a.s.segs;
  const int64_t per_cache = static_cast<int64_t>(a.n) * parts;
  for (int64_t u = warp0; u < per_cache * a.s.num_caches; u += warps) {
    const int cache = static_cast<int>(u / per_cache);
    const int rem = static_cast<int>(u - cache * per_cache);
    const int i = rem / parts, tok0 = (rem - i * parts) * kForkToks;
    const int4 e = a.entries[i];
    if (e.y < 0 || e.w < 0) continue;
    const int toks = min(e.z % a.t.block_size - tok0, kForkToks);
    if (toks <= 0) continue;
    const int64_t from = load_index64(a.t.table, e.x * a.t.stride + e.z / a.t.block_size, a.t.table_i64);
    const uint8_t* sp = set.base[cache] + from * a.s.stride_block + tok0 * a.s.stride_tok;
    uint8_t* dp = set.base[cache] + static_cast<int64_t>(e.w) * a.s.stride_block + tok0 * a.s.stride_tok;
    for (int x = lane; x < row_pieces; x += 32) {
      const int seg = x / seg_pieces;
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
  int n, idx_i64;
};

// One block per row.  An entry is taken out of the table before its page's
// count goes down, so a row named twice is released once.
template <int kUnused = 0>
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
    const int64_t len = max(load_index64(a.t.seq_lens, row, a.t.len_i64), static_cast<int64_t>(0));
    first = (len + a.t.block_size - 1) / a.t.block_size;
  }
  for (int64_t col = first + threadIdx.x; col < a.t.cols; col += kPageThreads) {
    if (load_index64(a.t.table, row * a.t.stride + col, a.t.table_i64) < 0) continue;
    const int64_t page = take_index(a.t.table, row * a.t.stride + col, a.t.table_i64);
    if (page < 0) continue;
    if (page >= a.t.num_blocks) {
      record_device_error(B200_DEVERR_PAGE_RANGE);
    } else if (atomicSub(&a.t.ref_counts[page], 1) <= 0) {
      atomicAdd(&a.t.ref_counts[page], 1);  // was free already
      record_device_error(B200_DEVERR_PAGE_RANGE);
    }
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
// that order without a barrier; the work is split over caches, sequences and
// 32-piece columns of a row.
constexpr int kKeepRun = 8;

template <typename V>
__global__ void __launch_bounds__(kPageThreads) keep_accepted_kernel(const __grid_constant__ PageCacheSet set,
                                                                     const KeepArgs a) {
  const int lane = threadIdx.x & 31;
  const int seg_pieces = a.s.seg_bytes / static_cast<int>(sizeof(V));
  const int row_pieces = seg_pieces * a.s.segs;
  const int cols = (row_pieces + 31) / 32;
  const int64_t per_cache = static_cast<int64_t>(a.num_seqs) * cols;
  const int64_t units = per_cache * a.s.num_caches;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kPageThreads / 32);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kPageThreads / 32) + threadIdx.x / 32; u < units; u += warps) {
    const int cache = static_cast<int>(u / per_cache);
    const int rem = static_cast<int>(u - cache * per_cache);
    const int b = rem / cols, x = (rem - b * cols) * 32 + lane;
    const bool first_unit = cache == 0 && rem == b * cols;  // reports errors and stores the length
    const int64_t ctx = load_index64(a.context_lens, b, a.t.len_i64);
    int64_t want = load_index64(a.counts, b, a.idx_i64);
    bool bad = ctx < 0 || ctx > 0x7fffffff - a.most || want < 0 || want > a.most;
    want = bad ? (ctx < 0 || want < 0 || ctx > 0x7fffffff - a.most ? 0 : a.most) : want;
    const int64_t trow = static_cast<int64_t>(b) * a.t.stride, arow = static_cast<int64_t>(b) * a.acc_stride;
    // Byte offset of token position `pos` in a cache, -1 where the table has no page for it.
    auto place = [&](int64_t pos) -> int64_t {
      const int64_t col = pos / a.t.block_size;
      if (col >= a.t.cols) return -1;
      const int64_t page = load_index64(a.t.table, trow + col, a.t.table_i64);
      if (page < 0 || page >= a.t.num_blocks) return -1;
      return page * a.s.stride_block + (pos - col * a.t.block_size) * a.s.stride_tok;
    };
    // The path ends at its first entry that does not rise, has no page, or would write a shared page.
    int n = static_cast<int>(want);
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool wrong = false;
      unsigned code = 0;
      if (i < n) {
        const int64_t at = load_index64(a.accepted, arow + i, a.idx_i64);
        const int64_t prev = i > 0 ? load_index64(a.accepted, arow + i - 1, a.idx_i64) : -1;
        if (at <= prev || at > 0x7fffffff) {
          wrong = true;
          code = B200_DEVERR_ACCEPT;
        } else if (place(ctx + at) < 0 || place(ctx + i) < 0) {
          wrong = true;
          code = B200_DEVERR_PAGE_RANGE;
        } else if (a.t.ref_counts && at != i &&
                   a.t.ref_counts[load_index64(a.t.table, trow + (ctx + i) / a.t.block_size, a.t.table_i64)] != 1) {
          wrong = true;
          code = B200_DEVERR_PAGE_SHARED;
        }
      }
      const unsigned any = __ballot_sync(0xffffffffu, wrong);
      if (any) {
        const int stop = __ffs(any) - 1;
        if (first_unit && lane == stop) record_device_error(code);
        n = i0 + stop;
      }
    }
    if (first_unit && lane == 0) {
      if (bad) record_device_error(B200_DEVERR_ACCEPT);
      store_index(a.t.seq_lens, b, a.t.len_i64, static_cast<int>(max(min(ctx, static_cast<int64_t>(0x7fffffff - a.most)), static_cast<int64_t>(0))) + n);
    }
    if (x >= row_pieces) continue;
    const int seg = x / seg_pieces;
    uint8_t* base = set.base[cache] + seg * a.s.seg_stride + static_cast<int64_t>(x - seg * seg_pieces) * sizeof(V);
    for (int i0 = 0; i0 < n; i0 += kKeepRun) {
      V v[kKeepRun];
      bool moves[kKeepRun];
#pragma unroll
      for (int k = 0; k < kKeepRun; ++k) {
        moves[k] = false;
        if (i0 + k < n) {
          const int64_t at = load_index64(a.accepted, arow + i0 + k, a.idx_i64);
          moves[k] = at != i0 + k;
          if (moves[k]) v[k] = load_piece<V>(base + place(ctx + at));
        }
      }
#pragma unroll
      for (int k = 0; k < kKeepRun; ++k)
        if (moves[k]) store_piece<V>(base + place(ctx + i0 + k), v[k]);
    }
  }
}

}  // namespace b200
