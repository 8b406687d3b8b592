// b200_pages.cu -- C ABI of the cache's page operators (kernels in kv_pages.cuh).
#include <algorithm>
#include <cstring>

#include "b200_host.h"
#include "kv_pages.cuh"
#include "minicpm_b200.h"

using namespace b200_host;

namespace b200_host {

cudaError_t pages_error_word(void** word) { return cudaGetSymbolAddress(word, b200::g_device_error); }

namespace {

struct CacheSet {
  b200::PageCacheSet set;
  b200::PageShape shape;
  bool wide;  // 16-byte pieces
};

int read_caches(const B200PageCaches* c, CacheSet* out) {
  if (!c || (c->num_caches > 0 && !c->base)) return fail(B200_ERR_INVALID, "null cache list");
  if (c->num_caches <= 0 || c->num_caches > b200::kMaxCaches)
    return fail(B200_ERR_UNSUPPORTED, "1 to %d caches in one call", b200::kMaxCaches);
  if (c->num_blocks <= 0 || c->block_size <= 0 || c->num_kv_heads <= 0 || c->row_bytes <= 0 || c->stride_block <= 0 ||
      c->stride_tok <= 0 || c->stride_head <= 0)
    return fail(B200_ERR_INVALID, "bad cache sizes");
  const int64_t heads = c->num_kv_heads, toks = c->block_size, row = c->row_bytes;
  const int64_t page = heads * toks * row;
  // Pages are dense, tokens outermost (NHD) or heads outermost (HND).
  const bool nhd = (heads == 1 || c->stride_head == row) && (toks == 1 || c->stride_tok == heads * row);
  const bool hnd = (toks == 1 || c->stride_tok == row) && (heads == 1 || c->stride_head == toks * row);
  if (!(nhd || hnd) || c->stride_block < page || page > 0x7fffffff)
    return fail(B200_ERR_UNSUPPORTED, "a page must be one dense run of [block_size, kv_heads, row] or [kv_heads, block_size, row]");
  memset(out, 0, sizeof(*out));
  uintptr_t bits = (uintptr_t)(c->stride_block | c->stride_tok | c->stride_head | row);
  for (int i = 0; i < c->num_caches; ++i) {
    if (!c->base[i]) return fail(B200_ERR_INVALID, "null cache pointer");
    out->set.base[i] = static_cast<uint8_t*>(const_cast<void*>(c->base[i]));
    bits |= reinterpret_cast<uintptr_t>(c->base[i]);
  }
  if (bits & 3) return fail(B200_ERR_UNSUPPORTED, "cache rows must be 4-byte aligned");
  out->wide = (bits & 15) == 0;
  b200::PageShape& s = out->shape;
  s.stride_block = c->stride_block;
  s.stride_tok = c->stride_tok;
  s.page_bytes = (int)page;
  s.segs = nhd ? 1 : (int)heads;
  s.seg_bytes = (int)(nhd ? heads * row : row);
  s.seg_stride = nhd ? 0 : c->stride_head;
  s.block_size = c->block_size;
  s.num_blocks = c->num_blocks;
  s.num_caches = c->num_caches;
  return B200_OK;
}

bool index_type(int32_t t) { return t == B200_DTYPE_I32 || t == B200_DTYPE_I64; }

int read_table(const B200SeqTable* p, b200::SeqTable* t) {
  if (!p) return fail(B200_ERR_INVALID, "null table");
  if (!index_type(p->table_dtype) || !index_type(p->seqlen_dtype))
    return fail(B200_ERR_INVALID, "block_table and the lengths must be int32 or int64");
  if (p->max_seqs < 0 || p->cols <= 0 || p->num_blocks <= 0 || p->block_size <= 0 || p->stride < p->cols)
    return fail(B200_ERR_INVALID, "bad table sizes");
  if (!p->block_table || !p->seq_lens) return fail(B200_ERR_INVALID, "null table pointer");
  t->table = p->block_table;
  t->seq_lens = p->seq_lens;
  t->ref_counts = p->ref_counts;
  t->stride = p->stride;
  t->cols = p->cols;
  t->table_i64 = p->table_dtype == B200_DTYPE_I64;
  t->len_i64 = p->seqlen_dtype == B200_DTYPE_I64;
  t->max_seqs = p->max_seqs;
  t->num_blocks = p->num_blocks;
  t->block_size = p->block_size;
  return B200_OK;
}

// CTAs for `warps` warps of work in each of `layers` grid rows, at most what fills the GPU.
dim3 warp_grid(int64_t warps, int layers = 1) {
  const int64_t per = b200::kPageThreads / 32, most = ((int64_t)sm_count() * 8 + layers - 1) / layers;
  return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>((warps + per - 1) / per, most)), (unsigned)layers);
}

template <typename... KArgs, typename... Args>
int launch_after(const char* what, void (*kernel)(KArgs...), dim3 grid, cudaStream_t s, const Args&... args) {
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(b200::kPageThreads);
  cfg.stream = s;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return check_launch(what);
}

size_t fork_bytes(int64_t n, int64_t max_seqs) {
  return align_up(sizeof(int4) * n, 256) + align_up(sizeof(int) * max_seqs, 256) + align_up(sizeof(int) * n, 256);
}

}  // namespace
}  // namespace b200_host

extern "C" {

int b200_copy_pages(const B200PageCaches* caches, const void* src_pages, const void* dst_pages, int32_t num_pairs,
                    int32_t index_dtype, void* stream) {
  CacheSet c;
  if (int r = read_caches(caches, &c)) return r;
  if (!index_type(index_dtype)) return fail(B200_ERR_INVALID, "page indices must be int32 or int64");
  if (num_pairs < 0) return fail(B200_ERR_INVALID, "bad sizes");
  if (num_pairs == 0) return B200_OK;
  if (!src_pages || !dst_pages) return fail(B200_ERR_INVALID, "null page indices");
  b200::CopyArgs a{};
  a.s = c.shape;
  a.src = src_pages;
  a.dst = dst_pages;
  a.num_pairs = num_pairs;
  a.idx_i64 = index_dtype == B200_DTYPE_I64;
  const int run = 32 * b200::kCopyRun * (c.wide ? 16 : 4);
  const dim3 grid = warp_grid((int64_t)num_pairs * ((c.shape.page_bytes + run - 1) / run) * c.shape.num_caches);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c.wide) b200::copy_pages_kernel<uint4><<<grid, b200::kPageThreads, 0, s>>>(c.set, a);
  else b200::copy_pages_kernel<uint32_t><<<grid, b200::kPageThreads, 0, s>>>(c.set, a);
  return check_launch("copy_pages_kernel");
}

size_t b200_fork_workspace_bytes(int32_t num_entries, int32_t max_seqs) {
  return fork_bytes(std::max(num_entries, 0), std::max(max_seqs, 0));
}

int b200_fork_sequences(const B200PageCaches* caches, const B200SeqTable* table, const void* parents,
                        const void* children, int32_t num_entries, int32_t index_dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
  CacheSet c;
  if (int r = read_caches(caches, &c)) return r;
  b200::ForkArgs a{};
  if (int r = read_table(table, &a.t)) return r;
  if (!a.t.ref_counts) return fail(B200_ERR_INVALID, "fork needs ref_counts");
  if (a.t.num_blocks != c.shape.num_blocks || a.t.block_size != c.shape.block_size)
    return fail(B200_ERR_INVALID, "the table and the caches disagree on the pages");
  if (!index_type(index_dtype)) return fail(B200_ERR_INVALID, "parents and children must be int32 or int64");
  if (num_entries < 0) return fail(B200_ERR_INVALID, "bad sizes");
  if (num_entries == 0 || a.t.max_seqs == 0) return B200_OK;
  if (!parents || !children) return fail(B200_ERR_INVALID, "null parents or children");
  const size_t need = fork_bytes(num_entries, a.t.max_seqs);
  if (!workspace || workspace_bytes < need)
    return fail(B200_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  if (!aligned16(workspace)) return fail(B200_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.s = c.shape;
  a.parents = parents;
  a.children = children;
  a.n = num_entries;
  a.idx_i64 = index_dtype == B200_DTYPE_I64;
  a.entries = reinterpret_cast<int4*>(ws);
  ws += align_up(sizeof(int4) * (size_t)num_entries, 256);
  a.claims = reinterpret_cast<int*>(ws);
  ws += align_up(sizeof(int) * (size_t)a.t.max_seqs, 256);
  a.free_pages = reinterpret_cast<int*>(ws);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  b200::fork_plan_kernel<<<1, b200::kForkThreads, 0, s>>>(a);
  if (int r = check_launch("fork_plan_kernel")) return r;
  const int64_t parts = (a.t.block_size + b200::kForkToks - 1) / b200::kForkToks;
  const dim3 grid = warp_grid(num_entries * std::max<int64_t>(parts, (a.t.cols + 31) / 32), c.shape.num_caches + 1);
  return c.wide ? launch_after("fork_apply_kernel", b200::fork_apply_kernel<uint4>, grid, s, c.set, a)
                : launch_after("fork_apply_kernel", b200::fork_apply_kernel<uint32_t>, grid, s, c.set, a);
}

int b200_free_sequences(const B200SeqTable* table, const void* rows, int32_t num_rows, int32_t index_dtype,
                        void* stream) {
  b200::FreeArgs a{};
  if (int r = read_table(table, &a.t)) return r;
  if (!a.t.ref_counts) return fail(B200_ERR_INVALID, "free needs ref_counts");
  if (!index_type(index_dtype)) return fail(B200_ERR_INVALID, "rows must be int32 or int64");
  if (num_rows < 0) return fail(B200_ERR_INVALID, "bad sizes");
  if (num_rows == 0) return B200_OK;
  if (!rows) return fail(B200_ERR_INVALID, "null rows");
  a.rows = rows;
  a.n = num_rows;
  a.idx_i64 = index_dtype == B200_DTYPE_I64;
  b200::free_pages_kernel<<<num_rows, b200::kPageThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return check_launch("free_pages_kernel");
}

int b200_keep_accepted(const B200PageCaches* caches, const B200SeqTable* table, const void* context_lens,
                       const void* accepted, int64_t accepted_stride, int32_t most, const void* num_accepted,
                       int32_t index_dtype, void* stream) {
  CacheSet c;
  if (int r = read_caches(caches, &c)) return r;
  b200::KeepArgs a{};
  if (int r = read_table(table, &a.t)) return r;
  if (a.t.num_blocks != c.shape.num_blocks || a.t.block_size != c.shape.block_size)
    return fail(B200_ERR_INVALID, "the table and the caches disagree on the pages");
  if (!index_type(index_dtype)) return fail(B200_ERR_INVALID, "accepted and num_accepted must be int32 or int64");
  if (most < 0 || accepted_stride < most) return fail(B200_ERR_INVALID, "bad sizes");
  if (a.t.max_seqs == 0) return B200_OK;
  if (context_lens == a.t.seq_lens || num_accepted == a.t.seq_lens)
    return fail(B200_ERR_INVALID, "seq_lens may not be context_lens or num_accepted");
  if (!context_lens || !num_accepted || (most > 0 && !accepted)) return fail(B200_ERR_INVALID, "null lengths or path");
  a.s = c.shape;
  a.context_lens = context_lens;
  a.accepted = accepted;
  a.counts = num_accepted;
  a.acc_stride = accepted_stride;
  a.num_seqs = a.t.max_seqs;
  a.most = most;
  a.idx_i64 = index_dtype == B200_DTYPE_I64;
  const int pieces = c.shape.seg_bytes * c.shape.segs / (c.wide ? 16 : 4);
  const dim3 grid = warp_grid((int64_t)a.num_seqs * ((pieces + 31) / 32), c.shape.num_caches);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c.wide) b200::keep_accepted_kernel<uint4><<<grid, b200::kPageThreads, 0, s>>>(c.set, a);
  else b200::keep_accepted_kernel<uint32_t><<<grid, b200::kPageThreads, 0, s>>>(c.set, a);
  if (int r = check_launch("keep_accepted_kernel")) return r;
  if (!a.t.ref_counts) return B200_OK;
  // Pages that no kept token lies on go back, once every cache's rows are moved.
  b200::FreeArgs fa{};
  fa.t = a.t;
  fa.n = a.num_seqs;
  fa.context_lens = context_lens;
  return launch_after("free_pages_kernel", b200::free_pages_kernel, dim3((unsigned)a.num_seqs), s, fa);
}

}  // extern "C"
