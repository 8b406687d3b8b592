// stream_combine.cuh -- the join of units that streamed CTAs share (attention of
// packed prompts and of draft trees).
#pragma once

#include "b200_host.h"
#include "paged_attention.cuh"

namespace b200 {

struct StreamCombineArgs {
  const int4* meta;       // [CTAs]: sequence, query unit, KV head, pieces of the unit that CTA i began (0: none)
  const float* o_part;    // [2 CTAs][D / 4][kUnitRows][4], normalised
  const float* m_part;    // [2 CTAs][kUnitRows]
  const float* l_part;
  const void* cu_q;
  void* out;
  int64_t out_st, out_sh;
  int len_i64, total_q;
  int group, pos_per_tile, pos_per_unit;
};

// out = sum_s w_s O_s / sum_s w_s, w_s = exp(m_s - max m) l_s, over the pieces of a
// unit that streamed CTAs share: the first in slot 2 i + 1, the others in the slots
// 2 (i + 1), 2 (i + 2), .. of the CTAs behind.  A block joins 32 rows of CTA i's
// unit: lane r of warp w has row r and the column quads w, w + 8, .., so that every
// load of a warp is one run of 512 bytes, with the pieces of kJoinRun slots in
// flight; the rows leave through shared memory as 16-byte pieces.  Latency and L2
// bound (the partials were just written); a CTA that shares no unit costs one load.
constexpr int kJoinRows = 32;
template <int D>
constexpr int kJoinRun = D == 64 ? 8 : D == 128 ? 4 : 2;

template <typename T, int D>
__global__ void __launch_bounds__(kCombineThreads) stream_combine_kernel(const StreamCombineArgs a) {
  constexpr int kWarps = kCombineThreads / 32;
  constexpr int kQuads = D / 4 / kWarps;  // column quads of a lane
  constexpr int kRun = kJoinRun<D>;
  __shared__ uint2 rows[kJoinRows][D / 4 + 1];
  griddep_wait();
  const int cta = blockIdx.x;
  const int4 su = a.meta[cta];
  if (su.w == 0) return;
  const int q_begin = load_clipped(a.cu_q, su.x, a.len_i64, 0, a.total_q);  // the rows that the pieces hold (seq_bounds)
  const int q_end = load_clipped(a.cu_q, su.x + 1, a.len_i64, q_begin, a.total_q);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto place = [&](int ur, int64_t& tok, int64_t& head) -> bool {  // where row ur of the unit goes, if it exists
    const int t = ur / kAttnTileM, r = ur % kAttnTileM;
    const int pos = su.y * a.pos_per_unit + t * a.pos_per_tile + r / a.group;
    tok = q_begin + pos;
    head = static_cast<int64_t>(su.z) * a.group + r % a.group;
    return r < a.group * a.pos_per_tile && t * a.pos_per_tile < a.pos_per_unit && pos < q_end - q_begin;
  };
  const int ur = blockIdx.y * kJoinRows + lane;
  int64_t tok, head;
  const bool valid = place(ur, tok, head);
  if (!__any_sync(0xffffffffu, valid)) return;  // the same in every warp
  float m_max = -INFINITY, den = 0.f;
  float acc[kQuads][4] = {};
  for (int s0 = 0; s0 < su.w; s0 += kRun) {
    float m[kRun], l[kRun];
    float4 x[kRun][kQuads];
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      const int s = s0 + k;
      m[k] = -INFINITY;
      l[k] = 0.f;
      if (valid && s < su.w) {
        const int64_t slot = 2 * (cta + s) + (s == 0 ? 1 : 0);
        m[k] = a.m_part[slot * kUnitRows + ur];
        l[k] = a.l_part[slot * kUnitRows + ur];
        const float4* p = reinterpret_cast<const float4*>(a.o_part) + slot * (D / 4) * kUnitRows + ur;
#pragma unroll
        for (int c = 0; c < kQuads; ++c) x[k][c] = p[(warp + c * kWarps) * kUnitRows];
      }
    }
    float m_new = m_max;
#pragma unroll
    for (int k = 0; k < kRun; ++k) m_new = fmaxf(m_new, m[k]);
    const float scale = m_max == -INFINITY ? 0.f : expf(m_max - m_new);
    den *= scale;
#pragma unroll
    for (int c = 0; c < kQuads; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[c][i] *= scale;
    m_max = m_new;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      // A piece in which the row saw no key has l = 0 and its O is left out by
      // selection.  A NaN among the row's scores makes l NaN: it is kept.
      if (l[k] == 0.f) continue;
      const float w = expf(m[k] - m_max) * l[k];
      den += w;
#pragma unroll
      for (int c = 0; c < kQuads; ++c) {
        acc[c][0] = fmaf(w, x[k][c].x, acc[c][0]);
        acc[c][1] = fmaf(w, x[k][c].y, acc[c][1]);
        acc[c][2] = fmaf(w, x[k][c].z, acc[c][2]);
        acc[c][3] = fmaf(w, x[k][c].w, acc[c][3]);
      }
    }
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
  for (int c = 0; c < kQuads; ++c)
    rows[lane][warp + c * kWarps] = make_uint2(Pack2<T>::pack(acc[c][0] * inv, acc[c][1] * inv),
                                               Pack2<T>::pack(acc[c][2] * inv, acc[c][3] * inv));
  __syncthreads();
  constexpr int kPieces = D / 8;  // 16-byte pieces of a row
  for (int i = threadIdx.x; i < kJoinRows * kPieces; i += kCombineThreads) {
    const int r = i / kPieces, c = i % kPieces;
    if (!place(blockIdx.y * kJoinRows + r, tok, head)) continue;
    const uint2 lo = rows[r][2 * c], hi = rows[r][2 * c + 1];
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + tok * a.out_st + head * a.out_sh + c * 8) =
        make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
}

}  // namespace b200

namespace b200_host {

// Launched behind the attention kernel, whose CTA count is `ctas` (b200_join.cu).
int launch_stream_combine(const b200::StreamCombineArgs& c, int dtype, int head_dim, int ctas, cudaStream_t s);

}  // namespace b200_host
