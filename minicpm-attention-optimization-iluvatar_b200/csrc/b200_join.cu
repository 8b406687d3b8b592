// b200_join.cu -- launch of stream_combine_kernel, which both attention forms share.
#include "minicpm_b200.h"
#include "stream_combine.cuh"

namespace b200_host {

namespace {

template <typename T>
int launch_typed(const b200::StreamCombineArgs& c, int head_dim, int ctas, cudaStream_t s) {
  auto kernel = head_dim == 256  ? b200::stream_combine_kernel<T, 256>
                : head_dim == 64 ? b200::stream_combine_kernel<T, 64>
                                 : b200::stream_combine_kernel<T, 128>;
  const unsigned chunks = b200::kUnitRows / b200::kJoinRows;
  return launch_form_kernel("stream_combine_kernel", true, kernel, dim3((unsigned)ctas, chunks), b200::kCombineThreads, 0, s,
                            c);
}

}  // namespace

int launch_stream_combine(const b200::StreamCombineArgs& c, int dtype, int head_dim, int ctas, cudaStream_t s) {
  return dtype == B200_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(c, head_dim, ctas, s)
                                  : launch_typed<__half>(c, head_dim, ctas, s);
}

}  // namespace b200_host
