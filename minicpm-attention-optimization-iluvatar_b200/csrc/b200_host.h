// b200_host.h -- host helpers that the translation units of the library share
// (defined in b200_lib.cu unless inline here).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace b200_host {

constexpr int kNumSmsB200 = 148;

// Sets the calling thread's error message and returns `code`.
int fail(int code, const char* fmt, ...);
const char* last_error();
// The launch error of the last kernel, as a status.
int check_launch(const char* what);
// SMs of the current device (148 without one).
int sm_count();
// A tensor map with 128-byte swizzle, 256-byte L2 promotion and zero fill.
int encode_map(CUtensorMap* map, CUtensorMapDataType dt, cuuint32_t rank, const void* base, const cuuint64_t* dims,
               const cuuint64_t* strides_bytes, const cuuint32_t* box, const char* what);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// The address of each translation unit's device error word (b200_lib.cu has its own).
cudaError_t prompt_error_word(void** word);
cudaError_t tree_error_word(void** word);
cudaError_t pages_error_word(void** word);

// `dependent`: a programmatic dependent of the launch before it, whose end its
// set-up overlaps; it waits (griddepcontrol.wait) before it reads that kernel's output.
template <typename... KArgs, typename... Args>
int launch_form_kernel(const char* what, bool dependent, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem,
                       cudaStream_t s, const Args&... args) {
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = pdl;
  cfg.numAttrs = dependent ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return check_launch(what);
}

}  // namespace b200_host
