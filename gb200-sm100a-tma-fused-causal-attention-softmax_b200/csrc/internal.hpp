// What the library's translation units share on the host: the error detail of
// the calling thread and the current device's properties.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cs_host {

// Record a message as cs_last_error_detail and return `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail_cuda(cudaError_t e, const char* what);

struct Device {
  int id = 0;
  int sms = 0;
  int max_smem = 0;  // opt-in shared memory per CTA
};

// Properties of the calling thread's current device; CS_ERR_DEVICE unless it is sm_10x.
int current_device(Device* out);

constexpr int kMaxDeviceIds = 64;

// Launch with programmatic stream serialisation: the kernel's CTAs may start
// while the previous kernel in the stream finishes (see pdl_wait).
template <typename Params>
cudaError_t launch(void (*kernel)(Params), dim3 grid, int block, size_t smem, void* stream, const Params& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace cs_host
