// Launches of the C ABI's entry points: error codes, programmatic stream serialisation, device properties.
#pragma once
#include <cuda_runtime.h>

#include <mutex>

#include "../../include/georefine_b200.h"

namespace grb {

inline int cuda_status(cudaError_t e) { return e == cudaSuccess ? GRB_OK : GRB_ERR_CUDA + int(e); }


// Launch of a decode-step kernel with programmatic stream serialisation: the kernel calls
// griddepcontrol.launch_dependents and griddepcontrol.wait before anything else, so the kernel after it in the stream
// (a fused linear, mostly) is set up and already streams its first weights on the SMs this one leaves idle, and every
// kernel still sees the complete output of the one before it.
template <class... Params, class... Args>
inline int launch_step(void (*kernel)(Params...), dim3 grid, dim3 block, uint32_t smem_bytes, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
}

// SM count of a device, looked up once.
inline int device_sm_count(int dev) {
  static std::mutex mu;
  static int sms[64] = {0};
  if (dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(mu);
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 0;
  return sms[dev];
}

}  // namespace grb
