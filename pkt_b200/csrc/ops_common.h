// What the stand-alone operators (layer norm, AdamW, 8-bit quantising and product)
// share on the host side: the device they run on, argument checks, launches.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "runtime_impl.h"

namespace pkb {

// The current device, checked once to be one this build runs on, its SM count and
// (where asked for) the address of its status word, which a kernel sets when one of
// its bounded waits runs out.
int op_device(int* dev, int* sms, int** status = nullptr);
// Raises a kernel's shared-memory limit, once per kernel and device.
int op_shared_memory(const void* kernel, std::atomic<uint64_t>* done, int dev, int bytes);
// `p` is memory of device `dev` (or managed memory), so that a host pointer or
// another GPU's buffer is an error here and not a fault in the kernel. Null passes. Until
// a graph has run, memory of its own allocation nodes looks like any unknown address and
// is refused with them.
int op_check_memory(const void* p, const char* what, int dev);
// cuTensorMapEncodeTiled, looked up once; null when the driver has none.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled op_encode_tiled();

// First calls may come inside a stream capture, where some queries are only allowed in
// relaxed mode; none of them touches the captured stream.
struct RelaxedCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// One launch, with programmatic stream serialization: it is made while the kernel before
// it still drains, and each kernel here begins with griddepcontrol.wait, which waits for
// all of that kernel and its memory (0.2 to 0.5 us of a call in a graph).
template <typename... KArgs, typename... Args>
cudaError_t op_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace pkb
