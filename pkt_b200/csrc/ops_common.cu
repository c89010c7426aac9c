#include "ops_common.h"

#include <atomic>
#include <mutex>

namespace pkb {

static void* driver_entry(const char* name) {
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
    return nullptr;
  return p;
}

EncodeTiled op_encode_tiled() {
  static const EncodeTiled fn = reinterpret_cast<EncodeTiled>(driver_entry("cuTensorMapEncodeTiled"));
  return fn;
}

int op_device(int* dev, int* sms) {
  static std::atomic<int> known[64];  // SM count of a device that passed, 0: not looked at
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (*dev < 0 || *dev >= 64) return fail(PKT_ERR_ARGS, "device id out of range");
  int n = known[*dev].load(std::memory_order_relaxed);
  if (n == 0) {
    int major = 0;
    e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    if (major != 10) return fail(PKT_ERR_UNSUPPORTED, "device %d is sm_%dx; this build targets sm_100a", *dev, major);
    known[*dev].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return PKT_OK;
}

int op_check_memory(const void* p, const char* what, int dev) {
  using GetAttributes = CUresult (*)(unsigned int, CUpointer_attribute*, void**, CUdeviceptr);
  static const GetAttributes get = reinterpret_cast<GetAttributes>(driver_entry("cuPointerGetAttributes"));
  if (!p) return PKT_OK;
  if (!get) return fail(PKT_ERR_CUDA, "cuPointerGetAttributes unavailable");
  unsigned int type = 0, managed = 0;
  int ordinal = -1;
  CUpointer_attribute which[3] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
                                  CU_POINTER_ATTRIBUTE_IS_MANAGED};
  void* into[3] = {&type, &ordinal, &managed};
  const CUresult r = get(3, which, into, reinterpret_cast<CUdeviceptr>(p));
  if (r != CUDA_SUCCESS) return fail(PKT_ERR_CUDA, "cuPointerGetAttributes(%s) failed (%d)", what, int(r));
  if (managed) return PKT_OK;
  if (type != CU_MEMORYTYPE_DEVICE) return fail(PKT_ERR_ARGS, "%s is not device memory", what);
  if (ordinal != dev) return fail(PKT_ERR_ARGS, "%s is memory of device %d, the current device is %d", what, ordinal, dev);
  return PKT_OK;
}

}  // namespace pkb
