#include "ops_common.h"

#include <atomic>
#include <mutex>

namespace pkb {

static __device__ int g_ops_status;

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

int op_device(int* dev, int* sms, int** status) {
  static std::atomic<int> known[64];  // SM count of a device that passed, 0: not looked at
  static int* words[64];
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (*dev < 0 || *dev >= 64) return fail(PKT_ERR_ARGS, "device id out of range");
  int n = known[*dev].load(std::memory_order_acquire);
  if (n == 0) {
    static std::mutex mu;
    std::lock_guard<std::mutex> lock(mu);
    RelaxedCapture relaxed;
    int major = 0;
    void* word = nullptr;
    e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    if (major != 10) return fail(PKT_ERR_UNSUPPORTED, "device %d is sm_%dx; this build targets sm_100a", *dev, major);
    e = cudaGetSymbolAddress(&word, g_ops_status);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetSymbolAddress");
    words[*dev] = static_cast<int*>(word);
    known[*dev].store(n, std::memory_order_release);
  }
  *sms = n;
  if (status) *status = words[*dev];
  return PKT_OK;
}

int op_shared_memory(const void* kernel, std::atomic<uint64_t>* done, int dev, int bytes) {
  const uint64_t bit = uint64_t(1) << dev;
  if (done->load(std::memory_order_acquire) & bit) return PKT_OK;
  RelaxedCapture relaxed;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shared memory)");
  done->fetch_or(bit, std::memory_order_acq_rel);
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

extern "C" int pkt_ops_status(int* code) {
  using namespace pkb;
  if (!code) return fail(PKT_ERR_ARGS, "null argument");
  int dev = 0, sms = 0, rc, *word = nullptr;
  if ((rc = op_device(&dev, &sms, &word))) return rc;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(code, word, sizeof(int), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && *code) e = cudaMemset(word, 0, sizeof(int));
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "read the operators' status");
}
