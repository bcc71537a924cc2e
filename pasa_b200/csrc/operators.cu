// Host helpers of the operators with kernels of their own: the driver's tensor
// map encoder and the error word that their bounded waits report to.
#include <atomic>

#include "umma.cuh"

namespace pasa {

__device__ uint32_t g_operator_errors;  // one a device; kernels only set bits

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    return nullptr;
  }();
  return fn;
}

uint32_t* operator_error_word() {
  constexpr int kDevices = 64;
  static std::atomic<uint32_t*> words[kDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return nullptr;
  uint32_t* word = words[dev].load(std::memory_order_acquire);
  if (word == nullptr) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_operator_errors) != cudaSuccess) return nullptr;
    word = static_cast<uint32_t*>(p);
    words[dev].store(word, std::memory_order_release);
  }
  return word;
}

}  // namespace pasa

extern "C" int pasa_operator_errors(void* stream, uint32_t* flags) {
  if (!flags) return PASA_ERR_NULL;
  uint32_t* word = pasa::operator_error_word();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!word || cudaMemcpyAsync(flags, word, sizeof(uint32_t), cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      cudaMemsetAsync(word, 0, sizeof(uint32_t), st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess)
    return PASA_ERR_CUDA;
  return PASA_OK;
}
