// Host helpers of the operators with kernels of their own: the driver's tensor
// map encoder and the error word that their bounded waits report to.
#include <atomic>
#include <mutex>

#include "umma.cuh"

namespace pasa {

// Of each device: the word in which kernels set bits, and what was last taken out of it.
__device__ uint32_t g_operator_errors[2];

namespace {
// Read and cleared at once: a bit that a kernel on another stream sets is in this report or in the next.
__global__ void take_errors(uint32_t* words) { words[1] = atomicExch(&words[0], 0u); }
std::mutex g_taking;  // from taking the bits to their arrival: there is one place for them
}  // namespace

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
  uint32_t* words = pasa::operator_error_word();
  if (!words) return PASA_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const std::lock_guard<std::mutex> hold(pasa::g_taking);
  pasa::take_errors<<<1, 1, 0, st>>>(words);
  if (cudaGetLastError() != cudaSuccess ||
      cudaMemcpyAsync(flags, words + 1, sizeof(uint32_t), cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return PASA_ERR_CUDA;
  return PASA_OK;
}
