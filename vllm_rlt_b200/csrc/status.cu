// The status words: where kernels report what they could not raise.
#include <mutex>

#include "common.cuh"

namespace rlt {
namespace {

// Allocated and cleared outside of whatever the calling thread captures. A word
// from a captured allocation would lie in that graph's pool, unset until the
// first replay, and its clearing would be a node that every replay repeats.
cudaError_t create(int32_t** word) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaError_t err = cudaThreadExchangeStreamCaptureMode(&mode);
  if (err != cudaSuccess) return err;
  cudaStream_t stream = nullptr;
  void* at = nullptr;
  err = cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking);
  if (err == cudaSuccess) err = cudaMalloc(&at, sizeof(int32_t));
  if (err == cudaSuccess) err = cudaMemsetAsync(at, 0, sizeof(int32_t), stream);
  if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  if (stream != nullptr) (void)cudaStreamDestroy(stream);
  if (err != cudaSuccess) {
    if (at != nullptr) (void)cudaFree(at);
    at = nullptr;
    (void)cudaGetLastError();
  }
  (void)cudaThreadExchangeStreamCaptureMode(&mode);
  *word = static_cast<int32_t*>(at);
  return err;
}

}  // namespace
}  // namespace rlt

extern "C" int rlt_status_word(int32_t** word) {
  constexpr int kDevices = 64;
  static std::mutex lock;
  static int32_t* words[kDevices];
  if (word == nullptr) return RLT_E_SHAPE;
  *word = nullptr;
  int dev = 0;
  if (const cudaError_t err = cudaGetDevice(&dev)) return static_cast<int>(err);
  if (dev < 0 || dev >= kDevices) return RLT_E_DEVICE;
  lock.lock();  // nothing below throws
  const cudaError_t err = words[dev] != nullptr ? cudaSuccess : rlt::create(&words[dev]);
  *word = words[dev];
  lock.unlock();
  return static_cast<int>(err);
}
