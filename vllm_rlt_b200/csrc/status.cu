// The status word: where kernels report what they could not raise.
#include "common.cuh"

// Allocated and cleared outside of whatever the calling thread captures. A word
// from a captured allocation would lie in that graph's pool, unset until the
// first replay, and its clearing would be a node that every replay repeats.
extern "C" int rlt_status_create(int32_t** word) {
  if (word == nullptr) return RLT_E_SHAPE;
  *word = nullptr;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaError_t err = cudaThreadExchangeStreamCaptureMode(&mode);
  if (err != cudaSuccess) return static_cast<int>(err);
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
  return static_cast<int>(err);
}
