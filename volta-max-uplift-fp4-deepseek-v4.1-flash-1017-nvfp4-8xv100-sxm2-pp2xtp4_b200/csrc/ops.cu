// The device error word of the stateless operators (permute.cu, fp8_*.cu): no
// layer object holds one for them.  One word per GPU, OR-ed by kernels that
// found a row or offset out of range; b200moe_op_errors reads it and clears the
// bits that it read.
#include <atomic>

#include "common.cuh"
#include "internal.h"

namespace b200moe {

__device__ uint32_t g_op_errors;

uint32_t* op_error_word() {
  static std::atomic<uint32_t*> word[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  uint32_t* p = word[dev].load(std::memory_order_relaxed);
  if (!p) {
    void* a = nullptr;
    if (cudaGetSymbolAddress(&a, g_op_errors) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    p = static_cast<uint32_t*>(a);
    word[dev].store(p, std::memory_order_relaxed);
  }
  return p;
}

int sm_count() {
  static std::atomic<int> count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = count[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
    count[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

namespace {

// Clears what was read and nothing else: another stream's kernel may have set a bit since.
__global__ void clear_errors_kernel(uint32_t* word, uint32_t seen) { atomicAnd(word, ~seen); }

}  // namespace
}  // namespace b200moe

extern "C" int b200moe_op_errors(void* stream, uint32_t* bits) {
  using namespace b200moe;
  uint32_t* word = op_error_word();
  if (!word) return B200MOE_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t b = 0;
  cudaError_t e = cudaMemcpyAsync(&b, word, sizeof(b), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && b) {
    clear_errors_kernel<<<1, 1, 0, s>>>(word, b);
    e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return B200MOE_ERR_CUDA;
  }
  if (bits) *bits = b;
  return b & kErrTimeout ? B200MOE_ERR_TIMEOUT : b ? B200MOE_ERR_BOUNDS : B200MOE_OK;
}
