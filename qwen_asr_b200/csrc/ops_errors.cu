// Error words of the 8-bit operators (OpsErrors, ops.h): the C entry points' own, one a device, and how a word is
// read.
#include "ops.h"

namespace qasr {
namespace {

__device__ OpsErrors g_api_errors;

__global__ void report_kernel(OpsErrors* word, int code) { ops_gave_up(word, code); }

}  // namespace

OpsErrors* ops_api_errors() {
  static std::atomic<OpsErrors*> words[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  OpsErrors* w = words[dev].load();
  if (!w) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_api_errors) != cudaSuccess) return nullptr;
    w = (OpsErrors*)p;
    words[dev].store(w);
  }
  return w;
}

int ops_errors(const OpsErrors* word, int& seen) {
  OpsErrors now{};
  if (!word || cudaMemcpy(&now, word, sizeof(now), cudaMemcpyDeviceToHost) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (now.count == seen) return 0;
  seen = now.count;
  return now.code;
}

cudaError_t ops_report(OpsErrors* word, int code) {
  if (!word) return cudaErrorInvalidValue;
  report_kernel<<<1, 1>>>(word, code);
  return cudaDeviceSynchronize();
}

}  // namespace qasr
