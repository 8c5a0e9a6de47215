// Library-wide entry points: version string and CUDA error bookkeeping.
#include "common.cuh"

namespace subspec {
namespace {
thread_local cudaError_t g_last_error = cudaSuccess;
__device__ uint32_t g_default_status;  // one in each device's image of the library, zero at load
}
int cuda_fail(cudaError_t e) {
  g_last_error = e;
  return SUBSPEC_ECUDA;
}
}  // namespace subspec

extern "C" const char* subspec_version(void) { return "subspec_b200 0.1 (sm_100a)"; }

extern "C" int subspec_default_status(uint32_t** word) {
  if (!word) return SUBSPEC_EINVAL;
  void* p = nullptr;
  const int rc = subspec::cuda_check(cudaGetSymbolAddress(&p, subspec::g_default_status));
  *word = rc ? nullptr : static_cast<uint32_t*>(p);
  return rc;
}

extern "C" const char* subspec_last_cuda_error(void) { return cudaGetErrorString(subspec::g_last_error); }
