// What the attention kernels on the tcgen05 tensor cores share: copies, descriptors, the exponential on the FMA pipe,
// bounded waits, the tensor-map encoder.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace subspec {

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, int src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)),
               "l"(gmem), "r"(src_bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// two floats -> one 32-bit word of the cache's 16-bit type (kHalf: fp16, else bf16), low half first
template <bool kHalf>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (kHalf) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^x for a pair of exponents without the special-function unit: x = n + f with n = round(x), f in [-0.5, 0.5];
// 2^f by a cubic (relative error below 8e-5: a twenty-fifth of what rounding P to bf16 costs, a sixth for fp16),
// n added into the exponent field.  The magic constant 1.5 * 2^23 leaves n in the low mantissa bits of x + magic.
__device__ __forceinline__ void exp2_pair_fma(float x0, float x1, float& p0, float& p1) {
  const uint64_t xc = f2_pack(fmaxf(x0, -125.f), fmaxf(x1, -125.f));  // -inf (masked away later) and underflow
  const uint64_t magic = f2_pack(12582912.f, 12582912.f), nmagic = f2_pack(-12582912.f, -12582912.f);
  const uint64_t t2 = f2_add(xc, magic);
  const uint64_t n2 = f2_add(t2, nmagic);
  const uint64_t f2 = f2_fma(n2, f2_pack(-1.f, -1.f), xc);
  uint64_t q = f2_fma(f2_pack(0.0551716685f, 0.0551716685f), f2, f2_pack(0.242611125f, 0.242611125f));
  q = f2_fma(q, f2, f2_pack(0.693260968f, 0.693260968f));
  q = f2_fma(q, f2, f2_pack(0.999928057f, 0.999928057f));
  float q0, q1, t0, t1;
  f2_unpack(q, q0, q1);
  f2_unpack(t2, t0, t1);
  p0 = __int_as_float(__float_as_int(q0) + (__float_as_int(t0) << 23));
  p1 = __int_as_float(__float_as_int(q1) + (__float_as_int(t1) << 23));
}

// Shared-memory matrix descriptor, 128-byte swizzle, 8-row atoms of 1024 bytes: [0,14) address >> 4, [16,30)
// leading byte offset >> 4, [32,46) stride byte offset >> 4, [46,48) version 1, [61,64) layout 2.
// K-major operand (Q and K tiles: rows x dims): stride = 1024 between 8-row groups, leading unused.
// MN-major operand (the V tile: N = dims, K = cache rows): stride = 1024 between groups of 8 cache rows,
// leading = the distance between the two 64-dim halves.
__device__ __forceinline__ uint64_t tc_desc(uint32_t smem_addr, uint32_t leading_bytes, uint32_t stride_bytes = 1024) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(leading_bytes >> 4) << 16;
  d |= (uint64_t)(stride_bytes >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// Instruction descriptor, kind::f16: D fp32 (bit 4), A and B bf16 (1 at [7,10) and [10,13)) or fp16 (0), bit 16 = B is
// MN-major, N >> 3 at [17,23), M >> 4 at [24,29).
__host__ __device__ constexpr uint32_t tc_idesc(int m, int n, bool b_mn_major, bool half) {
  return (1u << 4) | ((half ? 0u : 1u) << 7) | ((half ? 0u : 1u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void tc_mma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The hand-overs between the roles of this kernel are short and on the critical path: try_wait without a
// suspend-time hint (the waiting warp is parked by the hardware and comes back when the phase completes, so its
// polls do not fill the queue that the exponentials of the softmax warps pass through).  Bounded like every
// wait here.
constexpr uint32_t kTcPollLimit = 1u << 24;
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t it = 0; it < kTcPollLimit; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 1023u) == 1023u && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (the library does not link libcuda).
typedef CUresult (*tensor_map_encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                         const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                         CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline tensor_map_encode_fn tensor_map_encoder() {
  static tensor_map_encode_fn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<tensor_map_encode_fn>(f);
  }();
  return fn;
}

}  // namespace subspec
