// Attention of packed chunks of new tokens over the paged cache: causal, or causal under a sliding window with sinks.
//
// Reference: the FlashInfer prefill of the paged generators, BatchPrefillWithPagedKVCacheWrapper.run with causal=True
// (specdecodes/models/utils/flashinfer/attention_wrapper.py:104-151, 288-316) on what getKvCacheBatchPosition
// (cache_manager.py:350-414) flattened.  For token t = i-th of n of request b, at row p = kv_len_b - n + i:
//
//   o_t = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q_t k_j - m),   over the rows j <= p with
//         window == 0  or  j > p - window  or  j < sinks
#include <math.h>

#include "common.cuh"

namespace subspec {
namespace {

struct ChunkArgs {
  subspec_chunk_attn_args a;
  int group;         // query heads per KV head
  float scale_log2;  // sm_scale * log2(e)
};

// The request of packed token t: the last b with q_indptr[b] <= t; -1 behind the last request.
__device__ __forceinline__ int request_of(const int* q_indptr, int batch, int t) {
  if (t < q_indptr[0] || t >= q_indptr[batch]) return -1;
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (q_indptr[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <bool kHalf>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if (kHalf) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <bool kHalf>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (kHalf) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One row by a warp, key by key, touching nothing but the rows that it sees: a lane takes every 32nd row for the
// scores, then every lane two (head_dim 64) or four dims of the output.  `qs`: head_dim floats of shared memory.
template <bool kHalf, int kDim>
__device__ void attn_row(const ChunkArgs& ka, int b, int pos, int t, int head, float* qs) {
  const subspec_chunk_attn_args& a = ka.a;
  constexpr int kPer = kDim / 32;
  const int lane = threadIdx.x & 31;
  const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (size_t)t * a.q_token_stride + (size_t)head * a.q_head_stride;
  __syncwarp();
  for (int d = lane; d < kDim; d += 32) qs[d] = unpack16<kHalf>((uint32_t)q[d]).x * ka.scale_log2;
  __syncwarp();
  const size_t row = (size_t)a.num_kv_heads * kDim, plane = (size_t)a.page_len * row;
  const uint16_t* pool = reinterpret_cast<const uint16_t*>(a.pool) + (size_t)a.layer * a.num_pages * 2 * plane +
                         (size_t)(head / ka.group) * kDim;
  const int* table = a.page_table + (size_t)b * a.pages_per_seq;
  const int lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
  const int head_rows = min(a.window > 0 ? a.sinks : 0, lo);  // rows [0, head_rows) and [lo, pos]
  const int seen = head_rows + pos + 1 - lo;
  float m = -INFINITY, l = 0.f, o[kPer] = {};
  for (int j0 = 0; j0 < seen; j0 += 32) {
    const int idx = j0 + lane, j = idx < head_rows ? idx : lo + idx - head_rows;
    long long at = -1;  // element offset of the K row
    float s = -INFINITY;
    if (idx < seen) {
      const int pi = j / a.page_len, pg = table[pi];
      if (pg >= 0 && pg < a.num_pages) {
        at = (long long)((size_t)pg * 2 * plane + (size_t)(j - pi * a.page_len) * row);
        const uint4* k = reinterpret_cast<const uint4*>(pool + at);
        s = 0.f;
#pragma unroll 4
        for (int c = 0; c < kDim / 8; ++c) {
          const uint4 w = k[c];
          const float2 x0 = unpack16<kHalf>(w.x), x1 = unpack16<kHalf>(w.y), x2 = unpack16<kHalf>(w.z), x3 = unpack16<kHalf>(w.w);
          const float* p = qs + 8 * c;
          s += p[0] * x0.x + p[1] * x0.y + p[2] * x1.x + p[3] * x1.y + p[4] * x2.x + p[5] * x2.y + p[6] * x3.x + p[7] * x3.y;
        }
      } else {
        flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
        s = 0.f;  // a row of zeros, as the tiles hold it
      }
    }
    float mx = s;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, mx, d);
      mx = (mx != mx || y != y) ? NAN : fmaxf(mx, y);
    }
    mx = (m != m) ? m : ((mx != mx) ? mx : fmaxf(m, mx));
    const float old = (m == -INFINITY) ? 0.f : exp2f(m - mx);  // nothing summed yet: nothing to rescale
    const float p = idx < seen && mx != -INFINITY ? exp2f(s - mx) : 0.f;  // (scores of -inf so far: weight 0)
    float ps = p;
#pragma unroll
    for (int d = 16; d; d >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, d);
    l = l * old + ps;
    m = mx;
#pragma unroll
    for (int c = 0; c < kPer; ++c) o[c] *= old;
    const int n = min(32, seen - j0);
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, p, i);
      const long long ra = __shfl_sync(0xffffffffu, at, i);
      if (ra < 0) continue;
      const uint32_t* v = reinterpret_cast<const uint32_t*>(pool + ra + plane);
#pragma unroll
      for (int c = 0; c < kPer / 2; ++c) {
        const float2 x = unpack16<kHalf>(v[lane * (kPer / 2) + c]);
        o[2 * c] += w * x.x;
        o[2 * c + 1] += w * x.y;
      }
    }
  }
  const float inv = seen > 0 ? 1.f / l : 0.f;
  uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + (size_t)t * a.o_token_stride +
                                              (size_t)head * a.o_head_stride);
#pragma unroll
  for (int c = 0; c < kPer / 2; ++c)
    out[lane * (kPer / 2) + c] = pack16<kHalf>(o[2 * c] * inv, o[2 * c + 1] * inv);
}

// A warp per (token, query head).
template <bool kHalf, int kDim>
__global__ void __launch_bounds__(128) chunk_attn_rows_kernel(const ChunkArgs ka) {
  __shared__ float qs[4][kDim];
  const subspec_chunk_attn_args& a = ka.a;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= (long long)a.tokens * a.num_q_heads) return;
  const int t = (int)(r / a.num_q_heads), head = (int)(r - (long long)t * a.num_q_heads);
  const int b = request_of(a.q_indptr, a.batch, t);
  if (b < 0) return;
  const int q0 = a.q_indptr[b], n = a.q_indptr[b + 1] - q0;
  if (n > a.max_q_len) {
    flag(a.dev_status, SUBSPEC_DEV_BAD_COUNT);
    if (t - q0 >= a.max_q_len) return;
  }
  int kv_len = a.kv_len[b];
  const int cap = a.pages_per_seq * a.page_len;
  if (kv_len < n || kv_len > cap) flag(a.dev_status, SUBSPEC_DEV_BAD_COUNT);
  const int pos = min(kv_len, cap) - n + (t - q0);
  attn_row<kHalf, kDim>(ka, b, pos, t, head, qs[threadIdx.x >> 5]);
}

int check_args(const subspec_chunk_attn_args* args) {
  if (!args || args->struct_size != sizeof(subspec_chunk_attn_args)) return SUBSPEC_EINVAL;
  const subspec_chunk_attn_args& a = *args;
  if (a.batch < 0 || a.tokens < 0 || a.max_q_len < 0 || a.num_q_heads < 1 || a.num_kv_heads < 1 || a.layers < 1 ||
      a.layer < 0 || a.layer >= a.layers || a.num_pages < 1 || a.page_len < 1 || a.pages_per_seq < 1 || a.window < 0 ||
      a.sinks < 0 || a.kv_splits < 0 || a.kv_splits > 1024 || !(a.sm_scale > 0.0) ||
      (a.dtype != SUBSPEC_BF16 && a.dtype != SUBSPEC_F16))
    return SUBSPEC_EINVAL;
  if ((a.head_dim != 64 && a.head_dim != 128) || a.num_q_heads % a.num_kv_heads ||
      (long long)a.pages_per_seq * a.page_len > (1LL << 30) || (long long)a.tokens * a.num_q_heads > (1LL << 31))
    return SUBSPEC_EUNSUPPORTED;
  return SUBSPEC_OK;
}

}  // namespace
}  // namespace subspec

using namespace subspec;

extern "C" int subspec_chunk_attention_scratch_bytes(const subspec_chunk_attn_args* args, size_t* bytes) {
  const int rc = check_args(args);
  if (rc) return rc;
  if (!bytes) return SUBSPEC_EINVAL;
  *bytes = 0;
  return SUBSPEC_OK;
}

extern "C" int subspec_chunk_attention_paged(const subspec_chunk_attn_args* args, subspec_stream_t stream) {
  int rc = check_args(args);
  if (rc) return rc;
  const subspec_chunk_attn_args& a = *args;
  if (a.batch == 0 || a.tokens == 0 || a.max_q_len == 0) return SUBSPEC_OK;
  if (!a.pool || !a.page_table || !a.kv_len || !a.q_indptr || !a.q || !a.out) return SUBSPEC_EINVAL;
  // 16-byte copies of cache, query and output rows
  if (((reinterpret_cast<uintptr_t>(a.pool) | reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15u) ||
      (a.q_token_stride % 8) || (a.q_head_stride % 8) || (a.o_token_stride % 8) || (a.o_head_stride % 8))
    return SUBSPEC_EUNSUPPORTED;
  ChunkArgs ka;
  ka.a = a;
  ka.group = a.num_q_heads / a.num_kv_heads;
  ka.scale_log2 = (float)(a.sm_scale * 1.4426950408889634);
  const bool half = a.dtype == SUBSPEC_F16;
  auto kernel = a.head_dim == 128 ? (half ? chunk_attn_rows_kernel<true, 128> : chunk_attn_rows_kernel<false, 128>)
                                  : (half ? chunk_attn_rows_kernel<true, 64> : chunk_attn_rows_kernel<false, 64>);
  const long long rows = (long long)a.tokens * a.num_q_heads;
  kernel<<<(unsigned)((rows + 3) / 4), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(ka);
  return cuda_check(cudaGetLastError());
}
