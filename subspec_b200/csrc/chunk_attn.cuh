// Attention of packed chunks over the paged cache: what its kernels share.
#pragma once

#include <math.h>

#include "attn_common.cuh"
#include "common.cuh"
#include "tma.cuh"

namespace subspec {

struct ChunkArgs {
  subspec_chunk_attn_args a;
  int group;         // query heads per KV head
  float scale_log2;  // sm_scale * log2(e)
  int page_shift;    // log2(page_len) when it is a power of two, else -1
  int box_rows;      // cache rows per tensor copy (0: the page length does not suit them)
  // row `slot` of page `pg`, KV head h: k_base (v_base) + pg * page_stride + slot * row_stride + h * head_dim * 2 bytes
  const unsigned char* k_base;
  const unsigned char* v_base;
  long long page_stride, row_stride;
  int page_units, units;  // a page, and the whole layer, in rows of one head (the tensor maps' outermost coordinate)
  int items;              // row tiles the grid has room for, per KV head
  int splits;             // CTAs that may share a row tile's cache tiles
  float* part_o;          // splits > 1: [token][head][split][head_dim] unnormalised outputs
  float* part_ml;         //             [token][head][split][2] reference point (log2 units) and sum
  int few_rows;           // requests of at most so many rows go to the kernel for few rows (0: none)
  float* few_o;           // [part][few_rows][head_dim], [part][few_rows][2]: the same for its parts
  float* few_ml;
};

constexpr float kRescaleAt = 8.f;  // log2 units the maximum may run ahead of the exponents' reference point

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

// What the rows of tokens [pmin, pmax] (cache rows) can see, as a list of 128-row tiles: the tiles of the sinks, then
// those from the lowest window row to the highest token.
template <int kTile>
struct TileList {
  int hi, lo, snk;  // rows [0, snk) and [lo, hi)
  int s_tiles, m0, n;
  __device__ __forceinline__ TileList(int pmin, int pmax, int window, int sinks) {
    hi = max(pmax + 1, 0);
    lo = window > 0 ? min(max(pmin - window + 1, 0), hi) : 0;
    snk = window > 0 ? min(sinks, hi) : 0;
    m0 = lo / kTile;
    s_tiles = min((snk + kTile - 1) / kTile, m0);
    n = s_tiles + (hi + kTile - 1) / kTile - m0;
  }
  __device__ __forceinline__ int first_row(int i) const { return (i < s_tiles ? i : m0 + i - s_tiles) * kTile; }
};

// Bits [0, n) of a word.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// One page's rows of one head: coordinates (dim, row of 8, half, group of 8 rows, unit), see chunk_tensor_map.
__device__ __forceinline__ void tma_load_5d(void* dst_smem, const CUtensorMap* map, int c3, int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst_smem)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}

// A request as the kernels read it: its tokens, and the cache row of its first one.
struct Request {
  int q0, n, first_pos, kv_len;  // n: tokens that get an output
};
__device__ __forceinline__ Request read_request(const subspec_chunk_attn_args& a, int b, bool report) {
  Request r;
  r.q0 = a.q_indptr[b];
  const int q1 = a.q_indptr[b + 1], n = max(q1 - r.q0, 0), cap = a.pages_per_seq * a.page_len, kv = a.kv_len[b];
  r.kv_len = min(max(kv, 0), cap);
  r.first_pos = r.kv_len - n;
  r.n = min(n, a.max_q_len);
  if (r.q0 < 0 || q1 > a.tokens || q1 < r.q0) r.n = 0;
  if (report && (r.n != n || q1 < r.q0 || kv < n || kv > cap)) flag(a.dev_status, SUBSPEC_DEV_BAD_COUNT);
  return r;
}

}  // namespace subspec
