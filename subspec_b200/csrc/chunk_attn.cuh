// Attention of packed chunks over the paged cache: what its kernels share.
#pragma once

#include <math.h>

#include "attn_common.cuh"
#include "common.cuh"
#include "tma.cuh"

namespace subspec {

struct ChunkArgs {
  subspec_chunk_attn_args a;
  int group;         // query heads per KV head; x / group = umulhi(x, group_mul) >> group_shift for 0 <= x < 2^31
  uint32_t group_mul, group_shift;
  float scale_log2;  // sm_scale * log2(e)
  int page_shift;    // log2(page_len) when it is a power of two, else -1
  int box_rows;      // cache rows per tensor copy (0: the page length does not suit them)
  // row `slot` of page `pg`, KV head h: k_base (v_base) + pg * page_stride + slot * row_stride + h * head_dim * 2 bytes
  const unsigned char* k_base;
  const unsigned char* v_base;
  long long page_stride, row_stride;
  int page_units, units;  // a page, and the whole layer, in rows of one head (the tensor map's outermost coordinate)
  int ctas;               // of the kernel for many rows (0: not launched)
  int4* runs;             // its runs: request, KV head, row tile of the first piece; 1: begun in an earlier run, 2: ends in this
  float* part_o;          // [run][2][256][head_dim] unnormalised rows: [0] of a row tile begun earlier, [1] of one that goes on
  float* part_ml;         // [run][2][256][2] reference point (log2 units) and sum
  int few_rows;           // requests of at most so many rows go to the kernel for few rows (0: none)
  int4* few_runs;         // the same for it
  float* few_o;
  float* few_ml;
};

// x / group without a division (four of which, at 150 cycles each, stand in front of every row tile).
__device__ __forceinline__ int by_group(const ChunkArgs& ka, int x) {
  return ka.group == 1 ? x : (int)(__umulhi((uint32_t)x, ka.group_mul) >> ka.group_shift);
}

constexpr float kRescaleAt = 8.f;  // log2 units the maximum may run ahead of the exponents' reference point

template <bool kHalf>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if (kHalf) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

// One row by a warp, key by key, touching nothing but the rows that it sees: every lane has two (head_dim 64) or four of
// the dims, four keys at a time.  (What the tiles leave undone: see their epilogues.)
template <bool kHalf, int kDim>
__device__ void attn_row(const ChunkArgs& ka, int b, int pos, int t, int head) {
  const subspec_chunk_attn_args& a = ka.a;
  constexpr int kPer = kDim / 32, kAtOnce = 4;
  const int lane = threadIdx.x & 31;
  auto load = [&](const uint16_t* p, float (&x)[kPer]) {
#pragma unroll
    for (int c = 0; c < kPer / 2; ++c) {
      const float2 y = unpack16<kHalf>(reinterpret_cast<const uint32_t*>(p)[lane * (kPer / 2) + c]);
      x[2 * c] = y.x, x[2 * c + 1] = y.y;
    }
  };
  float q[kPer];
  load(reinterpret_cast<const uint16_t*>(a.q) + (size_t)t * a.q_token_stride + (size_t)head * a.q_head_stride, q);
  const size_t row = (size_t)a.num_kv_heads * kDim, plane = (size_t)a.page_len * row;
  const uint16_t* pool = reinterpret_cast<const uint16_t*>(a.pool) + (size_t)a.layer * a.num_pages * 2 * plane +
                         (size_t)(head / ka.group) * kDim;
  const int* table = a.page_table + (size_t)b * a.pages_per_seq;
  const int lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
  const int head_rows = min(a.window > 0 ? a.sinks : 0, lo);  // rows [0, head_rows) and [lo, pos]
  const int seen = head_rows + pos + 1 - lo;
  float m = -INFINITY, l = 0.f, o[kPer] = {};
  for (int j0 = 0; j0 < seen; j0 += kAtOnce) {
    float s[kAtOnce], v[kAtOnce][kPer];
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      const int idx = j0 + x, j = idx < head_rows ? idx : lo + idx - head_rows;
      s[x] = 0.f;
#pragma unroll
      for (int c = 0; c < kPer; ++c) v[x][c] = 0.f;
      if (idx >= seen) continue;
      const int pi = j / a.page_len, pg = table[pi];
      if (pg < 0 || pg >= a.num_pages) {
        flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
        continue;  // a row of zeros, as the tiles hold it
      }
      const uint16_t* at = pool + (size_t)pg * 2 * plane + (size_t)(j - pi * a.page_len) * row;
      float k[kPer];
      load(at, k);
      load(at + plane, v[x]);
#pragma unroll
      for (int c = 0; c < kPer; ++c) s[x] += q[c] * k[c];
    }
#pragma unroll
    for (int d = 16; d; d >>= 1)
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) s[x] += __shfl_xor_sync(0xffffffffu, s[x], d);
    float mx = m;
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      s[x] = j0 + x < seen ? s[x] * ka.scale_log2 : -INFINITY;
      mx = (mx != mx || s[x] != s[x]) ? NAN : fmaxf(mx, s[x]);
    }
    const float old = m == -INFINITY ? 0.f : exp2f(m - mx);  // nothing summed yet: nothing to rescale
    m = mx;
    l *= old;
#pragma unroll
    for (int c = 0; c < kPer; ++c) o[c] *= old;
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      if (j0 + x >= seen) continue;
      const float p = mx == -INFINITY ? 0.f : exp2f(s[x] - mx);  // (scores of -inf so far: weight 0)
      l += p;
#pragma unroll
      for (int c = 0; c < kPer; ++c) o[c] += p * v[x][c];
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
  TileList() = default;
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

// One page's rows of one head: coordinates (dim, row of 8, half, group of 8 rows, unit), see chunk_tensor_map (the last: V rows lie half a page behind K rows).
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

__device__ __forceinline__ Request shfl_request(const Request& r, int src) {
  return Request{__shfl_sync(0xffffffffu, r.q0, src), __shfl_sync(0xffffffffu, r.n, src), __shfl_sync(0xffffffffu, r.first_pos, src),
                 __shfl_sync(0xffffffffu, r.kv_len, src)};
}

}  // namespace subspec
