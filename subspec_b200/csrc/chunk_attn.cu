// Attention of packed chunks of new tokens over the paged cache: causal, or causal under a sliding window with sinks.
//
// Reference: the FlashInfer prefill of the paged generators, BatchPrefillWithPagedKVCacheWrapper.run with causal=True
// (specdecodes/models/utils/flashinfer/attention_wrapper.py:104-151, 288-316) on what getKvCacheBatchPosition
// (cache_manager.py:350-414) flattened.  For token t = i-th of n of request b, at row p = kv_len_b - n + i:
//
//   o_t = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q_t k_j - m),   over the rows j <= p with
//         window == 0  or  j > p - window  or  j < sinks
#include <string.h>

#include <type_traits>

#include "chunk_attn.cuh"
#include "chunk_attn_few.cuh"
#include "tcgen05.cuh"

namespace subspec {
namespace {

// ------------------------------------------------------------------------------------------------------------------
// Tiles on the tensor cores.
//
// The rows of the problem are (token, head of the GQA group) pairs, token-major, so that a block of 128 rows is a run
// of neighbouring tokens: their KV head's cache rows are read once for the whole group, and the causal border crosses
// few tiles.  One CTA = 256 rows of one (request, KV head), two blocks that share every K / V tile of 128 cache rows:
//
//   warps 0-7   softmax, four warps per block: thread = query row = lane of tensor memory.  Per tile a thread reads its
//               128 scores, m = the running maximum, and writes P = 2^(S c - m) as 16-bit pairs over the first half of
//               the columns it read, summing P in fp32.  m moves, and the row of O in tensor memory is rescaled, only
//               when the maximum has run 2^8 ahead of it.
//   warp 8      issues the MMAs, one block after the other: O += P V (P from tensor memory, V MN-major as the cache has
//               it), in two halves of 64 cache rows as their P comes, then S = Q K^T of the next tile (128 x 128 x
//               head_dim, both K-major in shared memory) over the P just consumed: the MMAs of a thread run in order.
//               While one block is in its softmax the other's MMAs run.  (Warp 9 idles.)
//   warp 10     brings the K tiles, warp 11 the V tiles, into a ring of five entries, K(0), V(0), K(1), V(1), ...
//
// A tile lies in shared memory as 16 groups of 8 rows; a group as one (head_dim 64) or two halves of 64 dims, a half as
// 8 rows of 128 bytes under the 128-byte swizzle: the layout the tensor cores read either way round, in which the rows
// of a page are contiguous -- so that one tensor copy brings a page's rows of one head, whatever the page length (a
// multiple of 8), instead of one copy per half.
//
// Tensor memory: per block 256 columns, S | O, 128 each (O: head_dim).
constexpr int kTileKeys = 128;
constexpr int kBlockRows = 128;
constexpr int kCtaRows = 2 * kBlockRows;
constexpr int kRing = 5;
constexpr int kChunkThreads = 384;
constexpr int kIssuerWarp = 8, kLoadWarp = 10;
constexpr uint32_t kBlockCols = 256, kOCol = 128;
constexpr int kMinSplitTiles = 4;  // a cache range for a CTA of its own holds at least so many tiles

// tiles per CTA when up to `splits` CTAs share a list of n
__device__ __forceinline__ int per_split(int n, int splits) {
  const int eff = max(1, min(splits, n / kMinSplitTiles));
  return (n + eff - 1) / eff;
}

template <int kDim>
constexpr size_t tc_smem() {
  return (size_t)kCtaRows * kDim * 2 + (size_t)kRing * kTileKeys * kDim * 2 + 1024;
}

template <bool kHalf, int kDim>
__global__ void __launch_bounds__(kChunkThreads, 1)
    chunk_attn_tc_kernel(const ChunkArgs ka, const __grid_constant__ CUtensorMap tmap_k,
                         const __grid_constant__ CUtensorMap tmap_v) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kRing], empty[kRing], s_ready[2], p_ready[2][2], o_done[2], q_ready, fix, drained;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  constexpr int kHalves = kDim / 64;
  constexpr int kGroupBytes = 1024 * kHalves;           // 8 rows of a tile
  constexpr int kTileBytes = kTileKeys * kDim * 2;
  constexpr int kQHalfBytes = kBlockRows * 128;         // 64 dims of a Q block's rows
  constexpr int kQBlockBytes = kHalves * kQHalfBytes;
  const subspec_chunk_attn_args& a = ka.a;
  const int kvh = blockIdx.y, G = ka.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = (int)blockIdx.x % ka.splits;
  grid_dep_launch();

  // ---- which request and which of its row tiles: every warp looks for itself ----
  int b = -1, qt = 0;
  Request rq{};
  {
    int rem = (int)blockIdx.x / ka.splits;
    for (int b0 = 0; b0 < a.batch && b < 0; b0 += 32) {
      Request r{};
      int tiles = 0;
      if (b0 + lane < a.batch) {
        r = read_request(a, b0 + lane, false);
        if (r.n * G > ka.few_rows) tiles = (r.n * G + kCtaRows - 1) / kCtaRows;
      }
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, incl > rem);
      if (hit) {
        const int src = __ffs(hit) - 1;
        b = b0 + src;
        qt = __shfl_sync(0xffffffffu, incl, src) - 1 - rem;  // the last row tile first: it has the most tiles
        rq.q0 = __shfl_sync(0xffffffffu, r.q0, src);
        rq.n = __shfl_sync(0xffffffffu, r.n, src);
        rq.first_pos = __shfl_sync(0xffffffffu, r.first_pos, src);
        rq.kv_len = __shfl_sync(0xffffffffu, r.kv_len, src);
      } else {
        rem -= __shfl_sync(0xffffffffu, incl, 31);
      }
    }
  }
  // lengths that do not fit are reported once a launch
  auto report = [&]() {
    if (blockIdx.x == 0 && kvh == 0)
      for (int x = lane; x < a.batch; x += 32) read_request(a, x, true);
  };
  if (b < 0) {
    if (warp == 0) report();
    return;
  }
  const int rows = rq.n * G, row0 = qt * kCtaRows;
  const int nblk = row0 + kBlockRows < rows ? 2 : 1;
  // cache rows of a block's first and last token
  auto block_pos = [&](int blk, int& first, int& last) {
    first = rq.first_pos + (row0 + blk * kBlockRows) / G;
    last = rq.first_pos + (min(row0 + (blk + 1) * kBlockRows, rows) - 1) / G;
  };
  int pmin, pmax, unused;
  block_pos(0, pmin, pmax);
  if (nblk == 2) block_pos(1, unused, pmax);
  const TileList<kTileKeys> tiles(pmin, pmax, a.window, a.sinks);
  const int per = per_split(tiles.n, ka.splits);
  const int i0 = split * per, ntiles = min(per, tiles.n - i0);  // this CTA's part of the list
  const bool partial = per < tiles.n;
  if (ntiles <= 0 && split > 0) return;
  if (ntiles <= 0) {  // nothing to attend to: zeros, as the sum of no terms
    if (warp == 0) report();
    const int row = row0 + (int)threadIdx.x;
    if (threadIdx.x < kCtaRows && row < rows) {
      uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + (size_t)(rq.q0 + row / G) * a.o_token_stride +
                                          (size_t)(kvh * G + row % G) * a.o_head_stride);
      for (int c = 0; c < kDim / 8; ++c) o[c] = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  // Whether a block's rows see anything of tile row t0, and whether all of them see all of it.
  auto block_sees = [&](int first, int last, int t0) {
    return t0 <= last && (a.window == 0 || t0 + kTileKeys - 1 > first - a.window || t0 < a.sinks);
  };
  auto block_sees_all = [&](int first, int last, int t0) {
    return t0 + kTileKeys - 1 <= first && (a.window == 0 || t0 > last - a.window || t0 + kTileKeys <= a.sinks);
  };

  unsigned char* qtiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* ring = qtiles + 2 * kQBlockBytes;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int k = 0; k < 2; ++k) {
      mbar_init(&s_ready[k], 1);
      mbar_init(&p_ready[k][0], 4);
      mbar_init(&p_ready[k][1], 4);
      mbar_init(&o_done[k], 1);
    }
    mbar_init(&q_ready, kCtaRows);
    mbar_init(&fix, 1);
    mbar_init(&drained, 1);
    mbar_init_fence();
    s_abort = 0;
  }
  if (warp == kIssuerWarp) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* abort_flag = &s_abort;

  if (warp < 8) {
    // ================= softmax =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int blk = warp >> 2, rr = (int)threadIdx.x & 127;
    const int row = row0 + (int)threadIdx.x;
    const bool row_ok = row < rows;
    const int tok = row / G, head = kvh * G + row - tok * G;
    {  // every thread brings its own row of Q (a row that does not exist: zeros)
      const unsigned char* src = reinterpret_cast<const unsigned char*>(a.q);
      if (row_ok) src += 2 * ((size_t)(rq.q0 + tok) * a.q_token_stride + (size_t)head * a.q_head_stride);
      unsigned char* d = qtiles + blk * kQBlockBytes + rr * 128;
#pragma unroll
      for (int c = 0; c < kDim / 8; ++c)
        cp_async16(d + (c >> 3) * kQHalfBytes + (((c & 7) ^ (rr & 7)) << 4), src + c * 16, row_ok ? 16 : 0);
      cp_async_commit();
      cp_async_wait<0>();
      fence_async_smem();
      mbar_arrive(&q_ready);
    }
    if (blk < nblk) {
      int bfirst, blast;
      block_pos(blk, bfirst, blast);
      const int pos = min(rq.first_pos + tok, blast);  // rows that do not exist look like the last one
      const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)blk * kBlockCols;
      const uint32_t o_addr = lane_base + kOCol;
      const float c2 = ka.scale_log2;
      // fp16 weights sit 2^7 higher, out of the subnormals: at most 2^(7 + 8) between moves of the reference point
      constexpr float kOffset = kHalf ? 7.f : 0.f;
      float m = -INFINITY, l = 0.f;
      uint32_t done = 0;  // tiles this block has worked on
      bool live = true;
      for (int i = 0; i < ntiles; ++i) {
        const int t0 = tiles.first_row(i0 + i);
        if (!block_sees(bfirst, blast, t0)) continue;
        live = __all_sync(0xffffffffu, tc_wait(&s_ready[blk], done & 1u, abort_flag));
        if (!live) break;
        tc_fence_after();
        uint32_t r[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32_async(lane_base + 32 * c, r[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld_dep(r[c]);
        const bool masked = !block_sees_all(bfirst, blast, t0);
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int p0 = t0 + 32 * c;
            uint32_t bits = bits_below(pos + 1 - p0);
            if (a.window > 0) bits &= ~bits_below(pos - a.window + 1 - p0) | bits_below(a.sinks - p0);
#pragma unroll
            for (int j = 0; j < 32; ++j) r[c][j] = (bits >> j) & 1u ? r[c][j] : 0xff800000u;
          }
        }
        // the row's maximum over the tile; NaN stays NaN (a NaN score makes the row NaN)
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = max3_nan(__uint_as_float(r[c][0]), __uint_as_float(r[c][1]), __uint_as_float(r[c][2]));
#pragma unroll
          for (int j = 3; j < 31; j += 2) mx[c] = max3_nan(mx[c], __uint_as_float(r[c][j]), __uint_as_float(r[c][j + 1]));
          mx[c] = max3_nan(mx[c], __uint_as_float(r[c][31]), mx[c]);
        }
        const float tmax = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * c2;  // c2 > 0
        float alpha = 1.f;
        if (!(tmax <= m + kRescaleAt) || m == -INFINITY) {
          const float m_new = max3_nan(m, tmax, tmax);
          alpha = m == -INFINITY ? 0.f : ex2f(m - m_new);
          m = m_new;
        }
        if (done > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // O is complete up to the tile before: its MMAs were committed together with this tile's scores
#pragma unroll
          for (int c = 0; c < kDim / 32; ++c) {
            uint32_t rc[32];
            tmem_ld32_async(o_addr + 32 * c, rc);
            tmem_wait_ld_dep(rc);
#pragma unroll
            for (int j = 0; j < 32; ++j) rc[j] = __float_as_uint(__uint_as_float(rc[j]) * alpha);
            tmem_st32(o_addr + 32 * c, rc);
          }
        }
        const float u = m == -INFINITY ? 0.f : m - kOffset;  // (-inf: nothing seen yet, every weight 0)
        uint64_t sm2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        const uint64_t c2p = f2_pack(c2, c2), nup = f2_pack(-u, -u);
        auto exp_tile = [&](auto plain) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float x0, x1, p0, p1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c][2 * j]), __uint_as_float(r[c][2 * j + 1])), c2p, nup), x0, x1);
              if (decltype(plain)::value && ((j & 3) == 3 || (j & 7) == 1)) {
                exp2_pair_fma(x0, x1, p0, p1);  // three pairs in eight on the FMA pipe
              } else {
                p0 = ex2f(x0);  // 2^-inf = 0: hidden entries get the weight 0 exactly
                p1 = ex2f(x1);
              }
              sm2[j & 1] = f2_add(sm2[j & 1], f2_pack(p0, p1));
              pk[j] = pack16<kHalf>(p0, p1);
            }
            tmem_st16(lane_base + 16 * c, pk);
            if (c & 1) {  // half of the tile: its share of O += P V can begin
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_ready[blk][c >> 1]);
            }
          }
        };
        if (masked)
          exp_tile(std::false_type{});
        else
          exp_tile(std::true_type{});
        float e0, e1, e2, e3;
        f2_unpack(sm2[0], e0, e1);
        f2_unpack(sm2[1], e2, e3);
        l = l * alpha + ((e0 + e1) + (e2 + e3));
        ++done;
      }
      // ---- the result: O / l ----
      if (live && done > 0) live = __all_sync(0xffffffffu, tc_wait(&o_done[blk], 0, abort_flag));
      if (live) {
        tc_fence_after();
        const float inv = l != 0.f ? 1.f / l : 0.f;
        bool odd = false;  // a value that is not finite although the sum of the weights is
        const size_t prow = ((size_t)(rq.q0 + tok) * a.num_q_heads + head) * ka.splits + split;
        uint16_t* out_row = reinterpret_cast<uint16_t*>(a.out) + (size_t)(rq.q0 + tok) * a.o_token_stride +
                            (size_t)head * a.o_head_stride;
        if (partial && row_ok) {
          ka.part_ml[prow * 2] = m;
          ka.part_ml[prow * 2 + 1] = l;
        }
#pragma unroll
        for (int c = 0; c < kDim / 32; ++c) {
          uint32_t rc[32];
          if (done > 0) {
            tmem_ld32_async(o_addr + 32 * c, rc);
            tmem_wait_ld_dep(rc);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) rc[j] = 0u;
          }
          if (partial) {
            if (row_ok) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                reinterpret_cast<uint4*>(ka.part_o + prow * kDim)[8 * c + j] =
                    make_uint4(rc[4 * j], rc[4 * j + 1], rc[4 * j + 2], rc[4 * j + 3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float x = pos < 0 ? 0.f : __uint_as_float(rc[j]) * inv;
              odd = odd || !(fabsf(x) < INFINITY);
              rc[j] = __float_as_uint(x);
            }
            if (row_ok) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint4 v;
                v.x = pack16<kHalf>(__uint_as_float(rc[8 * j]), __uint_as_float(rc[8 * j + 1]));
                v.y = pack16<kHalf>(__uint_as_float(rc[8 * j + 2]), __uint_as_float(rc[8 * j + 3]));
                v.z = pack16<kHalf>(__uint_as_float(rc[8 * j + 4]), __uint_as_float(rc[8 * j + 5]));
                v.w = pack16<kHalf>(__uint_as_float(rc[8 * j + 6]), __uint_as_float(rc[8 * j + 7]));
                reinterpret_cast<uint4*>(out_row)[4 * c + j] = v;
              }
            }
          }
        }
        tc_fence_before();
        // 0 * inf from a V row that this row does not see but others of the tile do, or scores of -inf alone: such
        // rows are done over key by key.  (A NaN sum comes from scores the row sees: NaN is the result.)
        uint32_t again = __ballot_sync(0xffffffffu, !partial && row_ok && l == l && (odd || (l == 0.f && pos >= 0)));
        while (again) {
          const int src = __ffs(again) - 1;
          again &= again - 1;
          attn_row<kHalf, kDim>(ka, b, __shfl_sync(0xffffffffu, pos, src), rq.q0 + __shfl_sync(0xffffffffu, tok, src),
                                __shfl_sync(0xffffffffu, head, src), reinterpret_cast<float*>(qtiles + blk * kQBlockBytes) + (warp & 3) * kDim);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < kLoadWarp) {
      // ================= MMA issue: one warp for both blocks, an elected lane issues =================
      // One issuer, one block after the other: with an issuer per block the two blocks' MMAs interleave, both get
      // their scores at the same time and then both sit in their softmax while the tensor cores idle (4660 cycles a
      // tile against 2048 of MMAs).
      if (warp == kIssuerWarp) {
        constexpr uint32_t idesc_s = tc_idesc(kBlockRows, kTileKeys, false, kHalf);
        constexpr uint32_t idesc_o = tc_idesc(kBlockRows, kDim, true, kHalf);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t q_u32 = smem_u32(qtiles), ring_u32 = smem_u32(ring);
        int bfirst[2], blast[2], last_seen[2] = {-1, -1};
        uint32_t done[2] = {0, 0};
        block_pos(0, bfirst[0], blast[0]);
        block_pos(nblk - 1, bfirst[1], blast[1]);
        auto sees = [&](int blk, int i) { return blk < nblk && block_sees(bfirst[blk], blast[blk], tiles.first_row(i0 + i)); };
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
          for (int i = ntiles - 1; i >= 0 && last_seen[blk] < 0; --i)
            if (sees(blk, i)) last_seen[blk] = i;
        auto issue_s = [&](int blk, uint32_t tile) {
#pragma unroll
          for (int ks = 0; ks < kDim / 16; ++ks)
            tc_mma_f16_ss(tm + (uint32_t)blk * kBlockCols,
                          tc_desc(q_u32 + (uint32_t)(blk * kQBlockBytes + (ks >> 2) * kQHalfBytes + (ks & 3) * 32), 16),
                          tc_desc(tile + (uint32_t)((ks >> 2) * 1024 + (ks & 3) * 32), 16, kGroupBytes), idesc_s, ks > 0 ? 1u : 0u);
          tc_commit(&s_ready[blk]);
        };
        auto issue_o = [&](int blk, int half, uint32_t tile) {
#pragma unroll
          for (int x = 0; x < kTileKeys / 32; ++x) {
            const int ks = half * (kTileKeys / 32) + x;
            tc_mma_f16_ta(tm + (uint32_t)blk * kBlockCols + kOCol, tm + (uint32_t)blk * kBlockCols + (uint32_t)(8 * ks),
                          tc_desc(tile + (uint32_t)(ks * 2 * kGroupBytes), 1024, kGroupBytes), idesc_o, (done[blk] > 0 || ks > 0) ? 1u : 0u);
          }
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          const bool ok = __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag));
          tc_fence_after();
          return ok;
        };
        int e = 0;        // ring entry, in the order they come: K(0), V(0), K(1), ...
        uint32_t ph = 0;  // and its phase
        auto next = [&]() {
          if (++e == kRing) e = 0, ph ^= 1u;
        };
        bool issued = false;
        bool ok = wait(&q_ready, 0) && wait(&full[0], 0);
        if (ok) {
          if (elect_one()) {
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
              if (sees(blk, 0)) issue_s(blk, ring_u32);
            tc_commit(&empty[0]);
          }
          __syncwarp();
          issued = true;
          next();
        }
        for (int i = 0; i < ntiles && ok; ++i) {
          const int ve = e;
          ok = wait(&full[ve], ph);
          next();
          const int ke = e;
          if (ok && i + 1 < ntiles) ok = wait(&full[ke], ph);
          if (!ok) break;
          const uint32_t v_tile = ring_u32 + (uint32_t)(ve * kTileBytes), k_tile = ring_u32 + (uint32_t)(ke * kTileBytes);
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
            if (sees(blk, i)) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (!ok || !(ok = wait(&p_ready[blk][half], done[blk] & 1u))) break;
                if (elect_one()) {
                  issue_o(blk, half, v_tile);
                  if (half == 1 && i == last_seen[blk]) tc_commit(&o_done[blk]);
                }
                __syncwarp();
              }
              if (!ok) break;
              ++done[blk];
            }
            if (i + 1 < ntiles && sees(blk, i + 1)) {  // over the P just consumed: the MMAs of a thread run in order
              if (elect_one()) issue_s(blk, k_tile);
              __syncwarp();
            }
          }
          if (!ok) break;
          if (elect_one()) {
            tc_commit(&empty[ve]);
            if (i + 1 < ntiles) tc_commit(&empty[ke]);
          }
          __syncwarp();
          if (i + 1 < ntiles) next();
        }
        if (!ok && issued) {  // gave up: let the MMAs in flight finish before tensor memory is freed
          if (elect_one()) tc_commit(&drained);
          __syncwarp();
          mbar_wait_bounded(&drained, 0);
        }
      }
    } else {
      // ================= K (warp 10) and V (warp 11) tiles =================
      const int is_v = warp - kLoadWarp;
      const CUtensorMap* map = is_v ? &tmap_v : &tmap_k;
      const unsigned char* base = (is_v ? ka.v_base : ka.k_base) + (size_t)kvh * kDim * 2;
      const int* table = a.page_table + (size_t)b * a.pages_per_seq;
      const int box = ka.box_rows, boxes = box > 0 ? kTileKeys / box : 0;
      const int chunk = lane % (kDim / 8), sub = lane / (kDim / 8);  // row-by-row copies
      constexpr int kRowsPerPass = 32 / (kDim / 8);
      int e = is_v;
      uint32_t ph = 1;  // the first round finds the entries empty
      // rows some token of this CTA sees
      auto wanted = [&](int lo, int hi) { return lo < tiles.hi && (hi > tiles.lo || lo < tiles.snk); };
      auto page_of = [&](int i) -> int {  // what this lane's copy of tile i reads; -2: nothing (zeros)
        if (lane >= boxes || i >= ntiles) return -2;
        const int kpos = tiles.first_row(i0 + i) + lane * box;
        if (!wanted(kpos, kpos + box)) return -2;
        return table[ka.page_shift >= 0 ? kpos >> ka.page_shift : kpos / a.page_len];
      };
      int page = page_of(0);
      for (int i = 0; i < ntiles; ++i) {
        const int next = page_of(i + 1);  // asked for a tile ahead: a trip to memory
        if (!tc_wait(&empty[e], ph, abort_flag)) break;
        const int t0 = tiles.first_row(i0 + i);
        unsigned char* dst = ring + (size_t)e * kTileBytes;
        if (boxes > 0) {
          // rows behind the cache's end, in a box with rows in front of it: whatever the page holds there must not
          // meet a weight of 0 in the V tile
          const int z0 = rq.kv_len - t0, z1 = min((rq.kv_len + box - 1) / box * box - t0, kTileKeys);
          const bool tail = is_v && z0 > 0 && z0 < z1 && wanted(t0 + z1 - box, t0 + z0);
          uint64_t* bar = tail ? &fix : &full[e];
          if (lane == 0) mbar_expect_tx(bar, (uint32_t)kTileBytes);
          __syncwarp();
          if (lane < boxes) {
            const int kpos = t0 + lane * box;
            int unit = ka.units, slot = 0;  // outside the tensor: zeros, no memory is touched
            if (page >= 0 && page < a.num_pages) {
              unit = page * ka.page_units + kvh;
              slot = ka.page_shift >= 0 ? kpos & (a.page_len - 1) : kpos % a.page_len;
            } else if (page != -2) {
              flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
            }
            tma_load_5d(dst + (size_t)lane * box * kDim * 2, map, slot >> 3, unit, bar);
          }
          if (tail) {
            if (!tc_wait(&fix, 0, abort_flag)) break;
            for (int x = lane; x < (z1 - z0) * (kDim / 8); x += 32) {
              const int rr = z0 + x / (kDim / 8), c = x % (kDim / 8);
              *reinterpret_cast<uint4*>(dst + (rr >> 3) * kGroupBytes + (c >> 3) * 1024 + (rr & 7) * 128 + ((c & 7) << 4)) =
                  make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[e]);
          }
        } else {
          // a page length that is no multiple of 8: 16-byte copies, row by row
#pragma unroll 4
          for (int pass = 0; pass < kTileKeys / kRowsPerPass; ++pass) {
            const int rr = pass * kRowsPerPass + sub, kpos = t0 + rr;
            const unsigned char* src = base;
            int bytes = 0;
            if (kpos < rq.kv_len && wanted(kpos, kpos + 1)) {
              const int pi = kpos / a.page_len, pg = table[pi];
              if (pg < 0 || pg >= a.num_pages) {
                flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
              } else {
                bytes = 16;
                src = base + (size_t)pg * ka.page_stride + (size_t)(kpos - pi * a.page_len) * ka.row_stride + chunk * 16;
              }
            }
            cp_async16(dst + (rr >> 3) * kGroupBytes + (chunk >> 3) * 1024 + (rr & 7) * 128 + (((chunk & 7) ^ (rr & 7)) << 4), src,
                       bytes);
          }
          cp_async_commit();
          cp_async_wait<0>();
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[e]);
        }
        page = next;
        if ((e += 2) >= kRing) e -= kRing, ph ^= 1u;
      }
      if (is_v) report();
      if (*abort_flag) {  // gave up: the copies in flight land before the CTA leaves
        for (int s = 0; s < kRing; ++s)
          for (uint32_t p = 0; p < 2; ++p) mbar_wait_bounded(&full[s], p);
      }
    }
  }
  __syncthreads();
  if (s_abort && threadIdx.x == 0) flag(a.dev_status, SUBSPEC_DEV_TIMEOUT);
  if (warp == kIssuerWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the cache ranges of a row: a warp per (token, query head) adds up the ranges' unnormalised rows, each weighted by
// 2^(its reference point - the largest one), and divides by the likewise weighted sum of their sums.
template <bool kHalf, int kDim>
__global__ void __launch_bounds__(128) chunk_merge_kernel(const ChunkArgs ka) {
  __shared__ float qs[4][kDim];
  const subspec_chunk_attn_args& a = ka.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = ka.group;
  const long long r = (long long)blockIdx.x * 4 + warp;
  grid_dep_wait();
  if (r >= (long long)a.tokens * a.num_q_heads) return;
  const int t = (int)(r / a.num_q_heads), head = (int)(r - (long long)t * a.num_q_heads);
  const int b = request_of(a.q_indptr, a.batch, t);
  if (b < 0) return;
  const Request rq = read_request(a, b, false);
  const int i = t - rq.q0;
  if (i >= rq.n || rq.n * G <= ka.few_rows) return;
  // the row tile this row was part of, its list of cache tiles, and how that was cut
  const int row0 = (i * G + head % G) / kCtaRows * kCtaRows;
  const TileList<kTileKeys> tiles(rq.first_pos + row0 / G, rq.first_pos + (min(row0 + kCtaRows, rq.n * G) - 1) / G, a.window, a.sinks);
  const int per = per_split(tiles.n, ka.splits);
  if (per >= tiles.n) return;  // one CTA did it all
  const int parts = (tiles.n + per - 1) / per;
  const float* ml = ka.part_ml + (size_t)r * ka.splits * 2;
  float mstar = -INFINITY;
  for (int s = 0; s < parts; ++s) mstar = ml[2 * s + 1] != 0.f ? max3_nan(mstar, ml[2 * s], ml[2 * s]) : mstar;
  constexpr int kPer = kDim / 32;
  float acc[kPer] = {}, lsum = 0.f;
  for (int s = 0; s < parts; ++s) {
    const float l = ml[2 * s + 1];
    if (l == 0.f) continue;  // nothing seen in this range
    const float w = ex2f(ml[2 * s] - mstar);
    const float* o = ka.part_o + ((size_t)r * ka.splits + s) * kDim + lane * kPer;
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] += w * o[c];
    lsum += w * l;
  }
  const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
  bool odd = lsum == 0.f;
#pragma unroll
  for (int c = 0; c < kPer; ++c) {
    acc[c] *= inv;
    odd = odd || !(fabsf(acc[c]) < INFINITY);
  }
  const int pos = rq.first_pos + i;
  if (__any_sync(0xffffffffu, odd) && lsum == lsum && pos >= 0) {  // see the epilogue above
    attn_row<kHalf, kDim>(ka, b, pos, t, head, qs[warp]);
    return;
  }
  uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + (size_t)t * a.o_token_stride +
                                              (size_t)head * a.o_head_stride);
#pragma unroll
  for (int c = 0; c < kPer / 2; ++c) out[lane * (kPer / 2) + c] = pack16<kHalf>(acc[2 * c], acc[2 * c + 1]);
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
      (long long)a.pages_per_seq * a.page_len > (1LL << 30) || (long long)a.tokens * a.num_q_heads > (1LL << 30))
    return SUBSPEC_EUNSUPPORTED;
  return SUBSPEC_OK;
}

}  // namespace
}  // namespace subspec

using namespace subspec;

static void chunk_sizes(ChunkArgs& ka) {
  const subspec_chunk_attn_args& a = ka.a;
  ka.group = a.num_q_heads / a.num_kv_heads;
  // Which kernel a request's rows go to.  Up to 32 rows for every request: the kernel for few rows does it all.  More
  // for some: it still takes the requests of up to 16, where the token counts leave room for such beside the longest
  // (on average at most 64 rows each).
  const long long most = (long long)a.max_q_len * ka.group;
  const long long others = (long long)(a.tokens - a.max_q_len) * ka.group;
  ka.few_rows = most <= 16 ? 16 : most <= 32 ? 32 : a.batch > 1 && others <= 64LL * (a.batch - 1) ? 16 : 0;
  if (ka.few_rows >= most) {
    ka.items = 0;
    ka.splits = 1;
    return;
  }
  const long long by_tokens = (long long)a.tokens * ka.group / kCtaRows + a.batch;
  const long long by_batch = (long long)a.batch * ((most + kCtaRows - 1) / kCtaRows);
  ka.items = (int)(by_tokens < by_batch ? by_tokens : by_batch);
  // Few row tiles with long caches would leave SMs idle: as many ranges as fill them once, none shorter than
  // kMinSplitTiles at the table's full width (shorter caches are cut into fewer ranges on the device).
  const long long ctas = (long long)ka.items * a.num_kv_heads;
  const long long cap = (long long)a.pages_per_seq * a.page_len;
  const long long seen = a.window > 0 ? (long long)a.window + a.sinks + a.max_q_len : cap;
  const long long tiles = ((seen < cap ? seen : cap) + kTileKeys - 1) / kTileKeys;
  long long s = a.kv_splits;
  if (s == 0) {
    s = kNumSMs / (ctas > 0 ? ctas : 1);
    if (s > tiles / kMinSplitTiles) s = tiles / kMinSplitTiles;
    if (s > 32) s = 32;
    if (s < 1) s = 1;
  }
  ka.splits = (int)s;
}

static size_t split_floats(const ChunkArgs& ka) {
  if (ka.splits <= 1) return 0;
  return (size_t)ka.a.tokens * ka.a.num_q_heads * ka.splits * (ka.a.head_dim + 2);
}
static size_t chunk_scratch_bytes(const ChunkArgs& ka) {
  return (split_floats(ka) + (ka.few_rows ? chunk_few_floats(ka) : 0)) * sizeof(float);
}

extern "C" int subspec_chunk_attention_scratch_bytes(const subspec_chunk_attn_args* args, size_t* bytes) {
  const int rc = check_args(args);
  if (rc) return rc;
  if (!bytes) return SUBSPEC_EINVAL;
  *bytes = 0;
  if (args->batch == 0 || args->tokens == 0 || args->max_q_len == 0) return SUBSPEC_OK;
  ChunkArgs ka{};
  ka.a = *args;
  chunk_sizes(ka);
  *bytes = chunk_scratch_bytes(ka);
  return SUBSPEC_OK;
}

// The K (or V) rows of a layer as the copies see them: (64 dims | row of a group of 8 | half of the head's dims | group
// of 8 rows in the page | unit), a unit being one row of one head: pages and heads both are whole numbers of units
// apart, so the outermost coordinate addresses (page, head) at once and a box = a page's rows (or box_rows of them)
// of one head, landing group by group, half by half.
static bool chunk_tensor_map(CUtensorMap* m, const ChunkArgs& ka, const unsigned char* base) {
  const subspec_chunk_attn_args& a = ka.a;
  const cuuint64_t halves = a.head_dim / 64;
  const cuuint64_t dims[5] = {64, 8, halves, (cuuint64_t)a.page_len / 8, (cuuint64_t)ka.units};
  const cuuint64_t strides[4] = {(cuuint64_t)ka.row_stride, 128, (cuuint64_t)ka.row_stride * 8, (cuuint64_t)a.head_dim * 2};
  const cuuint32_t box[5] = {64, 8, (cuuint32_t)halves, (cuuint32_t)ka.box_rows / 8, 1}, estr[5] = {1, 1, 1, 1, 1};
  return tensor_map_encoder()(m, a.dtype == SUBSPEC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                              const_cast<unsigned char*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace subspec {
void chunk_tensor_maps(ChunkArgs& ka, int rows, CUtensorMap* k, CUtensorMap* v) {
  memset(k, 0, sizeof(*k));
  memset(v, 0, sizeof(*v));
  int box = rows;
  while (box > 1 && ka.a.page_len % box) box /= 2;  // the largest power of two up to a tile that divides a page
  ka.box_rows = box >= 8 && tensor_map_encoder() ? box : 0;
  if (ka.box_rows && !(chunk_tensor_map(k, ka, ka.k_base) && chunk_tensor_map(v, ka, ka.v_base))) ka.box_rows = 0;
}
}  // namespace subspec

template <bool kHalf, int kDim>
static int launch_chunk(ChunkArgs& ka, cudaStream_t stream) {
  const subspec_chunk_attn_args& a = ka.a;
  const int rc = allow_smem<chunk_attn_tc_kernel<kHalf, kDim>>(tc_smem<kDim>());
  if (rc) return rc;
  CUtensorMap tmap_k, tmap_v;
  chunk_tensor_maps(ka, kTileKeys, &tmap_k, &tmap_v);
  chunk_attn_tc_kernel<kHalf, kDim><<<dim3((unsigned)(ka.items * ka.splits), (unsigned)a.num_kv_heads), kChunkThreads,
                                      tc_smem<kDim>(), stream>>>(ka, tmap_k, tmap_v);
  if (ka.splits > 1) {
    const long long rows = (long long)a.tokens * a.num_q_heads;
    const int rc2 = cuda_check(cudaGetLastError());
    return rc2 ? rc2 : launch_dependent(chunk_merge_kernel<kHalf, kDim>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, ka);
  }
  return cuda_check(cudaGetLastError());
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
  ChunkArgs ka{};
  ka.a = a;
  chunk_sizes(ka);
  ka.scale_log2 = (float)(a.sm_scale * 1.4426950408889634);
  ka.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1 << s) == a.page_len) ka.page_shift = s;
  ka.row_stride = (long long)a.num_kv_heads * a.head_dim * 2;
  ka.page_stride = 2 * a.page_len * ka.row_stride;
  ka.k_base = reinterpret_cast<const unsigned char*>(a.pool) + (size_t)a.layer * a.num_pages * ka.page_stride;
  ka.v_base = ka.k_base + a.page_len * ka.row_stride;
  ka.page_units = 2 * a.page_len * a.num_kv_heads;
  const long long units = (long long)(a.num_pages - 1) * ka.page_units + a.num_kv_heads;
  if (units > 0x7fffffffLL) return SUBSPEC_EUNSUPPORTED;
  ka.units = (int)units;
  const size_t need = chunk_scratch_bytes(ka);
  if (need && (!a.scratch || (reinterpret_cast<uintptr_t>(a.scratch) & 15u) || a.scratch_bytes < need)) return SUBSPEC_ESCRATCH;
  ka.part_o = reinterpret_cast<float*>(a.scratch);
  ka.part_ml = ka.part_o + (size_t)a.tokens * a.num_q_heads * ka.splits * a.head_dim;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (ka.few_rows) {
    rc = launch_chunk_few(ka, ka.part_o + split_floats(ka), st);
    if (rc || ka.items == 0) return rc;
  }
  if (a.dtype == SUBSPEC_F16) return a.head_dim == 128 ? launch_chunk<true, 128>(ka, st) : launch_chunk<true, 64>(ka, st);
  return a.head_dim == 128 ? launch_chunk<false, 128>(ka, st) : launch_chunk<false, 64>(ka, st);
}
