// Chunk attention for requests with few rows: decode steps and short drafts, where the cache is read once and little is
// computed on it (2 * rows flop a byte: HBM-bound up to hundreds of rows).
//
// The work of the call is one line of cache tiles -- requests, their KV heads, their tiles of 64 cache rows one behind
// the other -- cut into equal runs, one per CTA: ragged batches and lone long caches load every SM alike.  Three CTAs an
// SM, so that the ends of one's pieces lie under the others' copies.  A run is walked in pieces, a piece being what it has of one (request, head).  Each of the CTA's four warps
// takes 16 of a tile's 64 rows and works on its own: it has a ring of stages (16 K and 16 V rows each) that its lanes
// fill by tensor copies, and computes, with Q in registers as the A operand of m16n8k16,
//
//   S = Q K^T (16 rows x 16 keys),  P = 2^(S c - m),  O += P V,  l += P
//
// under its own running maximum m, which moves only when it is overtaken by 2^8.  (mma.sync: 16 rows do not fill a
// tcgen05 tile of 128, and the tensor pipe is idle most of the time either way.)  At the end of a piece the four warps'
// (m, l, O) are joined in shared memory; a piece that is all of its (request, head) is divided and written, any other
// goes to scratch, and a second kernel joins those.
//
// Measured (B200, 28 query heads on 4 KV heads of 128 dims, bf16): 64 single tokens behind 4k to 8k rows 120 us for
// 714 MB = 5.95 TB/s, 0.91 of the card's copy; with the join and its launch 127 us.  A lone token behind 4095 rows, 15 us:
// launch, lengths, page list, copies and join one after the other.  Two CTAs an SM with twice the stages are as fast
// on long caches and slower on short pieces (48 windows of 1024 rows: 51.5 against 48.5 us); runs of at least 8 tiles
// instead of 4 cost the lone token 3 us.
//
// That is the variant of up to 16 rows.  The one of 17 to 32 keeps two row tiles of Q and O under the same bound of 168
// registers and spills (head_dim 128: 932 bytes stored and 964 loaded, 64: 88 and 116): 64 requests of 2 to 4 tokens, 28
// rows at most, behind 2k to 8k rows take 370 us where 1 or 2 tokens take 112 (floors 116 and 93).
//
// P is rounded to the cache's type, as in the tiles for many rows (chunk_attn.cu) and for the same reason.  Page lengths
// that are no multiple of 8 are copied 16 bytes a lane: the 64 single tokens 303 us instead of 126 at pages of 20 rows.
#include "chunk_attn.cuh"
#include "chunk_attn_few.cuh"

namespace subspec {
namespace {

constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps;
constexpr int kWarpKeys = 16;
constexpr int kFewTile = kFewWarps * kWarpKeys;
constexpr int kFewPerSm = 3;
constexpr int kFewCtas = kFewPerSm * kNumSMs;
constexpr int kFewMinTiles = 4;  // tiles a run holds at least: a part costs as much to join as a tile to read

template <int kDim>
constexpr int few_stages() { return 256 / kDim; }  // 16 KB a warp
template <int kDim>
constexpr int few_stage_bytes() { return 2 * kWarpKeys * kDim * 2; }
template <int kDim>
constexpr size_t few_smem() { return (size_t)kFewWarps * few_stages<kDim>() * few_stage_bytes<kDim>() + 1024; }

// Tiles of a request in the line; 0: not this kernel's.  (A request whose tokens see nothing has one, for the zeros.)
__device__ __forceinline__ int few_tiles(const ChunkArgs& ka, const Request& rq, TileList<kFewTile>* list) {
  const int rows = rq.n * ka.group;
  if (rows == 0 || rows > ka.few_rows) return 0;
  const TileList<kFewTile> l(rq.first_pos, rq.first_pos + rq.n - 1, ka.a.window, ka.a.sinks);
  if (list) *list = l;
  return max(l.n, 1);
}
// Runs the line of `total` tiles is cut into; run c is [c total / runs, (c + 1) total / runs).
__device__ __forceinline__ int few_runs(long long total, int ctas) {
  return (int)max(1LL, min((long long)ctas, total / kFewMinTiles));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kHalf)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A place in the line of tiles.
struct Cursor {
  int b, h, i, n;  // request, KV head, tile of its list, tiles in the list
  Request rq;
  TileList<kFewTile> list;
  __device__ __forceinline__ Cursor() : b(-1), h(0), i(0), n(0), rq{}, list(-1, -1, 0, 0) {}
  __device__ __forceinline__ void next_request(const ChunkArgs& ka) {
    n = 0;
    while (n == 0 && ++b < ka.a.batch) {
      rq = read_request(ka.a, b, false);
      n = few_tiles(ka, rq, &list);
    }
  }
  __device__ __forceinline__ void next(const ChunkArgs& ka) {
    if (++i < n) return;
    i = 0;
    if (++h < ka.a.num_kv_heads) return;
    h = 0;
    next_request(ka);
  }
};

template <bool kHalf, int kDim, int kMT>
__global__ void __launch_bounds__(kFewThreads, kFewPerSm)
    chunk_attn_few_kernel(const ChunkArgs ka, const __grid_constant__ CUtensorMap tmap) {
  extern __shared__ unsigned char smem_raw[];
  constexpr int kStages = few_stages<kDim>(), kStageBytes = few_stage_bytes<kDim>(), kPlane = kStageBytes / 2;
  constexpr int kHalves = kDim / 64, kGroupBytes = 1024 * kHalves;
  constexpr int kSteps = kDim / 16;
  __shared__ __align__(8) uint64_t full[kFewWarps][kStages];
  __shared__ float s_ml[kFewWarps][16][2];
  __shared__ int s_abort;
  const subspec_chunk_attn_args& a = ka.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = ka.group, H = a.num_kv_heads;
  grid_dep_launch();
  if (blockIdx.x == 0 && warp == 0)
    for (int x = lane; x < a.batch; x += 32) read_request(a, x, true);

  // ---- the line's length, and where this CTA's run begins ----
  long long total = 0;
  int first_tiles = 0;  // of this lane's request among the first 32
#pragma unroll 4
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    const int tiles = b < a.batch ? few_tiles(ka, read_request(a, b, false), nullptr) : 0;
    if (b0 == 0) first_tiles = tiles;
    total += __reduce_add_sync(0xffffffffu, tiles);
  }
  total *= H;
  const int runs = few_runs(total, (int)gridDim.x), run = (int)blockIdx.x;
  if (total == 0 || run >= runs) {
    if (threadIdx.x == 0) ka.few_runs[run] = make_int4(0, 0, 0, 0);
    return;
  }
  const long long g0 = run * total / runs, g1 = (run + 1) * total / runs;
  Cursor at;
  {
    long long rem = g0;
    int b0 = 0;
    for (;; b0 += 32) {
      const int b = b0 + lane;
      const int tiles = b0 == 0 ? first_tiles : b < a.batch ? few_tiles(ka, read_request(a, b, false), nullptr) : 0;
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, (long long)incl * H > rem);
      if (hit) {
        const int src = __ffs(hit) - 1;
        rem -= (long long)__shfl_sync(0xffffffffu, incl - tiles, src) * H;
        at.b = b0 + src - 1;
        break;
      }
      rem -= (long long)__shfl_sync(0xffffffffu, incl, 31) * H;
      if (b0 + 32 >= a.batch) return;  // (total says that this does not happen)
    }
    at.next_request(ka);
    at.h = (int)(rem / at.n);
    at.i = (int)(rem - (long long)at.h * at.n);
  }

  // what the join needs: the run's first (request, head), whether it began in an earlier run, whether it ends in this one
  if (threadIdx.x == 0)
    ka.few_runs[run] = make_int4(at.b, at.h, 0, (at.i > 0 ? 1 : 0) | (at.i + (g1 - g0) >= at.n ? 2 : 0));

  unsigned char* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u) + (size_t)warp * kStages * kStageBytes;
  const int box = ka.box_rows, boxes = box > 0 ? kWarpKeys / box : 0;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], box > 0 ? 1 : 32);
    mbar_init_fence();
    if (warp == 0) s_abort = 0;
  }
  __syncthreads();
  volatile int* abort_flag = &s_abort;

  // ---- the copies of this warp, a few tiles ahead of the arithmetic ----
  Cursor put = at;
  long long put_g = g0;
  const bool copy_v = lane >= boxes;
  const int copy_box = lane - (copy_v ? boxes : 0);
  auto wanted = [&](const TileList<kFewTile>& l, int lo, int hi) { return lo < l.hi && (hi > l.lo || lo < l.snk); };
  auto page_of = [&]() -> int {  // what this lane's copy reads; -2: nothing (zeros)
    if (lane >= 2 * boxes || put_g >= g1) return -2;
    const int kpos = put.list.first_row(put.i) + warp * kWarpKeys + copy_box * box;
    if (!wanted(put.list, kpos, kpos + box)) return -2;
    return a.page_table[(size_t)put.b * a.pages_per_seq + (ka.page_shift >= 0 ? kpos >> ka.page_shift : kpos / a.page_len)];
  };
  int page = page_of();  // always looked up a tile ahead of its use
  auto produce = [&](int s) {
    if (put_g >= g1) return;
    unsigned char* dst = ring + s * kStageBytes;
    const int t0 = put.list.first_row(put.i) + warp * kWarpKeys;
    if (boxes > 0) {
      if (lane == 0) mbar_expect_tx(&full[warp][s], (uint32_t)kStageBytes);
      __syncwarp();
      if (lane < 2 * boxes) {
        const int kpos = t0 + copy_box * box;
        int unit = ka.units, slot = 0;  // outside the tensor: zeros, no memory is touched
        if (page >= 0 && page < a.num_pages) {
          unit = page * ka.page_units + (copy_v ? ka.page_units / 2 : 0) + put.h;
          slot = ka.page_shift >= 0 ? kpos & (a.page_len - 1) : kpos % a.page_len;
        } else if (page != -2) {
          flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
        }
        tma_load_5d(dst + (copy_v ? kPlane : 0) + copy_box * box * kDim * 2, &tmap, slot >> 3, unit,
                    &full[warp][s]);
      }
    } else {  // page lengths that are no multiple of 8: 16-byte copies, row by row
      constexpr int kChunks = kDim / 8;
      for (int x = lane; x < 2 * kWarpKeys * kChunks; x += 32) {
        const int c = x % kChunks, rr = x / kChunks % kWarpKeys, is_v = x / (kChunks * kWarpKeys);
        const int kpos = t0 + rr;
        const unsigned char* src = is_v ? ka.v_base : ka.k_base;
        int bytes = 0;
        if (wanted(put.list, kpos, kpos + 1)) {
          const int pi = kpos / a.page_len, pg = a.page_table[(size_t)put.b * a.pages_per_seq + pi];
          if (pg < 0 || pg >= a.num_pages) {
            flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
          } else {
            bytes = 16;
            src += (size_t)pg * ka.page_stride + (size_t)(kpos - pi * a.page_len) * ka.row_stride + (size_t)put.h * kDim * 2 + c * 16;
          }
        }
        cp_async16(dst + is_v * kPlane + (rr >> 3) * kGroupBytes + (c >> 3) * 1024 + (rr & 7) * 128 + (((c & 7) ^ (rr & 7)) << 4), src,
                   bytes);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[warp][s])) : "memory");
    }
    ++put_g;
    if (put_g < g1) put.next(ka);
    page = page_of();
  };
  for (int s = 0; s < kStages; ++s) produce(s);

  // ---- the arithmetic ----
  constexpr float kOffset = kHalf ? 7.f : 0.f;  // fp16 weights sit 2^7 higher, out of the subnormals
  const float c2 = ka.scale_log2;
  const int r4 = lane >> 2, c4 = lane & 3;
  int s = 0;
  uint32_t ph = 0;
  bool live = true;
  long long g = g0;
  while (g < g1 && live) {
    // a piece: what the run has of one (request, head)
    const int rows = at.rq.n * G, first_i = at.i;
    const int last_pos = at.rq.first_pos + at.rq.n - 1;
    uint32_t q[kMT][kSteps][4];
    int pos[kMT][2];
    float m[kMT][2], l[kMT][2], o[kMT][kDim / 8][4];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 16 * mt + 8 * x + r4, tok = min(row, rows - 1) / G;
        pos[mt][x] = at.rq.first_pos + tok;
        m[mt][x] = -INFINITY, l[mt][x] = 0.f;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(
            reinterpret_cast<const uint16_t*>(a.q) + (size_t)(at.rq.q0 + tok) * a.q_token_stride +
            (size_t)(at.h * G + min(row, rows - 1) - tok * G) * a.q_head_stride);
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
          q[mt][ks][x] = row < rows ? src[8 * ks + c4] : 0u;
          q[mt][ks][x + 2] = row < rows ? src[8 * ks + 4 + c4] : 0u;
        }
      }
#pragma unroll
      for (int d = 0; d < kDim / 8; ++d) o[mt][d][0] = o[mt][d][1] = o[mt][d][2] = o[mt][d][3] = 0.f;
    }
    for (;;) {
      live = __all_sync(0xffffffffu, tc_wait(&full[warp][s], ph, abort_flag));
      if (!live) break;
      unsigned char* stage = ring + s * kStageBytes;
      const int t0 = at.list.first_row(at.i) + warp * kWarpKeys;
      const bool all = t0 + kWarpKeys - 1 <= at.rq.first_pos &&
                       (a.window == 0 || t0 > last_pos - a.window || t0 + kWarpKeys <= a.sinks);
      if (!all) {
        // V rows that no row of the piece sees: whatever the page holds there must not meet a weight of 0
        for (int rr = 0; rr < kWarpKeys; ++rr)
          if (!wanted(at.list, t0 + rr, t0 + rr + 1) && lane < kDim / 8)
            *reinterpret_cast<uint4*>(stage + kPlane + (rr >> 3) * kGroupBytes + (lane >> 3) * 1024 + (rr & 7) * 128 +
                                      ((lane & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
        fence_async_smem();
        __syncwarp();
      }
      const uint32_t k_u32 = smem_u32(stage), v_u32 = k_u32 + kPlane;
      const int mi = lane >> 3, mr = lane & 7;
      float sc[kMT][2][4];
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int x = 0; x < 2; ++x) sc[mt][x][0] = sc[mt][x][1] = sc[mt][x][2] = sc[mt][x][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        uint32_t kb[4];
        const int c = 2 * ks + (mi & 1);
        ldsm4(kb, k_u32 + (uint32_t)((mi >> 1) * kGroupBytes + (c >> 3) * 1024 + mr * 128 + (((c & 7) ^ mr) << 4)));
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          mma16816<kHalf>(sc[mt][0], q[mt][ks], kb[0], kb[1]);
          mma16816<kHalf>(sc[mt][1], q[mt][ks], kb[2], kb[3]);
        }
      }
      uint32_t p[kMT][4];
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        if (!all) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int key = t0 + 8 * x + 2 * c4 + (y & 1), at_row = pos[mt][y >> 1];
              const bool see = key <= at_row && (a.window == 0 || key > at_row - a.window || key < a.sinks);
              sc[mt][x][y] = see ? sc[mt][x][y] : -INFINITY;
            }
        }
        float alpha[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float mx = max3_nan(max3_nan(sc[mt][0][2 * x], sc[mt][0][2 * x + 1], sc[mt][1][2 * x]), sc[mt][1][2 * x + 1], sc[mt][1][2 * x + 1]);
          float y = __shfl_xor_sync(0xffffffffu, mx, 1);
          mx = max3_nan(mx, y, y);
          y = __shfl_xor_sync(0xffffffffu, mx, 2);
          mx = max3_nan(mx, y, y) * c2;  // c2 > 0
          alpha[x] = 1.f;
          if (!(mx <= m[mt][x] + kRescaleAt) || m[mt][x] == -INFINITY) {
            const float m_new = max3_nan(m[mt][x], mx, mx);
            alpha[x] = m[mt][x] == -INFINITY ? 0.f : ex2f(m[mt][x] - m_new);
            m[mt][x] = m_new;
          }
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
          l[mt][0] *= alpha[0], l[mt][1] *= alpha[1];
#pragma unroll
          for (int d = 0; d < kDim / 8; ++d) {
            o[mt][d][0] *= alpha[0], o[mt][d][1] *= alpha[0];
            o[mt][d][2] *= alpha[1], o[mt][d][3] *= alpha[1];
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float u = m[mt][x] == -INFINITY ? 0.f : m[mt][x] - kOffset;  // (-inf: nothing seen yet, every weight 0)
          const float p0 = ex2f(fmaf(sc[mt][0][2 * x], c2, -u)), p1 = ex2f(fmaf(sc[mt][0][2 * x + 1], c2, -u));
          const float p2 = ex2f(fmaf(sc[mt][1][2 * x], c2, -u)), p3 = ex2f(fmaf(sc[mt][1][2 * x + 1], c2, -u));
          l[mt][x] += (p0 + p1) + (p2 + p3);
          p[mt][x] = pack16<kHalf>(p0, p1);
          p[mt][x + 2] = pack16<kHalf>(p2, p3);
        }
      }
#pragma unroll
      for (int dt = 0; dt < kSteps; ++dt) {
        uint32_t vb[4];
        const int c = 2 * dt + (mi >> 1);
        ldsm4t(vb, v_u32 + (uint32_t)((mi & 1) * kGroupBytes + (c >> 3) * 1024 + mr * 128 + (((c & 7) ^ mr) << 4)));
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          mma16816<kHalf>(o[mt][2 * dt], p[mt], vb[0], vb[1]);
          mma16816<kHalf>(o[mt][2 * dt + 1], p[mt], vb[2], vb[3]);
        }
      }
      __syncwarp();
      ++g;
      if (at.i + 1 == at.n || g == g1) break;  // the piece ends: the stage serves the join before it is filled again
      produce(s);
      if (++s == kStages) s = 0, ph ^= 1u;
      ++at.i;
    }
    // ---- the piece's end: the warps' parts are joined, 16 rows at a time, through the stage just read ----
    const bool whole = first_i == 0 && at.i + 1 == at.n;
    const size_t slot = (size_t)2 * run + (first_i == 0 ? 1 : 0);
    if (__syncthreads_or(!live)) {
      live = false;
      break;
    }
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      if (16 * mt >= rows) break;
      float2* mine = reinterpret_cast<float2*>(ring + s * kStageBytes);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float sum = l[mt][x];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int row = 8 * x + r4;
        if (c4 == 0) s_ml[warp][row][0] = m[mt][x], s_ml[warp][row][1] = sum;
#pragma unroll
        for (int d = 0; d < kDim / 8; ++d)
          mine[row * (kDim / 2) + ((4 * d + c4) ^ (r4 << 2))] = make_float2(o[mt][d][2 * x], o[mt][d][2 * x + 1]);
      }
      __syncthreads();
      const int row = (int)threadIdx.x >> 3, grow = 16 * mt + row, tok = min(grow, rows - 1) / G;
      float mstar = -INFINITY, w[kFewWarps], lsum = 0.f;
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k)
        if (s_ml[k][row][1] != 0.f) mstar = max3_nan(mstar, s_ml[k][row][0], s_ml[k][row][0]);
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k) {
        const float lk = s_ml[k][row][1];
        w[k] = lk != 0.f ? ex2f(s_ml[k][row][0] - mstar) : 0.f;
        lsum += w[k] * lk;
      }
      const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
      const int row_pos = at.rq.first_pos + tok;
      const int t = at.rq.q0 + tok, head = at.h * G + min(grow, rows - 1) - tok * G;
      const unsigned char* all_rings = ring - (size_t)warp * kStages * kStageBytes + s * kStageBytes;
      bool odd = lsum == 0.f;
#pragma unroll
      for (int j = 0; j < kDim / 64; ++j) {
        const int ch = ((int)threadIdx.x & 7) + 8 * j;
        float acc[8] = {};
#pragma unroll
        for (int k = 0; k < kFewWarps; ++k) {
          if (w[k] == 0.f) continue;  // (a warp that saw nothing)
          const float4* src = reinterpret_cast<const float4*>(all_rings + (size_t)k * kStages * kStageBytes) + row * (kDim / 4) +
                              2 * (ch ^ (row & 7));
          const float4 x = src[0], y = src[1];
          acc[0] += w[k] * x.x, acc[1] += w[k] * x.y, acc[2] += w[k] * x.z, acc[3] += w[k] * x.w;
          acc[4] += w[k] * y.x, acc[5] += w[k] * y.y, acc[6] += w[k] * y.z, acc[7] += w[k] * y.w;
        }
        if (whole) {
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            acc[x] = row_pos < 0 ? 0.f : acc[x] * inv;
            odd = odd || !(fabsf(acc[x]) < INFINITY);
          }
          if (grow < rows) {
            const uint4 v = make_uint4(pack16<kHalf>(acc[0], acc[1]), pack16<kHalf>(acc[2], acc[3]), pack16<kHalf>(acc[4], acc[5]),
                                       pack16<kHalf>(acc[6], acc[7]));
            reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + (size_t)t * a.o_token_stride + (size_t)head * a.o_head_stride)[ch] = v;
          }
        } else {
          float4* dst = reinterpret_cast<float4*>(ka.few_o + (slot * (16 * kMT) + grow) * kDim) + 2 * ch;
          dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
          dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
          if (ch == 0) {
            ka.few_ml[(slot * (16 * kMT) + grow) * 2] = mstar;
            ka.few_ml[(slot * (16 * kMT) + grow) * 2 + 1] = lsum;
          }
        }
      }
      // 0 * inf from a V row that only other rows of the tile see, or scores of -inf alone: key by key
      uint32_t again = __ballot_sync(0xffffffffu, whole && grow < rows && odd && lsum == lsum && row_pos >= 0);
      __syncwarp();  // what eight lanes wrote of such a row lies before what all 32 write over it
      while (again) {
        const int src = __ffs(again) - 1;
        again &= ~(0xffu << (src & ~7));  // the eight lanes of a row
        attn_row<kHalf, kDim>(ka, at.b, __shfl_sync(0xffffffffu, row_pos, src), __shfl_sync(0xffffffffu, t, src),
                              __shfl_sync(0xffffffffu, head, src));
      }
      __syncthreads();
    }
    fence_async_smem();  // the stage goes back to the copies
    __syncwarp();
    produce(s);
    if (++s == kStages) s = 0, ph ^= 1u;
    if (g < g1) at.next(ka);
  }
  if (!live) {  // gave up: the copies in flight land before the CTA leaves
    if (box == 0) cp_async_wait<0>();
    for (int x = 0; x < kStages && box > 0; ++x)
      for (uint32_t y = 0; y < 2; ++y) mbar_wait_bounded(&full[warp][x], y);
    if (threadIdx.x == 0) flag(a.dev_status, SUBSPEC_DEV_TIMEOUT);
  }
}

// Joins the (request, KV head)s that lie in several runs: a warp per (run that holds the end of one, row).
template <bool kHalf, int kDim>
__global__ void __launch_bounds__(128) chunk_few_join_kernel(const ChunkArgs ka) {
  const subspec_chunk_attn_args& a = ka.a;
  const int lane = threadIdx.x & 31, G = ka.group, grow = (int)(blockIdx.y * 4 + (threadIdx.x >> 5));
  grid_dep_launch();  // (the kernel for many rows needs nothing of this one's)
  grid_dep_wait();
  const int4 rec = ka.few_runs[blockIdx.x];
  if (rec.w != 3) return;
  const int c1 = (int)blockIdx.x;
  int c0 = c1;
  for (bool more = true; more;) {  // back over the runs that lie inside it, 32 at a time, to the one where it begins
    const int c = c0 - 1 - lane;
    const uint32_t stop = __ballot_sync(0xffffffffu, c <= 0 || ka.few_runs[c].w != 1);
    more = stop == 0;
    c0 -= more ? 32 : __ffs(stop);
  }
  const int b = rec.x;
  const Request rq = read_request(a, b, false);
  const int i = grow / G, t = rq.q0 + i, head = rec.y * G + grow - i * G, pos = rq.first_pos + i;
  if (i >= rq.n) return;
  constexpr int kPer = kDim / 32;
  auto row_of = [&](int c) { return ((size_t)2 * c + (c == c0 ? 1 : 0)) * ka.few_rows + grow; };
  float mstar = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) {
    const float2 ml = reinterpret_cast<const float2*>(ka.few_ml)[row_of(c)];
    if (ml.y != 0.f) mstar = max3_nan(mstar, ml.x, ml.x);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float y = __shfl_xor_sync(0xffffffffu, mstar, d);
    mstar = max3_nan(mstar, y, y);
  }
  float acc[kPer] = {}, lsum = 0.f;
#pragma unroll 8
  for (int c = c0; c <= c1; ++c) {
    const size_t r = row_of(c);
    const float2 ml = reinterpret_cast<const float2*>(ka.few_ml)[r];
    float o[kPer];
    if (kPer == 4)
      *reinterpret_cast<float4*>(o) = reinterpret_cast<const float4*>(ka.few_o + r * kDim)[lane];
    else
      *reinterpret_cast<float2*>(o) = reinterpret_cast<const float2*>(ka.few_o + r * kDim)[lane];
    const float w = ml.y == 0.f ? 0.f : ex2f(ml.x - mstar);  // (0: nothing seen in this part)
    lsum += w == 0.f ? 0.f : w * ml.y;
#pragma unroll
    for (int x = 0; x < kPer; ++x) acc[x] += w == 0.f ? 0.f : w * o[x];
  }
  const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
  bool odd = lsum == 0.f;
#pragma unroll
  for (int x = 0; x < kPer; ++x) {
    acc[x] *= inv;
    odd = odd || !(fabsf(acc[x]) < INFINITY);
  }
  if (__any_sync(0xffffffffu, odd) && lsum == lsum && pos >= 0) {
    attn_row<kHalf, kDim>(ka, b, pos, t, head);
    return;
  }
  uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + (size_t)t * a.o_token_stride +
                                              (size_t)head * a.o_head_stride);
#pragma unroll
  for (int x = 0; x < kPer / 2; ++x) out[lane * (kPer / 2) + x] = pack16<kHalf>(acc[2 * x], acc[2 * x + 1]);
}

template <bool kHalf, int kDim, int kMT>
int launch(ChunkArgs& ka, cudaStream_t stream) {
  const int rc = allow_smem<chunk_attn_few_kernel<kHalf, kDim, kMT>>(few_smem<kDim>());
  if (rc) return rc;
  CUtensorMap tmap;
  chunk_tensor_map(ka, kWarpKeys, &tmap);
  chunk_attn_few_kernel<kHalf, kDim, kMT><<<kFewCtas, kFewThreads, few_smem<kDim>(), stream>>>(ka, tmap);
  const int launched = cuda_check(cudaGetLastError());
  if (launched) return launched;
  const long long rows = (long long)ka.a.max_q_len * ka.group;
  return launch_dependent(chunk_few_join_kernel<kHalf, kDim>, dim3(kFewCtas, (unsigned)((rows < 16 * kMT ? rows : 16 * kMT) + 3) / 4),
                          dim3(128), 0, stream, ka);
}

template <int kMT>
int launch_mt(ChunkArgs& ka, cudaStream_t stream) {
  if (ka.a.dtype == SUBSPEC_F16) return ka.a.head_dim == 128 ? launch<true, 128, kMT>(ka, stream) : launch<true, 64, kMT>(ka, stream);
  return ka.a.head_dim == 128 ? launch<false, 128, kMT>(ka, stream) : launch<false, 64, kMT>(ka, stream);
}

}  // namespace

size_t chunk_few_scratch_bytes(const ChunkArgs& ka) {
  return kFewCtas * sizeof(int4) + (size_t)2 * kFewCtas * ka.few_rows * (ka.a.head_dim + 2) * sizeof(float);
}

int launch_chunk_few(ChunkArgs& ka, float* scratch, cudaStream_t stream) {
  ka.few_runs = reinterpret_cast<int4*>(scratch);
  ka.few_o = reinterpret_cast<float*>(ka.few_runs + kFewCtas);
  ka.few_ml = ka.few_o + (size_t)2 * kFewCtas * ka.few_rows * ka.a.head_dim;
  return ka.few_rows == 16 ? launch_mt<1>(ka, stream) : launch_mt<2>(ka, stream);
}

}  // namespace subspec
