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
// The work of the call is one line of row tiles -- requests, their KV heads, their tiles of 256 rows one behind the
// other, each as long as it has cache tiles (and one more for its start and end) -- cut into equal runs, one per CTA, one
// CTA an SM: 224 row tiles are otherwise two rounds of 148 SMs, the second half empty, and a lone short chunk behind a
// long cache keeps four.  A row tile that a cut falls into leaves unnormalised parts in scratch, which a second kernel
// joins; short row tiles are not cut.
//
// The rows of the problem are (token, head of the GQA group) pairs, token-major, so that a block of 128 rows is a run
// of neighbouring tokens: their KV head's cache rows are read once for the whole group, and the causal border crosses
// few tiles.  A row tile = 256 rows of one (request, KV head), two blocks that share every K / V tile of 128 cache rows:
//
//   warps 0-15  softmax, eight warps per block: thread = query row = lane of tensor memory, two warps per row, one for
//               either half of a tile's 128 scores.  A thread writes P = 2^(S c - m) as 16-bit pairs over the first of the
//               columns it read and sums P in fp32.  (P is rounded to the cache's type because an MMA takes both operands
//               in it: P in two 16-bit terms would be half as many MMAs again.  Half a step a weight; against 64 bits
//               the output is off by 2.3e-3 of its norm in bf16 and 2.8e-4 in fp16, where rounding it alone makes 1.7e-3
//               and 2.1e-4.)  m, the reference point, is the maximum of the first tile, and moves
//               (the row of O in tensor memory is rescaled) only when the sums say that a later score has run far ahead of
//               it.  They also bring the block's Q and write its output.
//   warps 16, 17  issue the MMAs of a block each, in turns: O += P V (P from tensor memory, V MN-major as the cache has
//               it), then S = Q K^T of the next tile (128 x 128 x head_dim, both K-major in shared memory) over the P just
//               consumed: the MMAs of a thread run in order.  While one block is in its softmax the other's MMAs run.
//   warp 18     brings the K tiles, warp 19 the V tiles, into a ring of five entries, K(0), V(0), K(1), V(1), ...;
//               warp 18 also walks the run and hands out its pieces.
//
// What it measured (B200, bf16, 28 query heads on 4 KV heads of 128 dims): 2048 tokens behind 30720 rows 870 us = 1.07
// PFLOP/s call after call, at the power cap (1.64 GHz; on another card 896); a few calls alone 754 us = 1236 TFLOP/s, 0.74
// of the card's cuBLAS burst.  A tile takes 2058 cycles of MMAs for both blocks and about 3600 in all.  64 prompts of 30
// to 60 tokens on 32/8 heads 44 us, 256 drafts of 3 to 6 tokens behind 50 to 200 rows 81 us (floors 9 and 13; in a launch
// list 45 and 74 for this kernel, which takes three or four, and seven, short row tiles one after the other, and 7 for a
// join that finds nothing to do).  Steps on the way, same case: an issuer per block without turns 1306 us (both blocks in
// their softmax at once); one issuer 1015; runs over all SMs instead of a CTA per row tile, half a tile of scores in
// registers instead of spilling, turns 790; two warps per row 756; Q rows by neighbouring lanes and 32-byte stores 745;
// waits that leave no warp behind when one gives up 754.  Tried and no faster: separate score buffers for the tile's
// halves (S of 64 columns: MMAs 2484 cycles a tile) 740 to 850; a share of the exponentials as a polynomial on the FMA
// pipe 737 to 760.
//
// A tile lies in shared memory as 16 groups of 8 rows; a group as one (head_dim 64) or two halves of 64 dims, a half as
// 8 rows of 128 bytes under the 128-byte swizzle: the layout the tensor cores read either way round, in which the rows
// of a page are contiguous -- so that one tensor copy brings a page's rows of one head, whatever the page length (a
// multiple of 8), instead of one copy per half.
//
// Tensor memory: per block 256 columns, S | O, 128 each (O: head_dim).
constexpr int kTileKeys = 128, kHalfKeys = kTileKeys / 2;
constexpr int kBlockRows = 128;
constexpr int kCtaRows = 2 * kBlockRows;
constexpr int kRing = 5;
constexpr int kSoftmaxWarps = 16;
constexpr int kChunkThreads = 32 * (kSoftmaxWarps + 4);
constexpr int kIssuerWarp = kSoftmaxWarps, kLoadWarp = kIssuerWarp + 2;
constexpr uint32_t kBlockCols = 256, kOCol = 128;
constexpr int kMinRun = 4;    // cost a run holds at least (its cache tiles and one for each row tile)
// Row tiles of up to so many cache tiles are not cut where runs are long.  (Measured at 0, 4, 8 and 16: six prompts 232, 233,
// 235, 228 us, two windowed prompts 192, 192, 190, 186; short chunks, drafts and mixed batches alike within 2 %.)
constexpr int kSnapTiles = 8;
constexpr int kGroups = 64;    // groups of requests whose costs are summed up side by side

template <int kDim>
constexpr size_t tc_smem() {
  return (size_t)kCtaRows * kDim * 2 + (size_t)kRing * kTileKeys * kDim * 2 + 1024;
}

// A sector: 32 bytes to an address that is a multiple of 32.
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// The two warps of a row: a barrier, and one that tells both whether either has a thread with `x`.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_or(int id, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)x), "r"(id)
      : "memory");
  return r != 0;
}

// First cache row of entry i of a tile list.
__device__ __forceinline__ int list_row(int s_tiles, int m0, int i) { return (i < s_tiles ? i : m0 + i - s_tiles) * kTileKeys; }

// A row tile: rows [row0, row0 + 256) of the n * group (token, head) rows of a request under one KV head.
struct RowTile {
  int row0, rows;             // first row, rows of the request
  TileList<kTileKeys> list;   // the cache tiles its rows see
  int n;                      // at least one: a tile whose rows see nothing still writes its zeros
  RowTile() = default;
  __device__ __forceinline__ RowTile(const ChunkArgs& ka, const Request& rq, int qt)
      : row0(qt * kCtaRows),
        rows(rq.n * ka.group),
        list(rq.first_pos + by_group(ka, row0), rq.first_pos + by_group(ka, min(row0 + kCtaRows, rows) - 1), ka.a.window, ka.a.sinks) {
    n = max(list.n, 1);
  }
  __device__ __forceinline__ int cost() const { return n + 1; }
};
__device__ __forceinline__ int row_tiles(const ChunkArgs& ka, const Request& rq) {
  const int rows = rq.n * ka.group;
  return rows > ka.few_rows ? (rows + kCtaRows - 1) / kCtaRows : 0;
}

// A place in the line: cache tile i of row tile qt of (request b, KV head h); b == batch: the end.
struct Place {
  int b, h, qt, i;
};

// What the requests of [b0, b1) cost under one KV head (a warp).
__device__ long long requests_cost(const ChunkArgs& ka, int b0, int b1) {
  const int lane = threadIdx.x & 31;
  if (b0 >= b1) return 0;
  long long sum = 0;
  for (int c0 = b0; c0 < b1; c0 += 32) {
    const Request mine = c0 + lane < b1 ? read_request(ka.a, c0 + lane, false) : Request{};
    uint32_t todo = __ballot_sync(0xffffffffu, row_tiles(ka, mine) > 0);
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      const Request rq = shfl_request(mine, src);
      const int nqt = row_tiles(ka, rq);
      for (int qt = lane; qt < nqt; qt += 32) sum += RowTile(ka, rq, qt).cost();
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return sum;
}

// The place `g` into the line (a warp).  Places inside short row tiles, or next to an edge, move to the edge: every CTA
// finds the same.
__device__ Place locate(const ChunkArgs& ka, long long g, const long long* group_cost, int group_size, int snap) {
  const int lane = threadIdx.x & 31, H = ka.a.num_kv_heads;
  // the group: kGroups <= 64, two per lane
  const long long c0 = group_cost[2 * lane], c1 = group_cost[2 * lane + 1];
  long long incl = c0 + c1;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  Place at{ka.a.batch, 0, 0, 0};
  const uint32_t hits = __ballot_sync(0xffffffffu, incl * H > g);
  if (!hits) return at;
  const int src = __ffs(hits) - 1;
  long long before = incl - c0 - c1;
  const bool second = (before + c0) * H <= g;
  if (second) before += c0;
  g -= __shfl_sync(0xffffffffu, before, src) * H;
  const int grp = 2 * src + __shfl_sync(0xffffffffu, (int)second, src);
  for (int b = grp * group_size; b < min((grp + 1) * group_size, ka.a.batch); ++b) {
    const long long cost = group_size == 1 ? group_cost[grp] : requests_cost(ka, b, b + 1);
    if (g >= cost * H) {
      g -= cost * H;
      continue;
    }
    at.b = b;
    at.h = (int)(g / cost);
    g -= at.h * cost;
    const Request rq = read_request(ka.a, b, false);
    const int nqt = row_tiles(ka, rq);
    for (int q0 = 0; q0 < nqt; q0 += 32) {
      const RowTile tile(ka, rq, min(q0 + lane, nqt - 1));
      int incl = q0 + lane < nqt ? tile.cost() : 0;
      const int own = incl;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, incl > g);
      if (hit) {
        const int src = __ffs(hit) - 1;
        at.qt = q0 + src;
        const int n = __shfl_sync(0xffffffffu, tile.n, src);
        at.i = (int)(g - __shfl_sync(0xffffffffu, incl - own, src));
        if (n <= snap)
          at.i = 2 * at.i < n ? 0 : n;
        else if (at.i < 2 || at.i > n - 2)
          at.i = at.i < 2 ? 0 : n;
        if (at.i == n) {  // the next row tile's start
          at.i = 0;
          if (++at.qt == nqt) {
            at.qt = 0;
            if (++at.h == H) at.h = 0, ++at.b;
          }
        }
        return at;
      }
      g -= __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  at.b = ka.a.batch;  // (the groups' costs say that this does not happen)
  return at;
}

// A piece: what a run has of one row tile.  Warp 18 walks the run and hands the pieces to the other warps through shared
// memory (a walker of thirty words in every warp pushes the softmax's scores out of the registers).
struct Piece {
  int valid;                    // 0: the run is over
  int b, h, q0, first_pos, kv_len;
  int row0, rows;               // rows [row0, row0 + 256) of the request's
  int i0, ntiles, whole;        // cache tiles [i0, i0 + ntiles) of the row tile's list; all of them?
  int s_tiles, m0, hi, lo, snk;  // the list (TileList)
  int last_seen[2];             // of the piece's tiles, the last one that a row of the block sees; -1: none
};
constexpr int kPieces = 4;  // in flight
constexpr int kPieceReaders = kSoftmaxWarps + 3;

struct Pieces {
  Place at, end;  // the run ends in front of `end`
  Request rq;
  RowTile tile;
  int nqt, i0, ntiles;  // row tiles of the request; this piece's cache tiles [i0, i0 + ntiles) of the row tile's list
  bool fresh;
  __device__ __forceinline__ Pieces(const Place& from, const Place& to) : at(from), end(to), rq{}, nqt(0), i0(0), ntiles(0), fresh(true) {}
  __device__ __forceinline__ bool next(const ChunkArgs& ka) {
    if (fresh) {
      request(ka);
    } else if (++at.qt == nqt) {
      at.qt = 0;
      if (++at.h == ka.a.num_kv_heads) {
        at.h = 0;
        ++at.b;
        request(ka);
      }
    }
    if (at.b > end.b || at.b >= ka.a.batch) return false;
    const bool in_last = at.b == end.b && at.h == end.h && at.qt == end.qt;
    if (at.b == end.b && !in_last && (at.h > end.h || (at.h == end.h && at.qt > end.qt))) return false;
    tile = RowTile(ka, rq, at.qt);
    i0 = fresh ? at.i : 0;
    fresh = false;
    ntiles = (in_last ? end.i : tile.n) - i0;
    return ntiles > 0;
  }
  __device__ __forceinline__ Piece piece(bool any) const {
    return Piece{any, at.b, at.h, rq.q0, rq.first_pos, rq.kv_len, tile.row0, tile.rows, i0, ntiles, ntiles == tile.n,
                 tile.list.s_tiles, tile.list.m0, tile.list.hi, tile.list.lo, tile.list.snk, {-1, -1}};
  }

 private:
  __device__ __forceinline__ void request(const ChunkArgs& ka) {  // the next one with row tiles
    for (nqt = 0; at.b < ka.a.batch && at.b <= end.b; ++at.b) {
      rq = read_request(ka.a, at.b, false);
      nqt = row_tiles(ka, rq);
      if (nqt > 0) return;
      at.h = at.qt = at.i = 0;
    }
  }
};

template <bool kHalf, int kDim>
__global__ void __launch_bounds__(kChunkThreads, 1)
    chunk_attn_tc_kernel(const ChunkArgs ka, const __grid_constant__ CUtensorMap tmap) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kRing], empty[kRing], s_ready[2], p_ready[2], o_done[2], my_turn[2], q_ready[2], fix, drained[2];
  __shared__ __align__(8) uint64_t pc_full[kPieces], pc_empty[kPieces], pair_move[8];
  __shared__ union {
    long long cost[kGroups];  // of the groups of requests; then
    float row[kCtaRows];      // what the two warps of a row tell each other
  } s_words;
  __shared__ uint32_t s_move[8];  // per pair of warps: the tile in front of which the reference points are to move
  __shared__ Place s_place[2];
  __shared__ Piece s_piece[kPieces];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  constexpr int kHalves = kDim / 64;
  constexpr int kGroupBytes = 1024 * kHalves;           // 8 rows of a tile
  constexpr int kTileBytes = kTileKeys * kDim * 2;
  constexpr int kQHalfBytes = kBlockRows * 128;         // 64 dims of a Q block's rows
  constexpr int kQBlockBytes = kHalves * kQHalfBytes;
  const subspec_chunk_attn_args& a = ka.a;
  const int G = ka.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, run = (int)blockIdx.x;
  grid_dep_launch();
  // lengths that do not fit are reported once a launch
  auto report = [&]() {
    if (run == 0)
      for (int x = lane; x < a.batch; x += 32) read_request(a, x, true);
  };

  // ---- this CTA's run of the line ----
  const int group_size = (a.batch + kGroups - 1) / kGroups;
  for (int g = warp; g < kGroups; g += kChunkThreads / 32) {
    const long long c = requests_cost(ka, min(g * group_size, a.batch), min((g + 1) * group_size, a.batch));
    if (lane == 0) s_words.cost[g] = c;
  }
  unsigned char* qtiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* ring = qtiles + 2 * kQBlockBytes;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);  // both blocks' issuers let go of an entry
    }
    for (int k = 0; k < 2; ++k) {
      mbar_init(&s_ready[k], 1);
      mbar_init(&p_ready[k], kSoftmaxWarps / 2);
      mbar_init(&o_done[k], 1);
      mbar_init(&q_ready[k], kSoftmaxWarps / 2);
      mbar_init(&my_turn[k], 1);
      mbar_init(&drained[k], 1);
    }
    for (int k = 0; k < kPieces; ++k) {
      mbar_init(&pc_full[k], 1);
      mbar_init(&pc_empty[k], kPieceReaders);
    }
    mbar_init(&fix, 1);
    for (int k = 0; k < 8; ++k) {
      mbar_init(&pair_move[k], 2);
      s_move[k] = 0xffffffffu;
    }
    mbar_init_fence();
    s_abort = 0;
  }
  __syncthreads();
  long long total = s_words.cost[lane] + s_words.cost[lane + 32];
#pragma unroll
  for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
  total *= a.num_kv_heads;
  const int runs = (int)max(1LL, min((long long)gridDim.x, total / kMinRun));
  // row tiles of up to so many cache tiles are not cut: a part costs about two tiles, an uneven run up to half the tile
  // (a half or an eighth of the run instead of a quarter: the same within 2 %)
  const int snap = (int)min((long long)kSnapTiles, total / runs / 4);
  int4* record = ka.runs + run;
  if (total == 0 || run >= runs) {
    if (warp == 0) report();
    if (threadIdx.x == 0) *record = make_int4(0, 0, 0, 0);
    grid_dep_wait();
    return;
  }
  if (warp < 2) {
    const int c = run + warp;
    const Place p = c < runs ? locate(ka, c * total / runs, s_words.cost, group_size, snap) : Place{a.batch, 0, 0, 0};
    if (lane == 0) s_place[warp] = p;
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

  // Every wait is bounded, and lanes may give up one by one: a warp goes on or leaves as a whole, with no lane behind at a
  // vote or a warp barrier of the others.
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag)) != 0; };

  // Reading the pieces: peek waits for the next one, pop lets go of its slot.
  int pc_slot = 0;
  uint32_t pc_phase = 0;
  auto peek = [&]() -> const Piece* {
    return warp_wait(&pc_full[pc_slot], pc_phase) && s_piece[pc_slot].valid ? &s_piece[pc_slot] : nullptr;
  };
  auto pop = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&pc_empty[pc_slot]);
    if (++pc_slot == kPieces) pc_slot = 0, pc_phase ^= 1u;
  };
  // Rows of a block of a piece: cache rows of its first and last token; a block without rows sees nothing.
  auto block_pos = [&](const Piece& pc, int blk, int& first, int& last) {
    const int r0 = pc.row0 + blk * kBlockRows;
    first = pc.first_pos + by_group(ka, r0);
    last = r0 < pc.rows ? pc.first_pos + by_group(ka, min(r0 + kBlockRows, pc.rows) - 1) : -1;
  };
  // Whether a block's rows see anything of tile row t0, and whether all of them see all of it.
  auto block_sees = [&](int first, int last, int t0) {
    return t0 <= last && (a.window == 0 || t0 + kTileKeys - 1 > first - a.window || t0 < a.sinks);
  };
  auto block_sees_all = [&](int first, int last, int t0) {
    return t0 + kTileKeys - 1 <= first && (a.window == 0 || t0 > last - a.window || t0 + kTileKeys <= a.sinks);
  };

  if (warp < kSoftmaxWarps) {
    // ================= softmax =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int blk = warp >> 3, half = (warp >> 2) & 1, rr = (warp & 3) * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)blk * kBlockCols;
    const uint32_t s_addr = lane_base + (uint32_t)(half * kHalfKeys);
    const uint32_t o_addr = lane_base + kOCol + (uint32_t)(half * (kDim / 2));  // its half of the dims, too
    const float c2 = ka.scale_log2;
    const uint64_t c2p = f2_pack(c2, c2);
    // fp16 weights sit 2^7 higher, out of the subnormals
    constexpr float kOffset = kHalf ? 7.f : 0.f;
    // Weights need a reference point near the row's maximum, not the maximum itself, and every weight is positive, so that
    // the sum of a tile's tells whether any is too large: no tile but a row's first is searched for its maximum.
    // bf16 (and the fp32 sums) hold weights of up to 2^100 as well as 1.  A tile that passes 2^40 makes the reference point
    // move in front of the next tile; one that passes 2^100 (scores that rise by 69 beyond a row's reference within one
    // tile) spoils the row, which is done over at the end.
    // fp16 holds 2^15: there a tile that does not fit is done again at once, against its own maximum.
    constexpr float kSumLimit = kHalf ? 32768.f : 1.0995116e12f, kSpoilt = 1.2676506e30f;
    const int pair = 1 + blk * 4 + (warp & 3);  // the named barrier of the two warps with these rows
    float& word = s_words.row[blk * kBlockRows + rr];
    // x of the one and of the other, put together by the second
    auto exchange = [&](float x, auto&& join) {
      if (half == 0) word = x;
      pair_sync(pair);
      if (half == 1) word = x = join(x, word);
      pair_sync(pair);
      return half == 0 ? word : x;
    };
    // The named barriers of a pair have no limit: they stand only where both warps come whatever either of them gave up
    // on, for reasons that both know.  Where one cannot tell whether the other comes, they meet at a barrier with one.
    uint32_t moves = 0;
    auto meet_to_move = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair_move[pair - 1]);
      return warp_wait(&pair_move[pair - 1], moves++ & 1u);
    };
    uint32_t seen = 0, finished = 0;  // tiles, and pieces with any, that this block has worked on
    // The warps of a block bring its rows of Q of a piece, sixteen each (rows that do not exist: zeros): neighbouring lanes
    // bring neighbouring chunks.  (A row per thread makes 32 scattered accesses of every instruction: 3500 cycles.)
    auto load_q = [&](const Piece& pc) {
      constexpr int kChunks = kDim / 8, kPass = 32 / kChunks;  // chunks of a row, rows at once
      const int c = lane % kChunks, r0 = (warp & 7) * 16 + lane / kChunks;
      int row = pc.row0 + blk * kBlockRows + r0, tok = by_group(ka, row), g = row - tok * G;
      unsigned char* d = qtiles + blk * kQBlockBytes + (c >> 3) * kQHalfBytes;
#pragma unroll 2
      for (int x = 0; x < 16; x += kPass) {
        const int r = r0 + x;
        const bool ok = row < pc.rows;
        const unsigned char* src = reinterpret_cast<const unsigned char*>(a.q);
        if (ok) src += 2 * ((size_t)(pc.q0 + tok) * a.q_token_stride + (size_t)(pc.h * G + g) * a.q_head_stride) + c * 16;
        cp_async16(d + r * 128 + (((c & 7) ^ (r & 7)) << 4), src, ok ? 16 : 0);
        row += kPass;
        g += kPass;
        while (g >= G) g -= G, ++tok;
      }
      cp_async_commit();
    };
    auto hand_q = [&]() {  // ... and the block's issuer may read it
      cp_async_wait<0>();
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[blk]);
    };
    // whether every row of the output begins on a sector
    const bool wide_out = !((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(2 * a.o_token_stride) | (uintptr_t)(2 * a.o_head_stride)) & 31u);
    bool live = true;
    // Q is handed over for the pieces that the block sees something of, and for no others: see the issuer's wait for it.
    const Piece* first = peek();
    if (first && first->last_seen[blk] >= 0) {
      load_q(*first);
      hand_q();
    }
    while (live) {
      const Piece* now = peek();
      if (pair_or(pair, now == nullptr)) break;  // (both or neither: they meet at barriers)
      const int row = now->row0 + blk * kBlockRows + rr;
      const bool row_ok = row < now->rows, block_ok = now->row0 + blk * kBlockRows < now->rows, whole = now->whole;
      const int tok = by_group(ka, row), head = now->h * G + row - tok * G, t = now->q0 + tok, b = now->b;
      int bfirst, blast;
      block_pos(*now, blk, bfirst, blast);
      const int pos = min(now->first_pos + tok, blast);  // rows that do not exist look like the last one
      const int ntiles = now->ntiles, i0 = now->i0, s_tiles = now->s_tiles, m0 = now->m0;
      pop();
      float m = -INFINITY, l = 0.f;
      uint32_t done = 0;       // tiles of this piece
      bool all_begun = false;  // no row of the warp without a reference point
      for (int i = 0; i < ntiles; ++i) {
        const int t0 = list_row(s_tiles, m0, i0 + i);
        if (!block_sees(bfirst, blast, t0)) continue;
        live = warp_wait(&s_ready[blk], seen & 1u);
        tc_fence_after();
        const bool masked = !block_sees_all(bfirst, blast, t0);
        auto hide = [&](int c, uint32_t (&r)[32]) {
          const int p0 = t0 + half * kHalfKeys + 32 * c;
          uint32_t bits = bits_below(pos + 1 - p0);
          if (a.window > 0) bits &= ~bits_below(pos - a.window + 1 - p0) | bits_below(a.sinks - p0);
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = (bits >> j) & 1u ? r[j] : 0xff800000u;
        };
        auto rescale_o = [&](float alpha) {  // this warp's half of the dims
          // (O is complete up to the tile before: its MMAs were committed together with this tile's scores)
          if (done == 0 || !__any_sync(0xffffffffu, alpha != 1.f)) return;
#pragma unroll 1
          for (int c = 0; c < kDim / 64; ++c) {
            uint32_t rc[32];
            tmem_ld32_async(o_addr + 32 * c, rc);
            tmem_wait_ld_dep(rc);
#pragma unroll
            for (int j = 0; j < 32; ++j) rc[j] = __float_as_uint(__uint_as_float(rc[j]) * alpha);
            tmem_st32(o_addr + 32 * c, rc);
          }
        };
        // The reference points of the rows go to the tile's maximum: of those that have none yet, or of all.
        auto move_to_max = [&](bool all) {
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {  // NaN stays NaN: a NaN score makes the row NaN
            uint32_t r[32];
            tmem_ld32_async(s_addr + 32 * c, r);
            tmem_wait_ld_dep(r);
            if (masked) hide(c, r);
            float mx = __uint_as_float(r[0]);
#pragma unroll
            for (int j = 1; j < 31; j += 2) mx = max3_nan(mx, __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
            top = max3_nan(top, mx, __uint_as_float(r[31]));
          }
          top = exchange(top * c2, [](float x, float y) { return max3_nan(x, y, y); });  // c2 > 0
          float alpha = 1.f;
          if (all || m == -INFINITY) {
            const float m_new = max3_nan(m, top, top);
            alpha = m == -INFINITY ? 0.f : ex2f(m - m_new);
            m = m_new;
            l *= alpha;
          }
          all_begun = __all_sync(0xffffffffu, m != -INFINITY);
          rescale_o(alpha);
        };
        // (m is the same in both warps, so that both find the same here; once all rows have begun they stay so.)
        if (!all_begun && __any_sync(0xffffffffu, m == -INFINITY)) {
          live = !pair_or(pair, !live);
          if (!live) break;
          move_to_max(false);
        } else if (!kHalf && !live) {
          break;  // (fp16: the pair meets below in every tile)
        }
        if (!kHalf && s_move[pair - 1] == seen) {
          // 2^k past the reference point in sum: it moves up by k
          if (half == 0) word = l;
          if (!(live = meet_to_move())) break;
          float both = l;
          if (half == 1) word = both = l + word;
          if (!(live = meet_to_move())) break;
          if (half == 0) both = word;
          const int k = both > 1.f && both < kSpoilt ? (__float_as_int(both) >> 23) - 127 : 0;
          const float alpha = __int_as_float((127 - k) << 23);
          m += (float)k;
          l *= alpha;
          rescale_o(alpha);
        }
        bool moved = false;
        float sum;
        for (;;) {
          const float u = m == -INFINITY ? 0.f : m - kOffset;  // (-inf: every score is -inf, every weight 0)
          const uint64_t nup = f2_pack(-u, -u);
          uint64_t sm2[4] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
          uint32_t pk[2][16];
          auto weights = [&](uint32_t (&r)[32], uint32_t (&pk)[16]) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float x0, x1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), c2p, nup), x0, x1);
              const float p0 = ex2f(x0), p1 = ex2f(x1);  // 2^-inf = 0: hidden entries get the weight 0 exactly
              sm2[j & 3] = f2_add(sm2[j & 3], f2_pack(p0, p1));
              pk[j] = pack16<kHalf>(p0, p1);
            }
          };
          uint32_t ra[32], rb[32];
          tmem_ld32_async(s_addr, ra);
          tmem_wait_ld_dep(ra);
          tmem_ld32_async(s_addr + 32, rb);  // (a load takes 100 to 300 cycles beside the MMAs: under the first's arithmetic)
          if (masked) hide(0, ra);
          weights(ra, pk[0]);
          tmem_wait_ld_dep(rb);
          if (!kHalf) tmem_st16(s_addr, pk[0]);  // over this warp's own scores, which are all in registers
          if (masked) hide(1, rb);
          weights(rb, pk[1]);
          if (!kHalf) tmem_st16(s_addr + 16, pk[1]);
          float e0, e1;
          f2_unpack(f2_add(f2_add(sm2[0], sm2[1]), f2_add(sm2[2], sm2[3])), e0, e1);
          sum = e0 + e1;
          if (kHalf) {  // both warps of a row together: what one finds the other hears
            if (pair_or(pair, !(sum <= kSumLimit) || !live)) {
              live = !pair_or(pair, !live);
              if (!moved && live) {
                moved = true;
                move_to_max(true);
                continue;
              }
            }
            tmem_st16(s_addr, pk[0]);
            tmem_st16(s_addr + 16, pk[1]);
          }
          break;
        }
        if (!kHalf) {
          if (__any_sync(0xffffffffu, !(sum <= kSumLimit)) && lane == 0) s_move[pair - 1] = seen + 1;
          if (sum > kSpoilt) sum = INFINITY;
        }
        l += sum;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[blk]);
        ++done;
        ++seen;
        if (!live) break;
      }
      live = !pair_or(pair, !live);
      l = exchange(l, [](float x, float y) { return x + y; });
      // The block's Q has served its last scores: the next piece's comes while the last MMAs run.
      const Piece* following = live ? peek() : nullptr;
      if (following && following->last_seen[blk] < 0) following = nullptr;
      if (following) load_q(*following);
      // ---- the result: O / l, or the part as it is ----
      if (live && done > 0) live = warp_wait(&o_done[blk], finished++ & 1u);
      if (following) hand_q();
      live = !pair_or(pair, !live);
      if (!live) break;
      if (!block_ok) continue;
      tc_fence_after();
      const float inv = l != 0.f ? 1.f / l : 0.f;
      bool odd = false;  // a value that is not finite although the sum of the weights is
      const size_t prow = ((size_t)2 * run + (i0 == 0 ? 1 : 0)) * kCtaRows + blk * kBlockRows + rr;
      uint16_t* out_row = reinterpret_cast<uint16_t*>(a.out) + (size_t)t * a.o_token_stride + (size_t)head * a.o_head_stride +
                          half * (kDim / 2);
      float* part_row = ka.part_o + prow * kDim + half * (kDim / 2);
      if (!whole && row_ok && half == 0) reinterpret_cast<float2*>(ka.part_ml)[prow] = make_float2(m, l);
      // (Sixteen columns at a time in a loop: this code runs once a row tile, out of a cold instruction cache.)
#pragma unroll 1
      for (int c = 0; c < kDim / 2; c += 16) {
        uint32_t rc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) rc[j] = 0u;
        if (done > 0) {
          tmem_ld16_async(o_addr + c, rc);
          tmem_wait_ld_dep(rc);
        }
        if (!whole) {
          if (row_ok) {
            store32(part_row + c, rc);
            store32(part_row + c + 8, rc + 8);
          }
          continue;
        }
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = pos < 0 ? 0.f : __uint_as_float(rc[2 * j]) * inv, y = pos < 0 ? 0.f : __uint_as_float(rc[2 * j + 1]) * inv;
          odd = odd || !(fabsf(x) < INFINITY) || !(fabsf(y) < INFINITY);
          v[j] = pack16<kHalf>(x, y);
        }
        if (row_ok && wide_out) {
          store32(out_row + c, v);
        } else if (row_ok) {
          reinterpret_cast<uint4*>(out_row + c)[0] = make_uint4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<uint4*>(out_row + c)[1] = make_uint4(v[4], v[5], v[6], v[7]);
        }
      }
      tc_fence_before();
      // 0 * inf from a V row that this row does not see but others of the tile do, or scores of -inf alone: such rows are
      // done over key by key, whole, after the other half of the dims has been written.  (A NaN sum comes from scores the
      // row sees: NaN is the result; an infinite one says that the row is spoilt.)
      const bool bad = whole && row_ok && l == l && (odd || l == INFINITY || (l == 0.f && pos >= 0));
      if (pair_or(pair, bad)) {
        uint32_t again = __ballot_sync(0xffffffffu, exchange(bad ? 1.f : 0.f, [](float x, float y) { return x + y; }) > 0.f);
        again &= half ? 0xffff0000u : 0xffffu;  // the two warps share them out
        while (again) {
          const int src = __ffs(again) - 1;
          again &= again - 1;
          attn_row<kHalf, kDim>(ka, b, __shfl_sync(0xffffffffu, pos, src), __shfl_sync(0xffffffffu, t, src),
                                __shfl_sync(0xffffffffu, head, src));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < kLoadWarp) {
      // ================= MMA issue: a warp per block, an elected lane issues, the blocks take turns =================
      // A thread's MMAs are held up at the tensor pipe (its queue is short), and every wait for a barrier costs a hundred
      // cycles or more even when it is over: while one warp's MMAs run the other does its waiting.  Turns, because with
      // free access the two blocks' MMAs interleave, both get their scores at the same time, and then both sit in their
      // softmax while the tensor cores idle (4660 cycles a tile against 2048 of MMAs).
      const int blk = warp - kIssuerWarp;
      constexpr uint32_t idesc_s = tc_idesc(kBlockRows, kTileKeys, false, kHalf);
      constexpr uint32_t idesc_o = tc_idesc(kBlockRows, kDim, true, kHalf);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0) + (uint32_t)blk * kBlockCols;
      // descriptors: only the address field, the lowest, changes
      const uint64_t q_desc = tc_desc(smem_u32(qtiles) + (uint32_t)(blk * kQBlockBytes), 16);
      const uint64_t k_desc = tc_desc(smem_u32(ring), 16, kGroupBytes), v_desc = tc_desc(smem_u32(ring), 1024, kGroupBytes);
      auto issue_s = [&](int entry) {
        const uint64_t kd = k_desc + (uint64_t)(uint32_t)(entry * (kTileBytes >> 4));
#pragma unroll
        for (int ks = 0; ks < kDim / 16; ++ks)
          tc_mma_f16_ss(tm, q_desc + (uint64_t)(((ks >> 2) * kQHalfBytes + (ks & 3) * 32) >> 4),
                        kd + (uint64_t)(((ks >> 2) * 1024 + (ks & 3) * 32) >> 4), idesc_s, ks > 0 ? 1u : 0u);
        tc_commit(&s_ready[blk]);
      };
      auto issue_o = [&](int entry, bool accumulate) {
        const uint64_t vd = v_desc + (uint64_t)(uint32_t)(entry * (kTileBytes >> 4));
#pragma unroll
        for (int ks = 0; ks < kTileKeys / 16; ++ks)  // 16 cache rows = 8 columns of P; a half's P begins where its scores did
          tc_mma_f16_ta(tm + kOCol, tm + (uint32_t)((ks >> 2) * kHalfKeys + 8 * (ks & 3)), vd + (uint64_t)((ks * 2 * kGroupBytes) >> 4),
                        idesc_o, (accumulate || ks > 0) ? 1u : 0u);
      };
      // (A wait that gave up is noticed at the end of the tile: what is issued until then works on old data in bounds.)
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = tc_wait(bar, parity, abort_flag) && ok;
        __syncwarp();
        tc_fence_after();
      };
      uint32_t turn = blk ^ 1;  // parity of the barrier that says it is this block's turn (block 0 begins)
      auto take_turn = [&]() { wait(&my_turn[blk], turn); };
      auto pass_turn = [&]() {
        if (lane == 0) mbar_arrive(&my_turn[blk ^ 1]);
        turn ^= 1u;
      };
      int e = 0;        // ring entry, in the order they come: K(0), V(0), K(1), ...
      uint32_t ph = 0;  // and its phase
      auto next_entry = [&]() {
        if (++e == kRing) e = 0, ph ^= 1u;
      };
      uint32_t seen = 0, queries = 0;
      bool issued = false;
      while (ok) {
        const Piece* now = peek();
        if (!now) break;
        const int n = now->ntiles, i0 = now->i0, s_tiles = now->s_tiles, m0 = now->m0, last_seen = now->last_seen[blk];
        int bfirst, blast;
        block_pos(*now, blk, bfirst, blast);
        pop();
        auto sees = [&](int i) { return block_sees(bfirst, blast, list_row(s_tiles, m0, i0 + i)); };
        bool begun = false, sees_now = sees(0);
        // One bit tells a phase of a barrier from the next, not from the one after it.  Nothing holds the softmax warps back
        // in a piece of which their block sees nothing (a row tile of up to 128 rows has such a second block): they may be
        // several pieces ahead of this warp.  So such pieces have no phase of q_ready.  Those that have one are at most one
        // apart: the softmax hands over the next behind o_done of the one before, which this warp commits behind its own wait
        // for that one's.  (The others: s_ready and p_ready answer each other, o_done is waited for before the p_ready that
        // the next one needs, my_turn goes to and fro, a slot of the pieces is free when all readers have let go of it.)
        if (last_seen >= 0) wait(&q_ready[blk], queries++ & 1u);
        wait(&full[e], ph);
        take_turn();
        if (elect_one()) {
          if (sees_now) issue_s(e);
          tc_commit(&empty[e]);
        }
        __syncwarp();
        pass_turn();
        issued = true;
        next_entry();
        ok = __all_sync(0xffffffffu, ok);
        for (int i = 0; i < n && ok; ++i) {
          const int ve = e;
          const uint32_t vph = ph;
          next_entry();
          const int ke = e;
          const bool more = i + 1 < n;
          // (Asking a barrier takes 160 cycles even when the answer is yes: these three answers come together.)
          const bool v_there = mbar_test_wait(&full[ve], vph), k_there = !more || mbar_test_wait(&full[ke], ph);
          const bool p_there = !sees_now || mbar_test_wait(&p_ready[blk], seen & 1u);
          const bool sees_next = more && sees(i + 1);
          if (!v_there) ok = tc_wait(&full[ve], vph, abort_flag) && ok;
          if (!k_there) ok = tc_wait(&full[ke], ph, abort_flag) && ok;
          take_turn();  // (comes while P is still being made)
          if (!p_there) ok = tc_wait(&p_ready[blk], seen & 1u, abort_flag) && ok;
          __syncwarp();
          tc_fence_after();
          if (elect_one()) {
            if (sees_now) {
              issue_o(ve, begun);
              if (i == last_seen) tc_commit(&o_done[blk]);
            }
            tc_commit(&empty[ve]);
            if (sees_next) issue_s(ke);  // over the P just consumed: the MMAs of a thread run in order
          }
          __syncwarp();
          pass_turn();
          if (more) {
            if (elect_one()) tc_commit(&empty[ke]);
            __syncwarp();
            next_entry();
          }
          seen += sees_now;
          begun = begun || sees_now;
          sees_now = sees_next;
          ok = __all_sync(0xffffffffu, ok);
        }
      }
      if (issued) {  // whoever gave up: the MMAs in flight finish before tensor memory is freed
        if (elect_one()) tc_commit(&drained[blk]);
        __syncwarp();
        mbar_wait_bounded(&drained[blk], 0);
      }
    } else {
      // ================= K (warp 18) and V (warp 19) tiles =================
      const int is_v = warp - kLoadWarp;
      const int box = ka.box_rows, boxes = box > 0 ? kTileKeys / box : 0;
      const int chunk = lane % (kDim / 8), sub = lane / (kDim / 8);  // row-by-row copies
      constexpr int kRowsPerPass = 32 / (kDim / 8);
      int e = is_v;
      uint32_t ph = 1, fixes = 0;  // the first round finds the entries empty
      bool live = true;
      Pieces walk(s_place[0], s_place[1]);
      uint32_t slot_ph = 1;  // the first round finds the pieces' slots empty, too
      bool first = true;
      while (live) {
        Piece now;
        if (is_v) {
          const Piece* p = peek();
          if (!p) break;
          now = *p;
          pop();
        } else {  // warp 18 walks the run and hands out its pieces
          const bool any = walk.next(ka);
          now = walk.piece(any);
          if (!(live = warp_wait(&pc_empty[pc_slot], slot_ph))) break;
          if (lane == 0) s_piece[pc_slot] = now;
          __syncwarp();
          if (any && lane < 2) {
            int bfirst, blast, i = now.ntiles - 1;
            block_pos(now, lane, bfirst, blast);
            while (i >= 0 && blast >= 0 && !block_sees(bfirst, blast, list_row(now.s_tiles, now.m0, now.i0 + i))) --i;
            s_piece[pc_slot].last_seen[lane] = blast >= 0 ? i : -1;
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&pc_full[pc_slot]);
            // what the join needs: the run's first row tile, whether it began in an earlier run, whether it ends in this
            if (first) *record = make_int4(now.b, now.h, walk.at.qt, any ? (now.i0 > 0 ? 1 : 0) | (now.i0 + now.ntiles == walk.tile.n ? 2 : 0) : 0);
          }
          __syncwarp();
          first = false;
          if (++pc_slot == kPieces) pc_slot = 0, slot_ph ^= 1u;
          if (!any) break;
        }
        const int ntiles = now.ntiles, i0 = now.i0, kv_len = now.kv_len, head = now.h;
        const int s_tiles = now.s_tiles, m0 = now.m0, rows_hi = now.hi, rows_lo = now.lo, rows_snk = now.snk;
        const unsigned char* base = (is_v ? ka.v_base : ka.k_base) + (size_t)head * kDim * 2;
        const int* table = a.page_table + (size_t)now.b * a.pages_per_seq;
        // rows some token of the row tile sees
        auto wanted = [&](int lo, int hi) { return lo < rows_hi && (hi > rows_lo || lo < rows_snk); };
        auto page_of = [&](int i) -> int {  // what this lane's copy of tile i reads; -2: nothing (zeros)
          if (lane >= boxes || i >= ntiles) return -2;
          const int kpos = list_row(s_tiles, m0, i0 + i) + lane * box;
          if (!wanted(kpos, kpos + box)) return -2;
          return table[ka.page_shift >= 0 ? kpos >> ka.page_shift : kpos / a.page_len];
        };
        int page = page_of(0);
        for (int i = 0; i < ntiles; ++i) {
          const int next = page_of(i + 1);  // asked for a tile ahead: a trip to memory
          if (!(live = warp_wait(&empty[e], ph))) break;
          const int t0 = list_row(s_tiles, m0, i0 + i);
          unsigned char* dst = ring + (size_t)e * kTileBytes;
          if (boxes > 0) {
            // rows behind the cache's end, in a box with rows in front of it: whatever the page holds there must not
            // meet a weight of 0 in the V tile
            const int z0 = kv_len - t0, z1 = min((kv_len + box - 1) / box * box - t0, kTileKeys);
            const bool tail = is_v && z0 > 0 && z0 < z1 && wanted(t0 + z1 - box, t0 + z0);
            uint64_t* bar = tail ? &fix : &full[e];
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)kTileBytes);
            __syncwarp();
            if (lane < boxes) {
              const int kpos = t0 + lane * box;
              int unit = ka.units, slot = 0;  // outside the tensor: zeros, no memory is touched
              if (page >= 0 && page < a.num_pages) {
                unit = page * ka.page_units + (is_v ? ka.page_units / 2 : 0) + head;
                slot = ka.page_shift >= 0 ? kpos & (a.page_len - 1) : kpos % a.page_len;
              } else if (page != -2) {
                flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
              }
              tma_load_5d(dst + (size_t)lane * box * kDim * 2, &tmap, slot >> 3, unit, bar);
            }
            if (tail) {
              if (!(live = warp_wait(&fix, fixes & 1u))) {
                mbar_wait_bounded(&fix, fixes & 1u);  // this tile's copies land before the CTA leaves, too
                break;
              }
              ++fixes;
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
              if (kpos < kv_len && wanted(kpos, kpos + 1)) {
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
  // (Launched behind the kernel for few rows it begins as that one's blocks leave, and needs nothing from it; but whoever
  // waits for this kernel waits for that one, too.)
  grid_dep_wait();
}

// Joins the row tiles that were cut: the run that holds a tile's end (blockIdx.x) adds up the runs' unnormalised rows, a
// warp per row, each part weighted by 2^(its reference point - the largest one), and divides by the likewise weighted
// sum of their sums.
template <bool kHalf, int kDim>
__global__ void __launch_bounds__(128) chunk_merge_kernel(const ChunkArgs ka) {
  const subspec_chunk_attn_args& a = ka.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = ka.group;
  grid_dep_wait();
  const int4 rec = ka.runs[blockIdx.x];
  if (rec.w != 3) return;  // not the end of a row tile that began in an earlier run
  const int c1 = (int)blockIdx.x;
  int c0 = c1 - 1;
  while (c0 > 0 && ka.runs[c0].w == 1) --c0;  // runs that lie inside the row tile
  const Request rq = read_request(a, rec.x, false);
  constexpr int kPer = kDim / 32;
  {
    const int r = (int)blockIdx.y * 4 + warp, row = rec.z * kCtaRows + r;
    if (row >= rq.n * G) return;
    const int tok = row / G, head = rec.y * G + row - tok * G, t = rq.q0 + tok, pos = rq.first_pos + tok;
    auto part = [&](int c) { return ((size_t)2 * c + (c == c0 ? 1 : 0)) * kCtaRows + r; };
    float mstar = -INFINITY;
    for (int c = c0 + lane; c <= c1; c += 32) {
      const float2 ml = reinterpret_cast<const float2*>(ka.part_ml)[part(c)];
      if (ml.y != 0.f) mstar = max3_nan(mstar, ml.x, ml.x);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, mstar, d);
      mstar = max3_nan(mstar, y, y);
    }
    float acc[kPer] = {}, lsum = 0.f;
    bool odd = false;
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const float2 ml = reinterpret_cast<const float2*>(ka.part_ml)[part(c)];
      float o[kPer];
#pragma unroll
      for (int x = 0; x < kPer; ++x) o[x] = ka.part_o[part(c) * kDim + lane * kPer + x];
      if (ml.y == 0.f) continue;  // nothing seen in this part
      if (ml.y == INFINITY) {  // spoilt
        odd = true;
        continue;
      }
      const float w = ex2f(ml.x - mstar);
#pragma unroll
      for (int x = 0; x < kPer; ++x) acc[x] += w * o[x];
      lsum += w * ml.y;
    }
    const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
    odd = odd || lsum == 0.f;
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      acc[c] *= inv;
      odd = odd || !(fabsf(acc[c]) < INFINITY);
    }
    if (__any_sync(0xffffffffu, odd) && lsum == lsum && pos >= 0) {  // see the epilogue above
      attn_row<kHalf, kDim>(ka, rec.x, pos, t, head);
      return;
    }
    uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + (size_t)t * a.o_token_stride +
                                                (size_t)head * a.o_head_stride);
#pragma unroll
    for (int c = 0; c < kPer / 2; ++c) out[lane * (kPer / 2) + c] = pack16<kHalf>(acc[2 * c], acc[2 * c + 1]);
  }
}

int check_args(const subspec_chunk_attn_args* args) {
  if (!args || args->struct_size != sizeof(subspec_chunk_attn_args)) return SUBSPEC_EINVAL;
  const subspec_chunk_attn_args& a = *args;
  if (a.batch < 0 || a.tokens < 0 || a.max_q_len < 0 || a.num_q_heads < 1 || a.num_kv_heads < 1 || a.layers < 1 ||
      a.layer < 0 || a.layer >= a.layers || a.num_pages < 1 || a.page_len < 1 || a.pages_per_seq < 1 || a.window < 0 ||
      a.sinks < 0 || !(a.sm_scale > 0.0) ||
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
  // (on average at most 64 rows each).  Measured on 32 requests beside a chunk of 1024 tokens, 4 heads a group, with and
  // without this kernel: 1 token each 134 and 138 us, 2 to 4 tokens 135 and 140; where it finds little or nothing to do its
  // launch and join cost: 4 to 8 tokens 151 and 135, 8 to 16 tokens 148 and 138, 16 to 32 tokens 152 and 142 (it is left out).
  // (A decode step that comes without max_q_len takes both kernels, too: 64 requests 137 us instead of 126.)
  const long long most = (long long)a.max_q_len * ka.group;
  const long long others = (long long)(a.tokens - a.max_q_len) * ka.group;
  ka.few_rows = most <= 16 ? 16 : most <= 32 ? 32 : a.batch > 1 && others <= 64LL * (a.batch - 1) ? 16 : 0;
  if (ka.group > 1) {
    int l = 0;
    while ((1LL << l) < ka.group) ++l;
    ka.group_mul = (uint32_t)(((1ULL << (31 + l)) + ka.group - 1) / ka.group);
    ka.group_shift = (uint32_t)(l - 1);
  }
  if (ka.few_rows >= most) {
    ka.ctas = 0;
    return;
  }
  // A CTA per SM, or fewer where even the longest caches of the table's width make fewer runs.
  const long long by_tokens = (long long)a.tokens * ka.group / kCtaRows + a.batch;
  const long long by_batch = (long long)a.batch * ((most + kCtaRows - 1) / kCtaRows);
  const long long row_tiles = (by_tokens < by_batch ? by_tokens : by_batch) * a.num_kv_heads;
  const long long cap = (long long)a.pages_per_seq * a.page_len;
  const long long seen = a.window > 0 ? (long long)a.window + a.sinks + a.max_q_len + 2 * kTileKeys : cap;
  const long long runs = row_tiles * ((seen < cap ? seen : cap) / kTileKeys + 3) / kMinRun + 1;
  ka.ctas = (int)(runs < kNumSMs ? runs : kNumSMs);
}

// Scratch: the runs' records (both kernels'), then the parts of the one, then those of the other.
static size_t part_floats(const ChunkArgs& ka) { return (size_t)2 * ka.ctas * kCtaRows * (ka.a.head_dim + 2); }
static size_t run_bytes(const ChunkArgs& ka) { return (size_t)ka.ctas * sizeof(int4) + 32; }  // up to a multiple of 32
static size_t chunk_scratch_bytes(const ChunkArgs& ka) {
  return run_bytes(ka) + part_floats(ka) * sizeof(float) + (ka.few_rows ? chunk_few_scratch_bytes(ka) : 0);
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

// The rows of a layer as the copies see them: (64 dims | row of a group of 8 | half of the head's dims | group of 8 rows in
// the page | unit), a unit being one row of one head: pages, their K and V rows and heads all are whole numbers of units
// apart, so the outermost coordinate addresses (page, K or V, head) at once and a box = a page's rows (or box_rows of them)
// of one head, landing group by group, half by half.
void subspec::chunk_tensor_map(ChunkArgs& ka, int rows, CUtensorMap* map) {
  const subspec_chunk_attn_args& a = ka.a;
  memset(map, 0, sizeof(*map));
  int box_rows = rows;
  while (box_rows > 1 && a.page_len % box_rows) box_rows /= 2;  // the largest power of two up to a tile that divides a page
  ka.box_rows = box_rows >= 8 && tensor_map_encoder() ? box_rows : 0;
  if (!ka.box_rows) return;
  const cuuint64_t halves = a.head_dim / 64;
  const cuuint64_t dims[5] = {64, 8, halves, (cuuint64_t)a.page_len / 8, (cuuint64_t)ka.units};
  const cuuint64_t strides[4] = {(cuuint64_t)ka.row_stride, 128, (cuuint64_t)ka.row_stride * 8, (cuuint64_t)a.head_dim * 2};
  const cuuint32_t box[5] = {64, 8, (cuuint32_t)halves, (cuuint32_t)box_rows / 8, 1}, estr[5] = {1, 1, 1, 1, 1};
  if (tensor_map_encoder()(map, a.dtype == SUBSPEC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                           const_cast<unsigned char*>(ka.k_base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    ka.box_rows = 0;
}

template <bool kHalf, int kDim>
static int launch_chunk(ChunkArgs& ka, cudaStream_t stream) {
  const int rc = allow_smem<chunk_attn_tc_kernel<kHalf, kDim>>(tc_smem<kDim>());
  if (rc) return rc;
  CUtensorMap tmap;
  chunk_tensor_map(ka, kTileKeys, &tmap);
  int launched;
  if (ka.few_rows) {
    launched = launch_dependent(chunk_attn_tc_kernel<kHalf, kDim>, dim3((unsigned)ka.ctas), dim3(kChunkThreads), tc_smem<kDim>(),
                                stream, ka, tmap);
  } else {
    chunk_attn_tc_kernel<kHalf, kDim><<<ka.ctas, kChunkThreads, tc_smem<kDim>(), stream>>>(ka, tmap);
    launched = cuda_check(cudaGetLastError());
  }
  if (launched) return launched;
  return launch_dependent(chunk_merge_kernel<kHalf, kDim>, dim3((unsigned)ka.ctas, kCtaRows / 4), dim3(128), 0, stream, ka);
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
  // beyond the capacity of a request's pages they say nothing more (and sums with them stay within 32 bits)
  const int cap = a.pages_per_seq * a.page_len;
  if (ka.a.window > cap) ka.a.window = cap;
  if (ka.a.sinks > cap) ka.a.sinks = cap;
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
  const long long units = (long long)(a.num_pages - 1) * ka.page_units + ka.page_units / 2 + a.num_kv_heads;
  if (units > 0x7fffffffLL) return SUBSPEC_EUNSUPPORTED;
  ka.units = (int)units;
  const size_t need = chunk_scratch_bytes(ka);
  if (need && (!a.scratch || (reinterpret_cast<uintptr_t>(a.scratch) & 15u) || a.scratch_bytes < need)) return SUBSPEC_ESCRATCH;
  ka.runs = reinterpret_cast<int4*>(a.scratch);
  ka.part_o = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(ka.runs + ka.ctas) + 31) & ~(uintptr_t)31);
  ka.part_ml = ka.part_o + (size_t)2 * ka.ctas * kCtaRows * a.head_dim;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (ka.few_rows) {
    rc = launch_chunk_few(ka, ka.part_o + part_floats(ka), st);
    if (rc || ka.ctas == 0) return rc;
  }
  if (a.dtype == SUBSPEC_F16) return a.head_dim == 128 ? launch_chunk<true, 128>(ka, st) : launch_chunk<true, 64>(ka, st);
  return a.head_dim == 128 ? launch_chunk<false, 128>(ka, st) : launch_chunk<false, 64>(ka, st);
}
