// Block tables and slot maps of a step from request lengths, and the append of packed K / V rows by slot.
//
// The reference keeps the page lists on the host (KvCachePool.allocate, RequestKvCache.increment,
// getKvCacheBatchPosition, specdecodes/models/utils/flashinfer/cache_manager.py:66-80, 237-414).  pages_update_kernel
// (pages.cu) is its device form for trees, one thread per request; a step that takes in prompts has hundreds of pages
// and thousands of tokens per request, so here pages and tokens are spread over threads:
//
//   base_b = set_len_b or kv_len_b        rows kept            len_b  = base_b + n_b
//   keep_b = min(n_pages_b, ceil(base_b / L)) pages kept       need_b = ceil(len_b / L)
//   F_b = sum_{c < b} (need_c - keep_c):  request b gets the free pages of rank F_b .. F_b + need_b - keep_b - 1
//   token t of b:  position base_b + t - indptr_b,  slot = table[b, position / L] * L + position % L
//
// Instead of looking for the r-th free page, every free page finds out its own rank (free pages in the words before
// it + bits below it) and, by a binary search over F, which request and list entry it goes to.
#include <cooperative_groups.h>

#include "common.cuh"

namespace subspec {
namespace {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024;
static_assert(kPlanThreads == 32 * 32, "the block scan takes a partial sum from each of 32 warps");
constexpr int kPlanMaxCtas = 8;  // one cluster of the portable size: its barrier orders the phases

// Exclusive scan of two ints per thread over the CTA (carried in one 64-bit word: both sums stay below 2^31).
__device__ __forceinline__ uint64_t block_scan2(uint64_t v, uint64_t* s_warp, uint64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  __syncthreads();  // s_warp may still be read from a previous scan
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const uint64_t w = s_warp[lane];
    uint64_t wi = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint64_t o = __shfl_up_sync(0xffffffffu, wi, d);
      if (lane >= d) wi += o;
    }
    s_warp[lane] = wi - w;
    if (lane == 31) *total = wi;
  }
  __syncthreads();
  return s_warp[warp] + incl - v;
}

// Largest i in [0, n) with a[i] <= x, for ascending a with a[0] <= x.
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Token t's entries: request b (-1: behind the last token), its row, and the pages the request got.
__device__ __forceinline__ void write_token(const subspec_chunk_plan_args& a, int t, int b, int pos, int pages) {
  long long slot = -1;
  const int pi = pos / a.page_len;
  if (b >= 0 && pi < pages) {
    const int pg = __ldcg(a.page_table + (size_t)b * a.pages_per_seq + pi);
    if (pg >= 0 && pg < a.num_pages)
      slot = (long long)pg * a.page_len + (pos - pi * a.page_len);
    else
      flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
  }
  a.slot_map[t] = slot;
  a.positions[t] = pos;
  a.batch_indices[t] = b;
}

__global__ void __launch_bounds__(kPlanThreads) chunk_plan_kernel(const subspec_chunk_plan_args a, int tokens_here) {
  extern __shared__ int sm[];
  __shared__ uint64_t s_warp[32];
  __shared__ uint64_t s_total;
  cg::cluster_group cluster = cg::this_cluster();
  grid_dep_launch();
  const int B = a.batch, P = a.pages_per_seq, L = a.page_len;
  const int words = (a.num_pages + 31) / 32;
  const int cta = (int)blockIdx.x, ctas = (int)gridDim.x;
  int* first = sm;             // [B + 1] rank of a request's first new page, the sum behind the last
  int* indptr = first + B + 1;  // [B + 1]
  int* base = indptr + B + 1;   // [B]
  int* keep = base + B;         // [B]
  int* word_rank = keep + B;    // [words] free pages in the words before this one

  // ---- lengths (every CTA for itself; the state is written back behind the second barrier) ----
  uint64_t carry = 0;
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + (int)threadIdx.x;
    uint64_t v = 0;
    if (b < B) {
      int rows = a.set_len ? a.set_len[b] : a.kv_len[b], n = a.n_new[b], have = a.n_pages[b];
      if (rows < 0 || n < 0 || have < 0 || have > P) {
        if (cta == 0) flag(a.dev_status, SUBSPEC_DEV_BAD_COUNT);
        rows = max(rows, 0), n = max(n, 0), have = min(max(have, 0), P);
      }
      if (rows > P * L || n > P * L) {
        if (cta == 0) flag(a.dev_status, SUBSPEC_DEV_BAD_COUNT);
        rows = min(rows, P * L), n = min(n, P * L);
      }
      const long long len = (long long)rows + n;
      long long need = (len + L - 1) / L;
      if (need > P) {  // the request's page list has no room for that many pages
        if (cta == 0) flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
        need = P;
      }
      const int kept = (int)min((long long)have, ((long long)rows + L - 1) / L);
      base[b] = rows;
      keep[b] = kept;
      v = (uint64_t)(need - kept) << 32 | (uint32_t)n;
    }
    const uint64_t ex = carry + block_scan2(v, s_warp, &s_total);
    if (b < B) first[b] = (int)(ex >> 32), indptr[b] = (int)(uint32_t)ex;
    carry += s_total;
  }
  if (threadIdx.x == 0) first[B] = (int)(carry >> 32), indptr[B] = (int)(uint32_t)carry;
  __syncthreads();
  const int wanted = first[B], tokens = indptr[B];

  // ---- pages behind the kept rows go back: a warp per request ----
  for (int b = cta * (kPlanThreads / 32) + (int)(threadIdx.x >> 5); b < B; b += ctas * (kPlanThreads / 32)) {
    const int have = min(max(a.n_pages[b], 0), P);
    for (int j = keep[b] + (int)(threadIdx.x & 31); j < have; j += 32) {
      int* entry = a.page_table + (size_t)b * P + j;
      const int pg = *entry;
      if (pg >= 0 && pg < a.num_pages)
        atomicOr(a.free_mask + (pg >> 5), 1u << (pg & 31));
      else if (pg != -1)  // (-1: given back before, behind a sliding window)
        flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);
      *entry = -1;
    }
  }
  __threadfence();
  cluster.sync();

  // ---- every free page finds its rank and its place ----
  int wcarry = 0;
  for (int w0 = 0; w0 < words; w0 += kPlanThreads) {
    const int w = w0 + (int)threadIdx.x;
    uint32_t bits = w < words ? __ldcg(a.free_mask + w) : 0u;
    if (w == words - 1 && (a.num_pages & 31)) bits &= (1u << (a.num_pages & 31)) - 1u;  // no pages past the pool
    const int ex = (int)block_scan2((uint64_t)__popc(bits), s_warp, &s_total);
    if (w < words) word_rank[w] = wcarry + ex;
    wcarry += (int)s_total;
    if (wcarry >= wanted) {  // (the same for every thread) the words from here on hand out nothing
      for (int r = w0 + kPlanThreads + (int)threadIdx.x; r < words; r += kPlanThreads) word_rank[r] = wcarry;
      break;
    }
  }
  __syncthreads();
  const int given = min(wanted, wcarry);
  if (wanted > wcarry && cta == 0 && threadIdx.x == 0) flag(a.dev_status, SUBSPEC_DEV_BAD_PAGE);  // out of cache pages
  for (int p = cta * kPlanThreads + (int)threadIdx.x; p < a.num_pages; p += ctas * kPlanThreads) {
    const int w = p >> 5;
    if (word_rank[w] >= given) break;  // ranks ascend: nothing behind this word is handed out
    const uint32_t bits = __ldcg(a.free_mask + w);
    if (!((bits >> (p & 31)) & 1u)) continue;
    const int rank = word_rank[w] + __popc(bits & ((1u << (p & 31)) - 1u));
    if (rank >= given) break;
    const int b = last_not_above(first, B, rank);
    a.page_table[(size_t)b * P + keep[b] + rank - first[b]] = p;
  }
  __threadfence();
  cluster.sync();

  // ---- the state, then the tokens ----
  if (cta == 0) {
    for (int b = (int)threadIdx.x; b < B; b += kPlanThreads) {
      const int n = indptr[b + 1] - indptr[b];
      const int got = min(max(given - first[b], 0), first[b + 1] - first[b]);
      const int len = (int)min((long long)base[b] + n, (long long)P * L);
      a.n_pages[b] = keep[b] + got;
      a.kv_len[b] = len;
      if (a.kv_last_page_len) a.kv_last_page_len[b] = len == 0 ? 0 : (len - 1) % L + 1;
    }
    for (int b = (int)threadIdx.x; b <= B; b += kPlanThreads) a.q_indptr[b] = indptr[b];
    if (threadIdx.x == 0 && tokens > a.max_tokens) flag(a.dev_status, SUBSPEC_DEV_BAD_COUNT);
  }
  for (int w = cta * kPlanThreads + (int)threadIdx.x; w < words; w += ctas * kPlanThreads) {
    int take = given - word_rank[w];
    if (take <= 0) break;
    uint32_t bits = __ldcg(a.free_mask + w), valid = bits;
    if (w == words - 1 && (a.num_pages & 31)) valid &= (1u << (a.num_pages & 31)) - 1u;
    if (take >= __popc(valid)) {
      bits &= ~valid;
    } else {
      while (take-- > 0) {
        const uint32_t low = valid & (0u - valid);
        valid ^= low;
        bits ^= low;
      }
    }
    a.free_mask[w] = bits;
  }
  if (!tokens_here) {  // the second kernel reads a request's kept rows from its first token's position
    for (int b = cta * kPlanThreads + (int)threadIdx.x; b < B; b += ctas * kPlanThreads)
      if (indptr[b] < indptr[b + 1] && indptr[b] < a.max_tokens) a.positions[indptr[b]] = base[b];
    return;
  }
  for (int t = cta * kPlanThreads + (int)threadIdx.x; t < a.max_tokens; t += ctas * kPlanThreads) {
    const int b = t < tokens ? last_not_above(indptr, B, t) : -1;
    write_token(a, t, b, b < 0 ? 0 : base[b] + t - indptr[b],
                b < 0 ? 0 : keep[b] + min(max(given - first[b], 0), first[b + 1] - first[b]));
  }
}

// The tokens of a large step, on all SMs.
constexpr int kTokenThreads = 512;
__global__ void __launch_bounds__(kTokenThreads) chunk_plan_tokens_kernel(const subspec_chunk_plan_args a) {
  extern __shared__ int sm[];
  const int B = a.batch;
  int* indptr = sm;            // [B + 1]
  int* base = indptr + B + 1;  // [B]
  int* pages = base + B;       // [B]
  grid_dep_wait();
  for (int b = (int)threadIdx.x; b <= B; b += kTokenThreads) {
    const int at = a.q_indptr[b];
    indptr[b] = at;
    if (b < B) {
      base[b] = at < a.max_tokens ? __ldcg(a.positions + at) : 0;  // (a request without tokens reads another's: not used)
      pages[b] = a.n_pages[b];
    }
  }
  __syncthreads();
  const int tokens = indptr[B];
  for (int t = (int)(blockIdx.x * kTokenThreads + threadIdx.x); t < a.max_tokens; t += (int)(gridDim.x * kTokenThreads)) {
    const int b = t < tokens ? last_not_above(indptr, B, t) : -1;
    write_token(a, t, b, b < 0 ? 0 : base[b] + t - indptr[b], b < 0 ? 0 : pages[b]);
  }
}

// One 16-byte chunk of a K and of a V row per thread and round.
__global__ void __launch_bounds__(256) kv_append_slots_kernel(const subspec_kv_append_slots_args a) {
  const int per_head = a.head_dim / 8, per_row = a.num_kv_heads * per_head;
  const long long total = (long long)a.tokens * per_row;
  const size_t plane = (size_t)a.page_len * per_row;  // 16-byte chunks of the K (V) rows of a page
  uint4* pool = reinterpret_cast<uint4*>(a.pool) + (size_t)a.layer * a.num_pages * 2 * plane;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(i / per_row), c = (int)(i - (long long)t * per_row);
    const long long slot = a.slot_map[t];
    if (slot < 0) continue;
    if (slot >= (long long)a.num_pages * a.page_len) {
      flag(a.dev_status, SUBSPEC_DEV_BAD_INDEX);
      continue;
    }
    const int h = c / per_head, x = c - h * per_head;
    const uint4 kk = reinterpret_cast<const uint4*>(a.k)[(t * a.k_token_stride + h * a.k_head_stride) / 8 + x];
    const uint4 vv = reinterpret_cast<const uint4*>(a.v)[(t * a.v_token_stride + h * a.v_head_stride) / 8 + x];
    const long long page = slot / a.page_len;
    uint4* dst = pool + (size_t)page * 2 * plane + (size_t)(slot - page * a.page_len) * per_row + c;
    dst[0] = kk;
    dst[plane] = vv;
  }
}

}  // namespace
}  // namespace subspec

using namespace subspec;

extern "C" int subspec_chunk_plan(const subspec_chunk_plan_args* args, subspec_stream_t stream) {
  if (!args || args->struct_size != sizeof(subspec_chunk_plan_args)) return SUBSPEC_EINVAL;
  const subspec_chunk_plan_args& a = *args;
  if (a.batch < 0 || a.num_pages < 1 || a.page_len < 1 || a.pages_per_seq < 1 || a.max_tokens < 0) return SUBSPEC_EINVAL;
  if (a.batch == 0) return SUBSPEC_OK;
  if (!a.free_mask || !a.page_table || !a.n_pages || !a.kv_len || !a.n_new || !a.q_indptr) return SUBSPEC_EINVAL;
  if (a.max_tokens > 0 && (!a.slot_map || !a.positions || !a.batch_indices)) return SUBSPEC_EINVAL;
  // positions, token counts and ranks are 32-bit
  const long long room = (long long)a.pages_per_seq * a.page_len;
  if (room > (1LL << 30) || room * (a.batch > 0 ? a.batch : 1) > 0x7fffffffLL ||
      (long long)a.pages_per_seq * a.batch > 0x7fffffffLL)
    return SUBSPEC_EUNSUPPORTED;
  const size_t words = ((size_t)a.num_pages + 31) / 32;
  const size_t smem = sizeof(int) * (4 * (size_t)a.batch + 2 + words);
  if (smem > 200 * 1024) return SUBSPEC_EUNSUPPORTED;
  int rc = allow_smem<chunk_plan_kernel>(200 * 1024);
  if (!rc) rc = allow_smem<chunk_plan_tokens_kernel>(200 * 1024);
  if (rc) return rc;
  // Up to 8192 tokens the planning CTAs write them too; more go to a kernel of their own on all SMs.
  const int tokens_here = a.max_tokens <= kPlanMaxCtas * kPlanThreads;
  // a CTA for every 1024 tokens, page lists of 32 requests or 32768 pages, at most one cluster of eight
  long long ctas = tokens_here ? (a.max_tokens + kPlanThreads - 1) / kPlanThreads : 1;
  if ((a.batch + 31) / 32 > ctas) ctas = (a.batch + 31) / 32;
  if (words / 1024 > (size_t)ctas) ctas = words / 1024;
  int n = 1;
  while (n < kPlanMaxCtas && n < ctas) n *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)n;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  rc = cuda_check(cudaLaunchKernelEx(&cfg, chunk_plan_kernel, a, tokens_here));
  if (rc || tokens_here) return rc;
  const long long blocks = ((long long)a.max_tokens + kTokenThreads - 1) / kTokenThreads;
  return launch_dependent(chunk_plan_tokens_kernel, dim3((unsigned)(blocks < 2 * kNumSMs ? blocks : 2 * kNumSMs)), dim3(kTokenThreads),
                          sizeof(int) * (3 * (size_t)a.batch + 1), cfg.stream, a);
}

extern "C" int subspec_kv_append_slots(const subspec_kv_append_slots_args* args, subspec_stream_t stream) {
  if (!args || args->struct_size != sizeof(subspec_kv_append_slots_args)) return SUBSPEC_EINVAL;
  const subspec_kv_append_slots_args& a = *args;
  if (a.tokens < 0 || a.num_kv_heads < 1 || a.head_dim < 1 || a.layers < 1 || a.layer < 0 || a.layer >= a.layers ||
      a.num_pages < 1 || a.page_len < 1)
    return SUBSPEC_EINVAL;
  if (a.head_dim % 8 || a.k_token_stride % 8 || a.k_head_stride % 8 || a.v_token_stride % 8 || a.v_head_stride % 8 ||
      (reinterpret_cast<uintptr_t>(a.pool) & 15u) || (reinterpret_cast<uintptr_t>(a.k) & 15u) ||
      (reinterpret_cast<uintptr_t>(a.v) & 15u))
    return SUBSPEC_EUNSUPPORTED;
  if (a.tokens == 0) return SUBSPEC_OK;
  if (!a.pool || !a.k || !a.v || !a.slot_map) return SUBSPEC_EINVAL;
  const long long chunks = (long long)a.tokens * a.num_kv_heads * (a.head_dim / 8);
  const long long blocks = (chunks + 255) / 256;
  kv_append_slots_kernel<<<(unsigned)(blocks < 16 * kNumSMs ? blocks : 16 * kNumSMs), 256, 0,
                           reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cuda_check(cudaGetLastError());
}
