// Block tables and slots from request lengths, on the device: pages go from a stack of free ones to the sequences that
// grow (extend), and back (shrink).  No counterpart in the reference, whose page manager stores no pages
// (integrations/vllm_backend.py:82-195).
//
// With L_i tokens held, N_i new ones, tables of W pages of bs tokens and F pages on the stack f:
//   have_i = ceil(L_i / bs), need_i = max(0, min(ceil((L_i + N_i) / bs), W) - have_i), P_i = sum of need_k over k < i
//   table[i][have_i + j] = f[F - 1 - (P_i + j)] for j < got_i = clamp(F - P_i, 0, need_i)
//   slot of new token t = page * bs + offset of position L_i + t while the pages last, else -1
// so two prefix sums over the sequences decide everything, and then every page and every token is on its own.
//
// Each CTA of ONE cluster forms the prefix sums for itself in shared memory (12 bytes a sequence) and takes its share
// of pages and tokens, finding the sequence by binary search.  Lengths and counts are written after a cluster barrier, so they may be written
// where they were read.  One launch; bound by its latency.
#include <cooperative_groups.h>

#include "paged8.cuh"

namespace qkv {
namespace {

constexpr int kMaxSeqs = QKV_PAGES_MAX_SEQS;
constexpr int kMostThreads = 1024;

struct ExtendArgs {
  int32_t* table; int64_t table_stride; int max_blocks;
  const int32_t* lens; const int32_t* new_lens; const int32_t* free_pages; int64_t n_pages;
  const int32_t* pool; int n, block_size; int64_t max_tokens;
  int64_t* slots; int32_t* starts; int32_t* lens_out; int32_t* start_out; int32_t* pool_out;
};

// Exclusive prefix sums of v[0 .. n) in place, the total in v[n]; all threads of the CTA.
__device__ void scan_cta(int32_t* v, int n) {
  __shared__ int32_t part[33];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = (n + blockDim.x - 1) / blockDim.x;
  const int lo = min(n, tid * per), hi = min(n, lo + per);
  int32_t sum = 0;
  for (int i = lo; i < hi; ++i) sum += v[i];
  int32_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t y = __shfl_up_sync(QKV_FULL_MASK, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int warps = blockDim.x >> 5;
    int32_t x = lane < warps ? part[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t y = __shfl_up_sync(QKV_FULL_MASK, x, o);
      if (lane >= o) x += y;
    }
    part[lane + 1] = x;
    if (lane == 0) part[0] = 0;
  }
  __syncthreads();
  int32_t at = part[warp] + inc - sum;
  for (int i = lo; i < hi; ++i) {
    const int32_t x = v[i];
    v[i] = at;
    at += x;
  }
  if (tid == blockDim.x - 1) v[n] = part[blockDim.x >> 5];
  __syncthreads();
}

// The last i of 0 .. n-1 with v[i] <= x (v ascending, v[0] <= x): with v[n] > x that i has v[i + 1] > x.
__device__ __forceinline__ int owner(const int32_t* v, int n, int32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_for(int64_t tokens, int bs, int most) {
  const int64_t p = (tokens + bs - 1) / bs;
  return p > most ? most : static_cast<int>(p);
}

__global__ void __launch_bounds__(kMostThreads) extend_kernel(ExtendArgs a) {
  extern __shared__ int32_t sh[];
  int32_t* len = sh;                       // [n]
  int32_t* start = sh + a.n;               // [n + 1] tokens in front of a sequence, within max_tokens
  int32_t* page = start + a.n + 1;         // [n + 1] pages in front of it
  __shared__ unsigned long long asked_s;
  const int tid = threadIdx.x, T = blockDim.x;
  const unsigned ctas = gridDim.x, rank = blockIdx.x;
  if (tid == 0) asked_s = 0;
  __syncthreads();
  unsigned long long asked = 0;
  for (int i = tid; i < a.n; i += T) {
    const int32_t L = max(a.lens[i], 0), N = max(a.new_lens[i], 0);
    len[i] = L;
    asked += N;
    // no length can be more than the slots of the call (and a longer sum stops there, below)
    start[i] = static_cast<int32_t>(min(static_cast<int64_t>(N), a.max_tokens));
  }
  for (int o = 16; o > 0; o >>= 1) asked += __shfl_xor_sync(QKV_FULL_MASK, asked, o);
  if ((tid & 31) == 0 && asked) atomicAdd(&asked_s, asked);
  const int64_t left = min(static_cast<int64_t>(max(a.pool[0], 0)), a.n_pages);
  const int32_t missed_before = a.pool[1];
  __syncthreads();
  if (asked_s > 0x7fffffffull) {           // the sums would pass 32 bits: one thread adds them up to the limit
    if (tid == 0) {
      int64_t at = 0;
      for (int i = 0; i < a.n; ++i) {
        const int64_t N = min(static_cast<int64_t>(start[i]), a.max_tokens - at);
        start[i] = static_cast<int32_t>(N);
        at += N;
      }
    }
    __syncthreads();
  }
  scan_cta(start, a.n);
  const int32_t most = static_cast<int32_t>(a.max_tokens);
  for (int i = tid; i <= a.n; i += T) start[i] = min(start[i], most);
  __syncthreads();
  for (int i = tid; i < a.n; i += T) {
    const int have = pages_for(len[i], a.block_size, a.max_blocks);
    page[i] = max(0, pages_for(static_cast<int64_t>(len[i]) + (start[i + 1] - start[i]), a.block_size, a.max_blocks) - have);
  }
  __syncthreads();
  scan_cta(page, a.n);
  const int32_t given = static_cast<int32_t>(min(left, static_cast<int64_t>(page[a.n])));
  auto granted = [&](int i) -> int32_t {   // tokens of sequence i that have a page
    const int have = pages_for(len[i], a.block_size, a.max_blocks);
    const int got = max(0, min(page[i + 1], given) - page[i]);
    const int64_t room = static_cast<int64_t>(have + got) * a.block_size - len[i];
    return static_cast<int32_t>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(start[i + 1] - start[i]), room)));
  };
  for (int32_t p = rank * T + tid; p < given; p += ctas * T) {
    const int i = owner(page, a.n, p);
    const int j = pages_for(len[i], a.block_size, a.max_blocks) + p - page[i];
    a.table[i * a.table_stride + j] = a.free_pages[left - 1 - p];
  }
  const int32_t total = start[a.n];
  for (int64_t t = rank * T + tid; t < a.max_tokens; t += ctas * T) {
    int64_t slot = -1;
    if (t < total) {
      const int i = owner(start, a.n, static_cast<int32_t>(t));
      const int32_t inside = static_cast<int32_t>(t) - start[i];
      if (inside < granted(i)) {
        const int64_t pos = static_cast<int64_t>(len[i]) + inside;
        const int have = pages_for(len[i], a.block_size, a.max_blocks), j = static_cast<int>(pos / a.block_size);
        // pages of this call come from the stack: their entries may not be in the table yet
        const int32_t id = j < have ? a.table[i * a.table_stride + j] : a.free_pages[left - 1 - (page[i] + j - have)];
        if (id >= 0) slot = static_cast<int64_t>(id) * a.block_size + pos % a.block_size;
      }
    }
    a.slots[t] = slot;
  }
  if (ctas > 1) cooperative_groups::this_cluster().sync();     // every CTA has read the lengths and the counts
  if (rank != 0) return;
  unsigned long long stored = 0;
  for (int i = tid; i < a.n; i += T) {
    const int32_t g = granted(i);
    stored += g;
    a.lens_out[i] = len[i] + g;
    if (a.start_out) a.start_out[i] = len[i];
  }
  for (int i = tid; i <= a.n; i += T) a.starts[i] = start[i];
  for (int o = 16; o > 0; o >>= 1) stored += __shfl_xor_sync(QKV_FULL_MASK, stored, o);
  if ((tid & 31) == 0 && stored) atomicAdd(&asked_s, 0ull - stored);
  __syncthreads();
  if (tid == 0) {
    const unsigned long long missed = asked_s + static_cast<unsigned long long>(max(missed_before, 0));
    a.pool_out[0] = static_cast<int32_t>(left - given);
    a.pool_out[1] = static_cast<int32_t>(missed > 0x7fffffffull ? 0x7fffffffull : missed);
  }
}

struct ShrinkArgs {
  const int32_t* table; int64_t table_stride; int max_blocks;
  int32_t* lens; const int32_t* keep; int32_t* free_pages; int64_t n_pages; int32_t* pool;
  int n, block_size;
};

// The pages behind the kept tokens go back in the order that makes shrink after extend leave the stack as it was.
__global__ void __launch_bounds__(kMostThreads) shrink_kernel(ShrinkArgs a) {
  extern __shared__ int32_t sh[];
  int32_t* len = sh;                       // [n] kept tokens
  int32_t* page = sh + a.n;                // [n + 1] pages given back in front of a sequence
  const int tid = threadIdx.x, T = blockDim.x;
  const unsigned ctas = gridDim.x, rank = blockIdx.x;
  for (int i = tid; i < a.n; i += T) {
    const int32_t L = max(a.lens[i], 0), K = min(max(a.keep[i], 0), L);
    len[i] = K;
    page[i] = pages_for(L, a.block_size, a.max_blocks) - pages_for(K, a.block_size, a.max_blocks);
  }
  const int64_t left = min(static_cast<int64_t>(max(a.pool[0], 0)), a.n_pages);
  __syncthreads();
  scan_cta(page, a.n);
  const int64_t now = left + page[a.n];
  for (int32_t p = rank * T + tid; p < page[a.n]; p += ctas * T) {
    const int i = owner(page, a.n, p);
    const int j = pages_for(len[i], a.block_size, a.max_blocks) + p - page[i];
    const int64_t at = now - 1 - p;
    if (at < a.n_pages) a.free_pages[at] = a.table[i * a.table_stride + j];
  }
  if (ctas > 1) cooperative_groups::this_cluster().sync();
  if (rank != 0) return;
  for (int i = tid; i < a.n; i += T) a.lens[i] = len[i];
  if (tid == 0) a.pool[0] = static_cast<int32_t>(min(now, a.n_pages));
}

template <typename Args>
int launch_cluster(void (*kernel)(Args), const Args& a, int64_t work, size_t smem, cudaStream_t st) {
  // A few items a thread, in at most eight CTAs (the portable size of a cluster); small calls stay in one CTA of few warps.
  int threads = 128;
  while (threads < kMostThreads && (threads < a.n || threads < work)) threads *= 2;
  int ctas = 1;
  while (ctas < 8 && static_cast<int64_t>(ctas) * threads * 4 < work) ctas *= 2;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return QKV_ELAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? check_launch() : QKV_ELAUNCH;
}

int check_tables(const void* table, int64_t stride, int max_blocks, int n, int block_size) {
  if (!table) return QKV_ENULL;
  if (n < 1 || n > kMaxSeqs || max_blocks < 1 || block_size < 1 || stride < max_blocks) return QKV_EDIM;
  // page counts are 32-bit sums, lengths 32-bit numbers
  if (static_cast<int64_t>(n) * max_blocks > 0x7fffffffLL || static_cast<int64_t>(max_blocks) * block_size > 0x7fffffffLL) return QKV_EDIM;
  return QKV_OK;
}

}  // namespace
}  // namespace qkv

using namespace qkv;

extern "C" int qkv_extend_pages(int32_t* block_table, int64_t table_stride, int max_blocks, const int32_t* seq_lens,
                                const int32_t* new_lens, const int32_t* free_pages, int64_t n_free_pages, const int32_t* pool,
                                int n_seq, int block_size, int64_t max_tokens, int64_t* slots, int32_t* query_starts,
                                int32_t* seq_lens_out, int32_t* start_lens_out, int32_t* pool_out, void* stream) {
  if (const int rc = check_tables(block_table, table_stride, max_blocks, n_seq, block_size)) return rc;
  if (!seq_lens || !new_lens || !free_pages || !pool || !query_starts || !seq_lens_out || !pool_out || (max_tokens > 0 && !slots))
    return QKV_ENULL;
  if (max_tokens < 0 || max_tokens > 0x7fffffffLL || n_free_pages < 0) return QKV_EDIM;
  const ExtendArgs a{block_table, table_stride, max_blocks, seq_lens, new_lens, free_pages, n_free_pages, pool, n_seq, block_size,
                     max_tokens, slots, query_starts, seq_lens_out, start_lens_out, pool_out};
  return launch_cluster(extend_kernel, a, max_tokens, (3 * static_cast<size_t>(n_seq) + 2) * 4, static_cast<cudaStream_t>(stream));
}

extern "C" int qkv_shrink_pages(const int32_t* block_table, int64_t table_stride, int max_blocks, int32_t* seq_lens,
                                const int32_t* keep_lens, int32_t* free_pages, int64_t n_free_pages, int32_t* pool, int n_seq,
                                int block_size, void* stream) {
  if (const int rc = check_tables(block_table, table_stride, max_blocks, n_seq, block_size)) return rc;
  if (!seq_lens || !keep_lens || !free_pages || !pool) return QKV_ENULL;
  if (n_free_pages < 0) return QKV_EDIM;
  const ShrinkArgs a{block_table, table_stride, max_blocks, seq_lens, keep_lens, free_pages, n_free_pages, pool, n_seq, block_size};
  // how many pages come back is known on the device only: a few CTAs where there can be many
  const int64_t most = static_cast<int64_t>(n_seq) * max_blocks;
  return launch_cluster(shrink_kernel, a, most < 8192 ? most : 8192, (2 * static_cast<size_t>(n_seq) + 1) * 4,
                        static_cast<cudaStream_t>(stream));
}
