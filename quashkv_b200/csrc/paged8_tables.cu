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
// Every CTA forms the prefix sums for itself in shared memory (12 bytes a sequence; with a few thousand sequences that is
// less than a launch) and takes its share of pages and tokens, finding the sequence by binary search.  Lengths and counts are written
// by the first CTA where they have places of their own; where they are updated in place, that waits for a second launch of one
// CTA behind the others, which have read them by then.  Bound by the latency of its few dependent loads.
// Measured, 512 sequences and 295,000 new tokens: 10.3 us (67 with eight CTAs of one cluster and 64-bit divisions), most of it the
// slots' searches; 32 single tokens: 10 us with the host's part (a tensor for each result), about 3 of them the kernel's.
#include <cooperative_groups.h>

#include "paged8.cuh"

namespace qkv {
namespace {

constexpr int kMaxSeqs = QKV_PAGES_MAX_SEQS;
constexpr int kMostThreads = 1024;

struct ExtendArgs {
  int32_t* table; int64_t table_stride; int max_blocks;
  const int32_t* lens; const int32_t* new_lens; const int32_t* free_pages; int64_t n_pages;
  const int32_t* pool; int n, block_size, bs_shift; int64_t max_tokens;
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

// Division by the block size: a shift where it is a power of two.
struct BlockSize {
  uint32_t bs; int shift;
  __device__ __forceinline__ uint32_t div(uint32_t x) const { return shift >= 0 ? x >> shift : x / bs; }
  // pages of `tokens`, at most `most` (tokens up to 2^32)
  __device__ __forceinline__ int pages(uint32_t tokens, int most) const {
    const uint32_t p = div(tokens) + (tokens - div(tokens) * bs != 0);
    return p > static_cast<uint32_t>(most) ? most : static_cast<int>(p);
  }
};

// slots: a share of the pages and tokens for each CTA;  state: lengths and counts, by the first CTA.
template <bool SLOTS, bool STATE>
__global__ void __launch_bounds__(kMostThreads) extend_kernel(ExtendArgs a) {
  extern __shared__ int32_t sh[];
  int32_t* len = sh;                       // [n]
  int32_t* start = sh + a.n;               // [n + 1] tokens in front of a sequence, within max_tokens
  int32_t* page = start + a.n + 1;         // [n + 1] pages in front of it
  __shared__ unsigned long long asked_s;
  const int tid = threadIdx.x, T = blockDim.x;
  const BlockSize bs{static_cast<uint32_t>(a.block_size), a.bs_shift};
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
  const int32_t left = static_cast<int32_t>(min(static_cast<int64_t>(max(a.pool[0], 0)), a.n_pages)), missed_before = a.pool[1];
  for (int o = 16; o > 0; o >>= 1) asked += __shfl_xor_sync(QKV_FULL_MASK, asked, o);
  if ((tid & 31) == 0 && asked) atomicAdd(&asked_s, asked);
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
  for (int i = tid; i < a.n; i += T) {
    const uint32_t N = min(start[i + 1], most) - min(start[i], most);
    page[i] = max(0, bs.pages(len[i] + N, a.max_blocks) - bs.pages(len[i], a.max_blocks));
  }
  __syncthreads();
  for (int i = tid; i <= a.n; i += T) start[i] = min(start[i], most);
  scan_cta(page, a.n);
  const int32_t given = min(left, page[a.n]);
  auto granted = [&](int i) -> int32_t {   // tokens of sequence i that have a page
    const int have = bs.pages(len[i], a.max_blocks);
    const int got = max(0, min(page[i + 1], given) - page[i]);
    const int64_t room = static_cast<int64_t>(have + got) * a.block_size - len[i];
    return static_cast<int32_t>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(start[i + 1] - start[i]), room)));
  };
  if (SLOTS) {
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * T + tid; p < given; p += static_cast<int64_t>(gridDim.x) * T) {
      const int i = owner(page, a.n, static_cast<int32_t>(p));
      const int j = bs.pages(len[i], a.max_blocks) + static_cast<int32_t>(p) - page[i];
      a.table[i * a.table_stride + j] = a.free_pages[left - 1 - p];
    }
    const int32_t total = start[a.n];
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * T + tid; t < a.max_tokens; t += static_cast<int64_t>(gridDim.x) * T) {
      int64_t slot = -1;
      if (t < total) {
        const int i = owner(start, a.n, static_cast<int32_t>(t));
        const int32_t inside = static_cast<int32_t>(t) - start[i];
        if (inside < granted(i)) {
          const uint32_t pos = static_cast<uint32_t>(len[i]) + inside;
          const int have = bs.pages(len[i], a.max_blocks), j = static_cast<int>(bs.div(pos));
          // pages of this call come from the stack: their entries may not be in the table yet
          const int32_t id = j < have ? a.table[i * a.table_stride + j] : a.free_pages[left - 1 - (page[i] + j - have)];
          if (id >= 0) slot = static_cast<int64_t>(id) * a.block_size + (pos - static_cast<uint32_t>(j) * bs.bs);
        }
      }
      a.slots[t] = slot;
    }
    // in place: the lengths before, which the launch behind this one reads in their stead
    if (!STATE && blockIdx.x == 0)
      for (int i = tid; i < a.n; i += T) a.start_out[i] = len[i];
  }
  if (!STATE || blockIdx.x != 0) return;
  __syncthreads();                         // asked_s and the lengths have been read
  unsigned long long stored = 0;
  for (int i = tid; i < a.n; i += T) {
    const int32_t g = granted(i);
    stored += g;
    a.lens_out[i] = len[i] + g;
    if (SLOTS && a.start_out) a.start_out[i] = len[i];
  }
  for (int i = tid; i <= a.n; i += T) a.starts[i] = start[i];
  for (int o = 16; o > 0; o >>= 1) stored += __shfl_xor_sync(QKV_FULL_MASK, stored, o);
  if ((tid & 31) == 0 && stored) atomicAdd(&asked_s, 0ull - stored);
  __syncthreads();
  if (tid == 0) {
    const unsigned long long missed = asked_s + static_cast<unsigned long long>(max(missed_before, 0));
    a.pool_out[0] = left - given;
    a.pool_out[1] = static_cast<int32_t>(missed > 0x7fffffffull ? 0x7fffffffull : missed);
  }
}

struct ShrinkArgs {
  const int32_t* table; int64_t table_stride; int max_blocks;
  int32_t* lens; const int32_t* keep; int32_t* free_pages; int64_t n_pages; int32_t* pool;
  int n, block_size, bs_shift;
};

// The pages behind the kept tokens go back in the order that makes shrink after extend leave the stack as it was.  One
// cluster: lengths and counts are written when all of its CTAs have read them.
__global__ void __launch_bounds__(kMostThreads) shrink_kernel(ShrinkArgs a) {
  extern __shared__ int32_t sh[];
  int32_t* len = sh;                       // [n] kept tokens
  int32_t* page = sh + a.n;                // [n + 1] pages given back in front of a sequence
  const int tid = threadIdx.x, T = blockDim.x;
  const BlockSize bs{static_cast<uint32_t>(a.block_size), a.bs_shift};
  for (int i = tid; i < a.n; i += T) {
    const int32_t L = max(a.lens[i], 0), K = min(max(a.keep[i], 0), L);
    len[i] = K;
    page[i] = bs.pages(L, a.max_blocks) - bs.pages(K, a.max_blocks);
  }
  const int64_t left = min(static_cast<int64_t>(max(a.pool[0], 0)), a.n_pages);
  __syncthreads();
  scan_cta(page, a.n);
  const int64_t now = left + page[a.n];
  for (int64_t p = static_cast<int64_t>(blockIdx.x) * T + tid; p < page[a.n]; p += static_cast<int64_t>(gridDim.x) * T) {
    const int i = owner(page, a.n, static_cast<int32_t>(p));
    const int j = bs.pages(len[i], a.max_blocks) + static_cast<int32_t>(p) - page[i];
    const int64_t at = now - 1 - p;
    if (at < a.n_pages) a.free_pages[at] = a.table[i * a.table_stride + j];
  }
  if (gridDim.x > 1) cooperative_groups::this_cluster().sync();
  if (blockIdx.x != 0) return;
  for (int i = tid; i < a.n; i += T) a.lens[i] = len[i];
  if (tid == 0) a.pool[0] = static_cast<int32_t>(min(now, a.n_pages));
}

// Tokens of a CTA: few, so that the searches and loads of a large call run side by side all over the chip, and not too few,
// since every CTA forms the sums.  512 sequences, 295,000 tokens: 512 tokens a CTA 14.5 us, 2048 10.3, 8192 16.6.
constexpr int kTokensPerCta = 2048;

int threads_for(int64_t items) {
  int threads = 128;
  while (threads < kMostThreads && threads < items) threads *= 2;
  return threads;
}

constexpr size_t kMostSmem = (3 * static_cast<size_t>(kMaxSeqs) + 2) * 4;

int shift_of(int bs) { return (bs & (bs - 1)) == 0 ? __builtin_ctz(bs) : -1; }

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
  const bool in_place = seq_lens_out == seq_lens || pool_out == pool;
  if (in_place && !start_lens_out) return QKV_ENULL;
  ExtendArgs a{block_table, table_stride, max_blocks, seq_lens, new_lens, free_pages, n_free_pages, pool, n_seq, block_size, shift_of(block_size),
               max_tokens, slots, query_starts, seq_lens_out, start_lens_out, pool_out};
  const size_t smem = (3 * static_cast<size_t>(n_seq) + 2) * 4;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t ctas = max_tokens > kTokensPerCta ? (max_tokens + kTokensPerCta - 1) / kTokensPerCta : 1;
  const int threads = threads_for(max_tokens > n_seq ? max_tokens : n_seq);
  const unsigned grid = static_cast<unsigned>(ctas < 4 * kNumSMs ? ctas : 4 * kNumSMs);
  if (!in_place || grid == 1) {            // (one CTA has read what it overwrites)
    if (const int rc = allow_smem<extend_kernel<true, true>>(kMostSmem)) return rc;
    extend_kernel<true, true><<<grid, threads, smem, st>>>(a);
    return check_launch();
  }
  if (const int rc = allow_smem<extend_kernel<true, false>>(kMostSmem)) return rc;
  if (const int rc = allow_smem<extend_kernel<false, true>>(kMostSmem)) return rc;
  extend_kernel<true, false><<<grid, threads, smem, st>>>(a);
  if (const int rc = check_launch()) return rc;
  a.lens = start_lens_out;
  extend_kernel<false, true><<<1, threads_for(n_seq), smem, st>>>(a);
  return check_launch();
}

extern "C" int qkv_shrink_pages(const int32_t* block_table, int64_t table_stride, int max_blocks, int32_t* seq_lens,
                                const int32_t* keep_lens, int32_t* free_pages, int64_t n_free_pages, int32_t* pool, int n_seq,
                                int block_size, void* stream) {
  if (const int rc = check_tables(block_table, table_stride, max_blocks, n_seq, block_size)) return rc;
  if (!seq_lens || !keep_lens || !free_pages || !pool) return QKV_ENULL;
  if (n_free_pages < 0) return QKV_EDIM;
  const ShrinkArgs a{block_table, table_stride, max_blocks, seq_lens, keep_lens, free_pages, n_free_pages, pool, n_seq, block_size, shift_of(block_size)};
  // How many pages come back is known on the device only: the portable eight CTAs of a cluster where there can be many.
  const size_t smem = (2 * static_cast<size_t>(n_seq) + 1) * 4;
  if (const int rc = allow_smem<shrink_kernel>(kMostSmem)) return rc;
  const int64_t most = static_cast<int64_t>(n_seq) * max_blocks;
  const int ctas = most > 4096 ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads_for(most));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, shrink_kernel, a) == cudaSuccess ? check_launch() : QKV_ELAUNCH;
}
