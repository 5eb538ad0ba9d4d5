// Append to a cache of 8-bit pages: keys and values are quantised with one scale for each page and KV head.
//
// A run is the tokens of a call that go to consecutive slots of one page.  Its largest magnitude a gives the least power
// of two s with a <= (largest code) s; the page's scale becomes s where the run begins the page, else the larger of s and
// what it was; codes that the page holds in front of the run move to a raised scale.  Powers of two, because then
// x / s is exact, moving an e4m3 code is exact but among its subnormals, and moving an int8 code is a rounded shift.
// A run with an infinity or a NaN gives its page and head the scale NaN and zeros as codes: whatever reads the page sees it, and
// nothing else does.
//
// One warp does a run of one head's keys or values: no two warps touch the same page and head, so there are no atomics and
// the result does not depend on an order.  Bound by the bytes of large calls and by latency in small ones: 2 x 4096 tokens of 8 heads of
// 128, bf16 to int8, 18.5 us (2.7 TB/s; half of it waits for slots, rows and the earlier scale, one after the other); 32 single tokens 6.7.
#include "paged8.cuh"

namespace qkv {
namespace {

constexpr int kWarps = 4;
__device__ unsigned long long g_tokens_dropped = 0;        // (token, head) pairs without a place in the pool

struct Append8Args {
  const void* x[2];                 // keys, values
  int64_t stride[2][3];             // elements from one sequence, token, head to the next
  int64_t tokens, total;            // per sequence, in all
  qkv_pages8_t p;
  const int64_t* slots;             // [total], or nullptr: positions start_lens[i] .. of row i of the block table
  const int32_t* table; int64_t table_stride; int max_blocks;
  const int32_t* start_lens;
  int window;                       // tokens whose runs one warp does: 1, 2, 4, 8 or 16
};

__device__ __forceinline__ int64_t slot_at(const Append8Args& a, int64_t t) {
  if (a.slots) return a.slots[t];
  const int64_t i = t / a.tokens;
  return p8::slot_of(a.table + i * a.table_stride, a.max_blocks, a.p.block_size, static_cast<int64_t>(a.start_lens[i]) + t % a.tokens);
}

// Eight coordinates of a row as they come, and how their magnitudes compare: as the bits of the largest (without signs an
// infinity is above every number and a NaN above that).
template <typename T> struct Raw;
template <> struct Raw<float> {
  uint4 w[2];
  __device__ __forceinline__ void load(const float* p) { w[0] = __ldg(reinterpret_cast<const uint4*>(p)); w[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1); }
  __device__ __forceinline__ void clear() { w[0] = w[1] = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t x[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, x[i] & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const uint32_t x[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(x[i]);
  }
  static __device__ __forceinline__ float magnitude(uint32_t bits) { return __uint_as_float(bits); }
};
template <typename T> struct Raw16 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t top() const {      // in the upper half of the word
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(x[i] & 0x7fff0000u, (x[i] << 16) & 0x7fff0000u));
    return m;
  }
};
template <> struct Raw<__nv_bfloat16> : Raw16<__nv_bfloat16> {
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(x[i] << 16);
      v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float magnitude(uint32_t bits) { return __uint_as_float(bits); }
};
template <> struct Raw<__half> : Raw16<__half> {
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float magnitude(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits >> 16))); }
};

// A head's keys (which = 0) or values: lanes of a row, rows of a step, steps of sixteen rows.
template <typename T, int CODE, int D> struct Head {
  static constexpr int kLanes = D / 8, kRows = 32 / kLanes, kSteps = (16 + kRows - 1) / kRows;
  const Append8Args& a;
  int which, h, row, col;
  const T* x;
  __device__ __forceinline__ Head(const Append8Args& args, int w, int head) : a(args), which(w), h(head) {
    const int lane = threadIdx.x & 31;
    row = lane / kLanes;                               // D = 96: eight lanes have no row
    col = 8 * (lane % kLanes);
    x = static_cast<const T*>(a.x[which]) + h * a.stride[which][2] + col;
  }
  __device__ __forceinline__ bool has(int s, int n) const { return row < kRows && s * kRows + row < (n < 16 ? n : 16); }
  __device__ __forceinline__ void load(Raw<T> (&v)[kSteps], int64_t t0, int n) const {      // rows t0 .. t0 + min(n, 16)
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      v[s].clear();
      if (!has(s, n)) continue;
      const int64_t t = t0 + s * kRows + row;
      v[s].load(x + (a.slots ? t * a.stride[which][1] : t / a.tokens * a.stride[which][0] + t % a.tokens * a.stride[which][1]));
    }
  }
  // One run: tokens t0 .. t0 + n of the call to rows at .. at + n of page `page`; v holds its first sixteen rows.
  __device__ __forceinline__ void store(Raw<T> (&v)[kSteps], int64_t t0, int n, int64_t page, int at) const {
    const int64_t* ps = which ? a.p.v_stride : a.p.k_stride;
    const int64_t* ss = which ? a.p.vs_stride : a.p.ks_stride;
    uint8_t* codes = (which ? a.p.v_codes : a.p.k_codes) + page * ps[0] + h * ps[1] + col;
    float* scale_p = (which ? a.p.v_scales : a.p.k_scales) + page * ss[0] + h * ss[1];
    const float old = at > 0 ? *scale_p : 0.f;
    uint32_t top = 0;
    for (int k0 = 0;;) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) top = max(top, v[s].top());
      if ((k0 += 16) >= n) break;
      load(v, t0 + k0, n - k0);
    }
    top = __reduce_max_sync(QKV_FULL_MASK, top);
    float scale = p8::scale_for<CODE>(Raw<T>::magnitude(top));
    if (at > 0) scale = (old != old || scale != scale) ? __int_as_float(0x7fc00000) : fmaxf(old, scale);
    // 0 for NaN: codes are zeros.  (A page whose own scale is below 2^-128 can only go on with zeros: these times a finite number.)
    const float inv = scale > 0.f ? fminf(1.f / scale, 0x1.fffffep127f) : 0.f;
    if (scale > 0.f && old != scale && at > 0) {                               // raised: what the page holds moves along
      const float ratio = old / scale;
      for (int k = row; k < at && row < kRows; k += kRows) {
        uint2* c = reinterpret_cast<uint2*>(codes + k * ps[2]);
        const uint2 w = *c;
        const float4 p = p8::decode4<CODE>(w.x), q = p8::decode4<CODE>(w.y);
        *c = make_uint2(p8::encode4<CODE>(p.x * ratio, p.y * ratio, p.z * ratio, p.w * ratio),
                        p8::encode4<CODE>(q.x * ratio, q.y * ratio, q.z * ratio, q.w * ratio));
      }
    }
    for (int k0 = 0; k0 < n; k0 += 16) {
      if (n > 16) load(v, t0 + k0, n - k0);                                    // a short run is still in registers
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (!has(s, n - k0)) continue;
        uint2 w = make_uint2(0, 0);
        if (inv > 0.f) {
          float f[8];
          v[s].values(f);
          w.x = p8::encode4<CODE>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
          w.y = p8::encode4<CODE>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
        }
        *reinterpret_cast<uint2*>(codes + (at + k0 + s * kRows + row) * ps[2]) = w;
      }
    }
    if ((threadIdx.x & 31) == 0) *scale_p = scale;
  }
};

template <typename T, int CODE, int D>
__global__ void __launch_bounds__(kWarps * 32) append8_kernel(Append8Args a) {
  const int lane = threadIdx.x & 31, bs = a.p.block_size;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t win = job / (2 * a.p.Hkv);
  const int hw = static_cast<int>(job - win * (2 * a.p.Hkv));
  const int64_t base = win * a.window;
  if (base >= a.total) return;
  const Head<T, CODE, D> head(a, hw & 1, hw >> 1);
  // The rows of the window travel while the slots do: nearly always they are one run, or its beginning.
  Raw<T> v[Head<T, CODE, D>::kSteps];
  const int64_t room = a.total - base;
  const int ahead = static_cast<int>(room < a.window ? room : a.window);
  head.load(v, base, ahead);
  // lane k holds the slot of token base - 1 + k; tokens 1 .. window of them begin runs where nothing continues
  const int64_t t = base - 1 + lane;
  const int64_t last_slot = a.p.num_blocks * bs;
  const int64_t slot = t >= 0 && t < a.total ? slot_at(a, t) : -1;
  const int64_t prev = __shfl_up_sync(QKV_FULL_MASK, slot, 1);
  const bool here = lane >= 1 && lane <= a.window && t < a.total;
  const bool lost = here && (slot >= last_slot || (slot < 0 && !a.slots));
  if (head.which == 0) {
    const unsigned dropped = __popc(__ballot_sync(QKV_FULL_MASK, lost));
    if (dropped && lane == 0) atomicAdd(&g_tokens_dropped, static_cast<unsigned long long>(dropped));
  }
  const bool goes_on = lane >= 1 && prev >= 0 && prev + 1 == slot && slot % bs != 0;
  const unsigned on = __ballot_sync(QKV_FULL_MASK, goes_on);
  unsigned todo = __ballot_sync(QKV_FULL_MASK, here && slot >= 0 && slot < last_slot && !goes_on);
  bool first = true;                                       // v still holds the window's rows
  while (todo) {
    const int k = __ffs(todo) - 1;
    todo &= todo - 1;
    const int64_t t0 = base - 1 + k, s0 = __shfl_sync(QKV_FULL_MASK, slot, k);
    const int at = static_cast<int>(s0 % bs);
    const unsigned more = k < 31 ? ~(on >> (k + 1)) : ~0u;
    int n = __ffs(more);                                   // tokens of the run among the lanes: itself and those that go on
    if (k + n == 32) {                                     // it may go on behind them, 32 tokens at a time
      for (;;) {
        const int64_t u = t0 + n + lane;
        const bool yes = u < a.total && at + n + lane < bs && slot_at(a, u) == s0 + n + lane;
        const unsigned m = __ballot_sync(QKV_FULL_MASK, yes);
        if (m == QKV_FULL_MASK) { n += 32; continue; }
        n += __ffs(~m) - 1;
        break;
      }
    }
    if (!first || k != 1 || (n > ahead && ahead < 16) || n < ahead) head.load(v, t0, n);
    first = false;
    head.store(v, t0, n, s0 / bs, at);
  }
}

template <typename T, int CODE>
void launch_d(const Append8Args& a, unsigned grid, cudaStream_t st) {
  switch (a.p.d) {
    case 32: append8_kernel<T, CODE, 32><<<grid, kWarps * 32, 0, st>>>(a); break;
    case 64: append8_kernel<T, CODE, 64><<<grid, kWarps * 32, 0, st>>>(a); break;
    case 96: append8_kernel<T, CODE, 96><<<grid, kWarps * 32, 0, st>>>(a); break;
    default: append8_kernel<T, CODE, 128><<<grid, kWarps * 32, 0, st>>>(a); break;
  }
}
template <typename T>
void launch_code(const Append8Args& a, unsigned grid, cudaStream_t st) {
  if (a.p.code == QKV_E4M3) launch_d<T, p8::kE4M3>(a, grid, st);
  else launch_d<T, p8::kInt8>(a, grid, st);
}

}  // namespace
}  // namespace qkv

using namespace qkv;

extern "C" int qkv_append_paged8(const void* keys, const void* values, int dtype, const int64_t* key_strides,
                                 const int64_t* value_strides, int64_t n_seq, int64_t tokens, qkv_pages8_t pages,
                                 const int64_t* slots, const int32_t* block_table, int64_t table_stride, int max_blocks,
                                 const int32_t* start_lens, void* stream) {
  if (!keys || !values || !key_strides || !value_strides || (!slots && (!block_table || !start_lens))) return QKV_ENULL;
  if (dtype != QKV_F32 && dtype != QKV_BF16 && dtype != QKV_F16) return QKV_EDTYPE;
  if (const int rc = check_pages8(pages)) return rc;
  if (n_seq < 0 || tokens < 0 || (!slots && max_blocks < 1)) return QKV_EDIM;
  if (slots && n_seq != 1) return QKV_EARG;
  if (n_seq == 0 || tokens == 0) return QKV_OK;
  if (tokens > (int64_t(1) << 40) / n_seq) return QKV_EDIM;
  const int item = dtype == QKV_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & 15u) return QKV_EALIGN;
  for (int i = 0; i < 3; ++i)
    if ((key_strides[i] * item & 15) || (value_strides[i] * item & 15)) return QKV_EALIGN;
  Append8Args a{};
  a.x[0] = keys;
  a.x[1] = values;
  for (int i = 0; i < 3; ++i) {
    a.stride[0][i] = key_strides[i];
    a.stride[1][i] = value_strides[i];
  }
  a.tokens = tokens;
  a.total = n_seq * tokens;
  a.p = pages;
  a.slots = slots;
  a.table = block_table;
  a.table_stride = table_stride;
  a.max_blocks = max_blocks;
  a.start_lens = start_lens;
  // Tokens of a warp: one while sixteen warps an SM are enough for that, so that runs of single tokens go side by side; more in
  // larger calls, whose tokens mostly continue a run, which their warps would only find out.  us by window, 8 heads of 128, all
  // tokens in a page of their own / all in runs: 64 tokens 1 7.6 / 8.0, 16 29.8 / 7.5; 592 tokens 1 15.8 / 13.1, 4
  // 14.0 / 9.0, 16 29.9 / 7.6; 1024 tokens 1 21.8 / 15.8, 8 21.9 / 10.1, 16 30.1 / 8.4; 2048 tokens 1 36.8 / 23.5, 16 36.1 / 9.7.
  a.window = 1;
  while (a.window < 16 && a.total * 2 * pages.Hkv > a.window * 16LL * kNumSMs) a.window *= 2;
  const int64_t jobs = (a.total + a.window - 1) / a.window * 2 * pages.Hkv, grid = (jobs + kWarps - 1) / kWarps;
  if (grid > 0x7fffffffLL) return QKV_EDIM;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == QKV_F32) launch_code<float>(a, static_cast<unsigned>(grid), st);
  else if (dtype == QKV_BF16) launch_code<__nv_bfloat16>(a, static_cast<unsigned>(grid), st);
  else launch_code<__half>(a, static_cast<unsigned>(grid), st);
  return check_launch();
}

extern "C" int64_t qkv_dropped_paged8_tokens(void) {
  unsigned long long v = 0;
  cudaMemcpyFromSymbol(&v, g_tokens_dropped, sizeof(v));
  return static_cast<int64_t>(v);
}
