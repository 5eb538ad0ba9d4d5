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
// the result does not depend on an order.  Bound by the bytes of large calls and by latency in small ones.
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
  int window;                       // tokens whose runs one warp does: 1 or 16
};

__device__ __forceinline__ int64_t slot_at(const Append8Args& a, int64_t t) {
  if (a.slots) return a.slots[t];
  const int64_t i = t / a.tokens;
  return p8::slot_of(a.table + i * a.table_stride, a.max_blocks, a.p.block_size, static_cast<int64_t>(a.start_lens[i]) + t % a.tokens);
}

// Eight coordinates as fp32.
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(x[i] << 16);
    v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
  }
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float (&v)[8]) {
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// One run: tokens t0 .. t0 + n of the call to rows at .. at + n of page `page`, head h, keys (which = 0) or values.
template <typename T, int CODE, int D>
__device__ __forceinline__ void store_run(const Append8Args& a, int which, int h, int64_t t0, int n, int64_t page, int at) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kSteps = (16 + kRows - 1) / kRows;    // lanes a row, rows a step
  const int lane = threadIdx.x & 31, row = lane / kLanes, col = 8 * (lane % kLanes);
  const bool on = row < kRows;                                                 // D = 96: eight lanes have no row
  const T* x = static_cast<const T*>(a.x[which]) + h * a.stride[which][2] + col;
  const int64_t* ps = which ? a.p.v_stride : a.p.k_stride;
  const int64_t* ss = which ? a.p.vs_stride : a.p.ks_stride;
  uint8_t* codes = (which ? a.p.v_codes : a.p.k_codes) + page * ps[0] + h * ps[1] + col;
  float* scale_p = (which ? a.p.v_scales : a.p.k_scales) + page * ss[0] + h * ss[1];
  auto source = [&](int k) {
    const int64_t t = t0 + k;
    return x + (a.slots ? t * a.stride[which][1] : t / a.tokens * a.stride[which][0] + t % a.tokens * a.stride[which][1]);
  };
  const float old = at > 0 ? *scale_p : 0.f;
  float v[kSteps][8];
  float top = 0.f;
  bool odd = false;                                                            // an infinity or a NaN
  for (int k0 = 0; k0 < n; k0 += 16) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k = k0 + s * kRows + row;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s][e] = 0.f;
      if (on && k < n && s * kRows + row < 16) load8<T>(source(k), v[s]);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float m = fabsf(v[s][e]);
        odd |= !(m < INFINITY);
        top = fmaxf(top, m);
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(QKV_FULL_MASK, top, o));
  if (__any_sync(QKV_FULL_MASK, odd)) top = INFINITY;
  float scale = p8::scale_for<CODE>(top);
  if (at > 0) scale = (old != old || scale != scale) ? __int_as_float(0x7fc00000) : fmaxf(old, scale);
  const float inv = scale > 0.f ? 1.f / scale : 0.f;                           // 0 for NaN: codes are zeros
  if (scale > 0.f && old != scale && at > 0) {                                 // raised: what the page holds moves along
    const float ratio = old / scale;
    for (int k = row; k < at && on; k += kRows) {
      uint2* c = reinterpret_cast<uint2*>(codes + k * ps[2]);
      const uint2 w = *c;
      const float4 p = p8::decode4<CODE>(w.x), q = p8::decode4<CODE>(w.y);
      *c = make_uint2(p8::encode4<CODE>(p.x * ratio, p.y * ratio, p.z * ratio, p.w * ratio),
                      p8::encode4<CODE>(q.x * ratio, q.y * ratio, q.z * ratio, q.w * ratio));
    }
  }
  for (int k0 = 0; k0 < n; k0 += 16) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k = k0 + s * kRows + row;
      if (!on || k >= n || s * kRows + row >= 16) continue;
      if (n > 16) load8<T>(source(k), v[s]);                                   // a short run is still in registers
      uint2 w = make_uint2(0, 0);
      if (inv > 0.f) {
        w.x = p8::encode4<CODE>(v[s][0] * inv, v[s][1] * inv, v[s][2] * inv, v[s][3] * inv);
        w.y = p8::encode4<CODE>(v[s][4] * inv, v[s][5] * inv, v[s][6] * inv, v[s][7] * inv);
      }
      *reinterpret_cast<uint2*>(codes + (at + k) * ps[2]) = w;
    }
  }
  if (lane == 0) *scale_p = scale;
}

template <typename T, int CODE, int D>
__global__ void __launch_bounds__(kWarps * 32) append8_kernel(Append8Args a) {
  const int lane = threadIdx.x & 31, bs = a.p.block_size;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t win = job / (2 * a.p.Hkv);
  const int hw = static_cast<int>(job % (2 * a.p.Hkv)), which = hw & 1, h = hw >> 1;
  const int64_t base = win * a.window;
  if (base >= a.total) return;
  // lane k holds the slot of token base - 1 + k; tokens 1 .. window of them begin runs where nothing continues
  const int64_t t = base - 1 + lane;
  const bool here = lane >= 1 && lane <= a.window && t < a.total;
  const int64_t last_slot = a.p.num_blocks * bs;
  const int64_t slot = (here || (lane == 0 && t >= 0)) ? slot_at(a, t) : -1;
  const int64_t prev = __shfl_up_sync(QKV_FULL_MASK, slot, 1);
  const bool lost = here && (slot >= last_slot || (slot < 0 && !a.slots));
  if (which == 0) {
    const unsigned dropped = __popc(__ballot_sync(QKV_FULL_MASK, lost));
    if (dropped && lane == 0) atomicAdd(&g_tokens_dropped, static_cast<unsigned long long>(dropped));
  }
  const bool first = here && slot >= 0 && slot < last_slot && !(prev >= 0 && prev + 1 == slot && slot % bs != 0);
  unsigned todo = __ballot_sync(QKV_FULL_MASK, first);
  while (todo) {
    const int k = __ffs(todo) - 1;
    todo &= todo - 1;
    const int64_t t0 = base - 1 + k, s0 = __shfl_sync(QKV_FULL_MASK, slot, k);
    const int at = static_cast<int>(s0 % bs);
    int n = 1;
    for (;;) {                                                                 // how far it goes, 32 tokens at a time
      const int64_t u = t0 + n + lane;
      const bool more = u < a.total && at + n + lane < bs && slot_at(a, u) == s0 + n + lane;
      const unsigned m = __ballot_sync(QKV_FULL_MASK, more);
      if (m == QKV_FULL_MASK) { n += 32; continue; }
      n += __ffs(~m) - 1;
      break;
    }
    store_run<T, CODE, D>(a, which, h, t0, n, s0 / bs, at);
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
  // Few tokens: a warp for each, so that their runs go side by side.  Many: a warp looks for the runs of sixteen tokens,
  // because nearly every token continues a run and its warp would only find that out and end.
  a.window = a.total * 2 * pages.Hkv <= 64 * kNumSMs ? 1 : 16;
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
