// What the attention kernels over 8-bit pages share: arguments, a sequence's rows and tokens, loads of query rows and
// the store of output rows.
#pragma once

#include "mma_decode.cuh"
#include "paged8.cuh"

namespace qkv {

struct Attn8Args {
  const void* q; int dtype;                 // queries and outputs: QKV_F32 / BF16 / F16
  int64_t q_stride[3], o_stride[3];         // elements from one sequence, token, query head to the next
  qkv_pages8_t p;
  const int32_t* table; int64_t table_stride; int bs_shift;      // log2 of block_size, -1 where it has none
  const int32_t* seq_lens;
  const int32_t* starts; int64_t total_q;   // ragged queries: rows starts[i] .. starts[i + 1] of total_q are sequence i's
  const int32_t* first;                     // position of a sequence's first query token; nullptr: its queries are its last positions
  int n_seq, Hkv, G, q_len, causal;         // q_len: of every sequence, or the most of any
  int64_t max_kv_len;                       // within the tables
  float scale;
  void* out;
  int row_tiles, tile_rows, most_rows, n_splits; int64_t chunk;
  float* part; float* ref;                  // [row][n_splits] sums, and their (m, M - m, l, -); rows as part_row8 numbers them
  int few_rows;                             // sequences of no more rows (query tokens x heads of a KV head) are not this kernel's,
  int by_token;                             // most_rows: nor are those of more.  by_token: see part_row8
  int in_cluster;                           // split kernel: the splits of a row tile are one cluster
  int behind_prefill;                       // split kernel: it overlaps the prefill kernel and has to end after it
  int test_drop_mma;                        // test hook of the prefill kernel
};

int prefill8_rows(int d);                   // query rows of a CTA of the prefill kernel
int launch_prefill8(const Attn8Args& a, cudaStream_t st);
unsigned int prefill8_timeouts();

// Tokens and queries of a sequence, within what the host has promised.
struct Span8 { int64_t len, tok0, pos0; int q_len, q_all; int64_t q_row0, o_row0; };      // tok0: query tokens in front of it; pos0: position of its first

__device__ __forceinline__ Span8 span8(const Attn8Args& a, int seq) {
  Span8 s;
  s.len = min(static_cast<int64_t>(max(a.seq_lens[seq], 0)), a.max_kv_len);
  if (a.starts) {
    const int64_t lo = min(static_cast<int64_t>(max(a.starts[seq], 0)), a.total_q);
    const int64_t hi = min(max(static_cast<int64_t>(a.starts[seq + 1]), lo), a.total_q);
    s.q_all = static_cast<int>(hi - lo);
    s.tok0 = lo;
    s.q_len = min(s.q_all, a.q_len);
    s.q_row0 = lo * a.q_stride[1];
    s.o_row0 = lo * a.o_stride[1];
  } else {
    s.q_len = s.q_all = a.q_len;
    s.tok0 = static_cast<int64_t>(seq) * a.q_len;
    s.q_row0 = seq * a.q_stride[0];
    s.o_row0 = seq * a.o_stride[0];
  }
  s.pos0 = a.first ? max(a.first[seq], 0) : s.len - s.q_all;
  return s;
}

// How many tokens the queries at token `tok` of the sequence's block see.
__device__ __forceinline__ int64_t visible8(const Attn8Args& a, const Span8& s, int tok) {
  if (!a.causal) return s.len;
  const int64_t v = s.pos0 + tok + 1;
  return v < 0 ? 0 : (v > s.len ? s.len : v);
}

// Ragged queries: output rows in front of the first sequence, behind the last one, and of a sequence beyond the promised
// q_len are zeros.  By the CTA that comes first for (sequence, KV head); all of a head's clear what is behind the last sequence.
__device__ __forceinline__ void zero_gaps8(const Attn8Args& a, const Span8& s, int seq, int h) {
  const int item = a.dtype == QKV_F32 ? 4 : 2, chunks = a.p.d * item / 16;
  auto clear = [&](int64_t lo, int64_t hi, int part, int parts) {      // tokens
    for (int64_t x = part * static_cast<int64_t>(blockDim.x) + threadIdx.x; x < (hi - lo) * a.G * chunks; x += parts * static_cast<int64_t>(blockDim.x)) {
      const int64_t row = x / chunks;
      const int c = static_cast<int>(x - row * chunks);
      char* at = static_cast<char*>(a.out) + ((lo + row / a.G) * a.o_stride[1] + (h * a.G + row % a.G) * a.o_stride[2]) * item;
      reinterpret_cast<uint4*>(at)[c] = make_uint4(0, 0, 0, 0);
    }
  };
  if (s.q_len < s.q_all) clear(s.tok0 + s.q_len, s.tok0 + s.q_all, 0, 1);
  if (seq == 0 && s.tok0 > 0) clear(0, s.tok0, 0, 1);
  clear(min(static_cast<int64_t>(max(a.starts[a.n_seq], 0)), a.total_q), a.total_q, seq, a.n_seq);
}

// Row r of KV head h among the partial results: places for most_rows rows of every sequence and head, or, where sequences differ
// much in their rows, for the query tokens that there are.
__device__ __forceinline__ int64_t part_row8(const Attn8Args& a, const Span8& s, int seq, int h, int r) {
  if (a.by_token) return (s.tok0 + r / a.G) * (static_cast<int64_t>(a.Hkv) * a.G) + h * a.G + r % a.G;
  return (static_cast<int64_t>(seq) * a.Hkv + h) * a.most_rows + r;
}

// 2^(K - e) for a magnitude 2^e <= x < 2^(e+1): x times it lies in [2^K, 2^(K+1)).  A normal number, and so is its inverse.
template <int K>
__device__ __forceinline__ float scale_to8(float x) {
  int e = 254 + K - static_cast<int>((__float_as_uint(x) >> 23) & 255u);
  e = e < 1 ? 1 : (e > 253 ? 253 : e);
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}
__device__ __forceinline__ float inverse8(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ float max_or_nan(float a, float b) { return a != a ? a : (b != b ? b : fmaxf(a, b)); }

// N coordinates (a multiple of 8) from element `at` of the queries.
template <int N>
__device__ __forceinline__ void load_row8(const void* q, int dtype, int64_t at, float (&v)[N]) {
  if (dtype == QKV_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 x = __ldg(p + i);
      v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
    }
    return;
  }
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q) + at);
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    const uint4 x = __ldg(p + i);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (dtype == QKV_BF16) {
        v[8 * i + 2 * k] = __uint_as_float(w[k] << 16);
        v[8 * i + 2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[8 * i + 2 * k] = f.x;
        v[8 * i + 2 * k + 1] = f.y;
      }
    }
  }
}

// From sums in units of 2^M to total weight l in units of 2^m (dM = M - m): times x, then times y.  Two factors, because 2^dM alone is below
// the normal numbers (and lost) where value scales are near 2^-126, though the results are not.  0 for a row that has seen nothing.
struct Unit8 { float x, y; };
__device__ __forceinline__ Unit8 unit8(float dM, float l) {
  if (l == 0.f) return {0.f, 0.f};
  const float half = floorf(0.5f * dM);
  return {ex2(half), ex2(dM - half) / l};
}

// Coordinates c .. c + 3 of output row r of KV head h: sums o in units of 2^(m + dM), total weight l in units of 2^m.  A row that has seen
// nothing is zeros.  One rounding, to the queries' type.
__device__ __forceinline__ void store_out8(const Attn8Args& a, const Span8& s, int h, int r, int c, float4 o, float dM, float l) {
  const Unit8 f = unit8(dM, l);                            // (dM is far below 0 where every value was zero)
  o.x = o.x * f.x * f.y; o.y = o.y * f.x * f.y; o.z = o.z * f.x * f.y; o.w = o.w * f.x * f.y;
  const int64_t at = s.o_row0 + static_cast<int64_t>(r / a.G) * a.o_stride[1] + static_cast<int64_t>(h * a.G + r % a.G) * a.o_stride[2] + c;
  if (a.dtype == QKV_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = o;
  } else if (a.dtype == QKV_BF16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(o.x, o.y), y = __floats2bfloat162_rn(o.z, o.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  } else {
    const __half2 x = __floats2half2_rn(o.x, o.y), y = __floats2half2_rn(o.z, o.w);
    *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

}  // namespace qkv
