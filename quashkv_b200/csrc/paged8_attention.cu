// Attention over a cache of 8-bit pages with a scale for each page and KV head: split over the tokens, for single query
// tokens and short blocks of them.
//
//   out_i = sum_j softmax_j(scale q_i . (ks_p kc_j)) vs_p vc_j        p the page of token j, kc and vc its codes
//
// A warp goes over granules of 16 tokens, which one page holds (a page is a multiple of 16 tokens).  Codes come by
// cp.async into a ring of the warp's own; there is no CTA barrier in the loop.  Both products run on the tensor core with
// the tokens in the place of the rows: scores = K (16 tokens x D) times up to eight query rows, outputs = V^T (D x 16
// tokens) times their weights, so a query row costs a column of eight and not a row of sixteen.  A code is exact in fp16;
// which coordinate stands at which place of the inner dimension is free as long as both operands agree, so each lane reads
// contiguous bytes of a token's key and needs no transposition.  Values are transposed by pairing the bytes of two tokens.
//
// Precision.  Query rows are scaled by a power of two to below 2^14 and held as fp16, which is exact for 16-bit types, and
// as hi + lo for fp32.  Weights go in as hi + lo (22 bits, or 2^-34 of the largest), with bf16 queries as hi alone: 2^-11
// at most of each, an eighth of what the output's own rounding takes.  Softmax in base 2 with two whole-number reference
// exponents a row, so that rescaling is exact: m for the scores t, M for t + log2 of the page's value scale.  The weights
// of the second product, 2^(t - M) vs, are then at most 2^15 and the largest at least 2^9 whatever the scales are: a page
// of large values that a row hardly weighs takes no bits from the others.  References rise when a score is 4 above them,
// which is rare after the first granules.  M is held as dM = M - m, which stays exact where scores are so large (from 2^24 on)
// that m + 1 is no number any more; there the largest score has all the weight, as it should.
//
// Bound by the bytes of the pages: (2 D + 8 / block_size) a token and KV head.  Measured, 32 x 8 KV heads x 32768 tokens of 128, four
// bf16 queries a head: 365-408 us by the box, 5.3-5.9 TB/s; the schedulers' issue slots are 48 % busy, their three warps mostly wait for results of their own.
// fp32 queries take four MMAs in place of one, and 16 rows fill the registers (two CTAs an SM): 32 sequences of up to 16384
// tokens, 16 rows a head: 242 us, 2.6 TB/s, bound by the latency of a warp's own chain.
#include <math.h>

#include <cooperative_groups.h>

#include "mma_decode.cuh"
#include "paged8.cuh"
#include "paged8_attention.cuh"

namespace qkv {

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 2;               // steps of 32 tokens in a warp's ring: one in work, one on its way
constexpr float kNone = -3e38f;          // reference exponent before anything has been seen, and below every score's
// What queries and weights are held as: fp16 once each (bf16), queries once and weights as hi + lo (fp16), both as hi + lo (fp32).
enum { kBF16 = 0, kF16 = 1, kF32 = 2 };
constexpr int kMostCluster = 8;          // CTAs of a cluster (the portable size)
constexpr float kSlack = 4.f;
constexpr float kLift = 10.f;            // the largest weight is at least 2^(kLift - 1): fp16's least step is 2^-33 of it at most, half of it 2^-34

// Bytes from one token's row to the next in the ring: without bank conflicts for both operands' reads.
template <int D> struct Pitch { static constexpr int kKey = D == 128 || D == 96 ? D + 16 : D, kVal = D + 16; };

template <int D, int NG> struct Split {
  static constexpr int kGranule = 16 * (Pitch<D>::kKey + Pitch<D>::kVal), kSlot = 2 * kGranule;
  static constexpr int kRows = 8 * NG;
  static constexpr int kAccPitch = D + 4;
  static constexpr size_t kRing = static_cast<size_t>(kWarps) * kStages * kSlot;
  static constexpr size_t kOwn = static_cast<size_t>(kWarps) * kRows * (kAccPitch + 4) * 4;      // where the CTA's sums stand for its cluster
  static constexpr size_t kMerge = kOwn + static_cast<size_t>(kRows) * (D + 4) * 4;
  static constexpr size_t kSmem = kRing > kMerge ? kRing : kMerge;
};

// N words from shared memory, as wide as their address allows.
template <int N> __device__ __forceinline__ void lds(uint32_t (&w)[N], const unsigned char* p) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 x = reinterpret_cast<const uint2*>(p)[i];
      w[2 * i] = x.x; w[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
}

// CTAs on an SM that the registers allow for.
__host__ __device__ constexpr int resident(int d, int ng) { return d > 64 ? (ng == 1 ? 3 : 2) : (ng == 1 ? 4 : 3); }

template <int D, int CODE, int KIND, int NG>
__global__ void __launch_bounds__(kWarps * 32, resident(D, NG)) paged8_split_kernel(Attn8Args a) {
  using P = Split<D, NG>;
  constexpr int QT = KIND == kF32 ? 2 : 1, WT = KIND == kBF16 ? 1 : 2;      // terms of queries and weights
  constexpr int kR = P::kRows, kKeyPitch = Pitch<D>::kKey, kValPitch = Pitch<D>::kVal;
  constexpr int kChunks = D;                               // 16-byte chunks of 16 rows of D bytes
  constexpr int kCopies = (kChunks + 31) / 32;
  constexpr int kKW = D / 16, kVW = D / 32;                // words of a lane: of a key row, of a value row
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");

  int item = blockIdx.x;
  const int rt = item % a.row_tiles;
  item /= a.row_tiles;
  const int h = item % a.Hkv, seq = item / a.Hkv;
  const Span8 s = span8(a, seq);
  // A launch that overlaps the prefill kernel in front of it ends after it: what follows may rely on both.
  auto leave = [&] {
    if (a.behind_prefill && blockIdx.x == 0 && blockIdx.y == 0) asm volatile("griddepcontrol.wait;\n" ::: "memory");
  };
  if (a.starts && rt == 0 && blockIdx.y == 0) zero_gaps8(a, s, seq, h);
  const int rows = a.G * s.q_len, r0 = rt * kR;
  if (r0 >= rows || rows > a.most_rows) return leave();
  const int r_end = min(r0 + kR, rows);
  const int64_t end = visible8(a, s, (r_end - 1) / a.G);
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * a.chunk, stop = min(end, begin + a.chunk);
  if (begin > 0 && begin >= end && !a.in_cluster) return leave();      // (in a cluster it goes on with nothing to add)

  // ---- queries: operand B of the scores, row r0 + 8 ng + g in column g ----
  uint32_t qf[NG][QT][kKW][2];
  float unit[NG][2];                                       // score (base 2) per unit of the product, rows 2t and 2t + 1
  int lim[NG][2];                                          // last token that they see, relative to `begin`
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int r = r0 + 8 * n + g;
    const bool live = r < r_end;
    float v[D / 4], mx = 0.f;
    if (live) {
      const int64_t at = s.q_row0 + static_cast<int64_t>(r / a.G) * a.q_stride[1] + static_cast<int64_t>(h * a.G + r % a.G) * a.q_stride[2] + t * (D / 4);
      load_row8<D / 4>(a.q, a.dtype, at, v);
    } else {
#pragma unroll
      for (int i = 0; i < D / 4; ++i) v[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) mx = fmaxf(mx, fabsf(v[i]));
    mx = fmaxf(mx, __shfl_xor_sync(QKV_FULL_MASK, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(QKV_FULL_MASK, mx, 2));
    const float up = scale_to8<13>(mx);
#pragma unroll
    for (int k = 0; k < kKW; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = v[4 * k + 2 * e] * up, y = v[4 * k + 2 * e + 1] * up;
        const __half2 hi = __floats2half2_rn(x, y);
        qf[n][0][k][e] = *reinterpret_cast<const uint32_t*>(&hi);
        if (QT == 2) {
          const float2 f = __half22float2(hi);
          qf[n][QT - 1][k][e] = pack_half2(x - f.x, y - f.y);
        }
      }
    const float u = a.scale * 1.4426950408889634f * inverse8(up);
    const int64_t see = live ? visible8(a, s, r / a.G) : 0;
    const int last = static_cast<int>(max(min(see - begin, a.chunk), static_cast<int64_t>(0))) - 1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      unit[n][e] = __shfl_sync(QKV_FULL_MASK, u, 4 * (2 * t + e));
      lim[n][e] = __shfl_sync(QKV_FULL_MASK, last, 4 * (2 * t + e));
    }
  }
  // tokens up to this one are seen by every row (rows behind the last one do not count: their results are not kept)
  const int all_see = static_cast<int>(max(min(visible8(a, s, r0 / a.G) - begin, a.chunk), static_cast<int64_t>(0))) - 1;

  float acc[NG][2 * kVW][4];                               // [m tile]: coordinates 2j, 2j + 1 of the lane's, rows 2t, 2t + 1
  float m[NG][2], dM[NG][2], l[NG][2];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
#pragma unroll
    for (int j = 0; j < 2 * kVW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) { m[n][e] = kNone; dM[n][e] = -0.5f * kNone; l[n][e] = 0.f; }
  }

  // ---- granules: this warp has the pairs warp, warp + 4, ... of the chunk ----
  // Two granules a step: their products are independent of one another, and the test of the references, the waits and the
  // bookkeeping are done once for both.
  const int pairs = stop > begin ? static_cast<int>((stop - begin + 31) >> 5) : 0;
  const int count = pairs > warp ? (pairs - warp + kWarps - 1) / kWarps : 0;
  const int stored = static_cast<int>(min(s.len - begin, a.chunk));        // tokens that the cache holds from `begin` on
  const int32_t* row = a.table + seq * a.table_stride;
  unsigned char* ring = smem + warp * kStages * P::kSlot;
  // page and scales of granule `lane` of the batch of 16 steps in work, and of the next one
  auto token_of = [&](int x) { return 32 * (warp + kWarps * (x >> 1)) + 16 * (x & 1); };      // x: granule of the warp, relative to begin
  auto page_of = [&](int x) -> int {
    const int rel = token_of(x);
    if ((x >> 1) >= count || rel >= stored) return -1;
    const int64_t tok = begin + rel;
    const int id = row[a.bs_shift >= 0 ? tok >> a.bs_shift : tok / a.p.block_size];
    return id >= 0 && id < a.p.num_blocks ? id : -1;
  };
  auto scale_k = [&](int id) { return id < 0 ? 0.f : a.p.k_scales[id * a.p.ks_stride[0] + h * a.p.ks_stride[1]]; };
  auto scale_v = [&](int id) { return id < 0 ? 0.f : a.p.v_scales[id * a.p.vs_stride[0] + h * a.p.vs_stride[1]]; };
  // first byte of the granule's keys and values: computed by its lane, once
  const uint8_t* k_head = a.p.k_codes + h * a.p.k_stride[1];
  const uint8_t* v_head = a.p.v_codes + h * a.p.v_stride[1];
  auto offset_of = [&](int x) {
    const int64_t tok = begin + token_of(x);
    return static_cast<int>(a.bs_shift >= 0 ? tok & ((1 << a.bs_shift) - 1) : tok % a.p.block_size);
  };
  auto key_at = [&](int x, int id) { return reinterpret_cast<uint64_t>(id < 0 ? nullptr : k_head + id * a.p.k_stride[0] + offset_of(x) * a.p.k_stride[2]); };
  auto val_at = [&](int x, int id) { return reinterpret_cast<uint64_t>(id < 0 ? nullptr : v_head + id * a.p.v_stride[0] + offset_of(x) * a.p.v_stride[2]); };
  int k_src[kCopies], dst_k[kCopies], dst_v[kCopies];      // this lane's chunks of a granule: row, then where they go
#pragma unroll
  for (int c = 0; c < kCopies; ++c) {
    const int x = lane + 32 * c, rw = x / (D / 16), col = 16 * (x % (D / 16));
    k_src[c] = rw << 8 | col;
    dst_k[c] = rw * kKeyPitch + col;
    dst_v[c] = 16 * kKeyPitch + rw * kValPitch + col;
  }
  auto issue = [&](int i, uint64_t kat, uint64_t vat) {    // codes of step i; addresses of its batch, by lane
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int from = (2 * i + u) & 31;
      const uint64_t kp = __shfl_sync(QKV_FULL_MASK, kat, from), vp = __shfl_sync(QKV_FULL_MASK, vat, from);
      unsigned char* dst = ring + (i % kStages) * P::kSlot + u * P::kGranule;
      if (i < count && kp) {
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          cp_async16(dst + dst_k[c], reinterpret_cast<const uint8_t*>(kp) + (k_src[c] >> 8) * a.p.k_stride[2] + (k_src[c] & 255), 16);
          cp_async16(dst + dst_v[c], reinterpret_cast<const uint8_t*>(vp) + (k_src[c] >> 8) * a.p.v_stride[2] + (k_src[c] & 255), 16);
        }
      }
    }
    cp_async_commit();                                     // one group a step, empty ones too
  };
  int pg = page_of(lane), pg_next = -1;
  uint64_t kat = key_at(lane, pg), vat = val_at(lane, pg), kat_next = 0, vat_next = 0;
  issue(0, kat, vat);
  float ksc = scale_k(pg), vsc = scale_v(pg), ksc_next = 0.f, vsc_next = 0.f;

  for (int i = 0; i < count; ++i) {
    const int b = i & 15;
    if (b == 0) {
      if (i > 0) { pg = pg_next; ksc = ksc_next; vsc = vsc_next; kat = kat_next; vat = vat_next; }
      pg_next = page_of(2 * i + 32 + lane);
    }
    if (b == 8) {
      ksc_next = scale_k(pg_next);
      vsc_next = scale_v(pg_next);
      kat_next = key_at(2 * (i - 8) + 32 + lane, pg_next);
      vat_next = val_at(2 * (i - 8) + 32 + lane, pg_next);
    }
    if (b == 15) issue(i + 1, kat_next, vat_next); else issue(i + 1, kat, vat);
    cp_async_wait<1>();
    __syncwarp();

    const unsigned char* slot = ring + (i % kStages) * P::kSlot;
    const int tok = 32 * (warp + kWarps * i);              // relative to begin
    float ks[2], vs[2];
    int valid[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int id = __shfl_sync(QKV_FULL_MASK, pg, 2 * b + u);
      ks[u] = __shfl_sync(QKV_FULL_MASK, ksc, 2 * b + u);
      vs[u] = __shfl_sync(QKV_FULL_MASK, vsc, 2 * b + u);
      valid[u] = id < 0 ? 0 : max(0, min(16, stored - tok - 16 * u));
    }
    const bool whole = valid[0] + valid[1] == 32 && tok + 31 <= all_see;   // every row sees every token

    // ---- scores ----
    float sc[2][NG][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t w0[kKW], w1[kKW];
      lds<kKW>(w0, slot + u * P::kGranule + g * kKeyPitch + t * (D / 4));
      lds<kKW>(w1, slot + u * P::kGranule + (g + 8) * kKeyPitch + t * (D / 4));
      float part[NG][2][4];
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[n][0][e] = part[n][1][e] = 0.f;
#pragma unroll
      for (int k = 0; k < kKW; ++k) {
        const uint32_t x = p8::biased<CODE>(w0[k]), y = p8::biased<CODE>(w1[k]);
        const uint32_t av[4] = {p8::halves_low<CODE>(x), p8::halves_low<CODE>(y), p8::halves_high<CODE>(x), p8::halves_high<CODE>(y)};
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          if (QT == 2) mma16816(part[n][k & 1], av, qf[n][QT - 1][k][0], qf[n][QT - 1][k][1]);
          mma16816(part[n][k & 1], av, qf[n][0][k][0], qf[n][0][k][1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[u][n][e] = (part[n][0][e] + part[n][1][e]) * (ks[u] * unit[n][e & 1]);
    }
    if (!whole) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = g + 8 * (e >> 1);
            if (k >= valid[u] || tok + 16 * u + k > lim[n][e & 1]) sc[u][n][e] = -INFINITY;
          }
    }

    // ---- weights ----
    // vs = mant * 2^ex; a scale of 0 weighs nothing
    float ex[2], mant[2];
    bool nan_page = false;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t vbits = __float_as_uint(vs[u]);
      const int vexp = static_cast<int>((vbits >> 23) & 255u);
      ex[u] = vexp ? static_cast<float>(vexp - 127) : kNone;
      mant[u] = vexp ? (vexp == 255 ? vs[u] : __uint_as_float((vbits & 0x807fffffu) | 0x3f800000u)) : 0.f;
      nan_page |= vexp == 255;
    }
    bool rise = false;
    float top[2][NG][2];                                   // of this lane's tokens
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int u = 0; u < 2; ++u) top[u][n][e] = fmaxf(sc[u][n][e], sc[u][n][e + 2]);
        const float t0 = top[0][n][e] - m[n][e], t1 = top[1][n][e] - m[n][e];
        rise |= fmaxf(t0, t1) > kSlack || fmaxf(t0 + ex[0], t1 + ex[1]) > dM[n][e] + (kLift + kSlack);
      }
    if (__any_sync(QKV_FULL_MASK, rise)) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = top[0][n][e], y = top[1][n][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            x = fmaxf(x, __shfl_xor_sync(QKV_FULL_MASK, x, o));
            y = fmaxf(y, __shfl_xor_sync(QKV_FULL_MASK, y, o));
          }
          const float m1 = fmaxf(m[n][e], ceilf(fmaxf(x, y)));
          const float was = dM[n][e] + (m[n][e] - m1), dM1 = fmaxf(was, ceilf(fmaxf(x - m1 + ex[0], y - m1 + ex[1])) - kLift);
          l[n][e] *= ex2(m[n][e] - m1);
          const float f = ex2(was - dM1);
          m[n][e] = m1;
          dM[n][e] = dM1;
#pragma unroll
          for (int j = 0; j < 2 * kVW; ++j) {
            acc[n][j][e] *= f;
            acc[n][j][e + 2] *= f;
          }
        }
    }
    uint32_t wh[2][NG][2], wl[2][NG][2];                   // operand B of the second product: tokens x rows
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = sc[u][n][e] - m[n][e & 1];
          l[n][e & 1] += ex2(x);
          w[e] = ex2(x + (ex[u] - dM[n][e & 1])) * mant[u];
        }
        if (!whole && nan_page) {                          // a page of NaN: nothing from tokens that are not seen
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (sc[u][n][e] == -INFINITY) w[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const __half2 hi = __floats2half2_rn(w[2 * e], w[2 * e + 1]);
          const float2 f = __half22float2(hi);
          wh[u][n][e] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&hi));
          if (WT == 2) wl[u][n][e] = movmatrix_trans(pack_half2(w[2 * e] - f.x, w[2 * e + 1] - f.y));
        }
      }

    // ---- values: row = coordinate, inner dimension = tokens 2t, 2t + 1, 2t + 8, 2t + 9 ----
    auto fetch = [&](int u, uint32_t (&v)[4][kVW]) {
      const unsigned char* vp = slot + u * P::kGranule + 16 * kKeyPitch + 2 * t * kValPitch + g * (D / 8);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row_of = (r & 1) + 8 * (r >> 1);
        lds<kVW>(v[r], vp + row_of * kValPitch);
        if (valid[u] < 16 && 2 * t + row_of >= valid[u]) { // bytes behind the last token may be anything
#pragma unroll
          for (int k = 0; k < kVW; ++k) v[r][k] = 0;
        }
      }
    };
    auto operands = [&](const uint32_t (&v)[4][kVW], int k, uint32_t (&x)[4], uint32_t (&y)[4]) {      // coordinates 4 k, + 1 and + 2, + 3 of the lane's
      const uint32_t a01 = p8::biased<CODE>(prmt(v[0][k], v[1][k], 0x5140)), a23 = p8::biased<CODE>(prmt(v[0][k], v[1][k], 0x7362));
      const uint32_t b01 = p8::biased<CODE>(prmt(v[2][k], v[3][k], 0x5140)), b23 = p8::biased<CODE>(prmt(v[2][k], v[3][k], 0x7362));
      x[0] = p8::halves_low<CODE>(a01); x[1] = p8::halves_high<CODE>(a01); x[2] = p8::halves_low<CODE>(b01); x[3] = p8::halves_high<CODE>(b01);
      y[0] = p8::halves_low<CODE>(a23); y[1] = p8::halves_high<CODE>(a23); y[2] = p8::halves_low<CODE>(b23); y[3] = p8::halves_high<CODE>(b23);
    };
    if constexpr (QT == 1) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t v[4][kVW];
        fetch(u, v);
#pragma unroll
        for (int k = 0; k < kVW; ++k) {
          uint32_t x[4], y[4];
          operands(v, k, x, y);
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            if (WT == 2) {
              mma16816(acc[n][2 * k], x, wl[u][n][0], wl[u][n][1]);
              mma16816(acc[n][2 * k + 1], y, wl[u][n][0], wl[u][n][1]);
            }
            mma16816(acc[n][2 * k], x, wh[u][n][0], wh[u][n][1]);
            mma16816(acc[n][2 * k + 1], y, wh[u][n][0], wh[u][n][1]);
          }
        }
      }
    } else {
      // The tensor core truncates what it adds to an accumulator: over many steps that would show in fp32, so each step's
      // sum is added in fp32.
      uint32_t v0[4][kVW], v1[4][kVW];
      fetch(0, v0);
      fetch(1, v1);
#pragma unroll
      for (int k = 0; k < kVW; ++k) {
        uint32_t x[2][4], y[2][4];
        operands(v0, k, x[0], y[0]);
        operands(v1, k, x[1], y[1]);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float c[4] = {0.f, 0.f, 0.f, 0.f}, d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < 2; ++u) { mma16816(c, x[u], wl[u][n][0], wl[u][n][1]); mma16816(d, y[u], wl[u][n][0], wl[u][n][1]); }
#pragma unroll
          for (int u = 0; u < 2; ++u) { mma16816(c, x[u], wh[u][n][0], wh[u][n][1]); mma16816(d, y[u], wh[u][n][0], wh[u][n][1]); }
#pragma unroll
          for (int e = 0; e < 4; ++e) { acc[n][2 * k][e] += c[e]; acc[n][2 * k + 1][e] += d[e]; }
        }
      }
    }
    __syncwarp();                                          // the slot may be filled again
  }
  cp_async_wait<0>();

  // ---- the four warps' sums ----
  __syncthreads();                                         // the ring has been read
  float* sums = reinterpret_cast<float*>(smem);            // [warp][row][kAccPitch], then [warp][row][4]: m, dM, l
  float* ref = sums + kWarps * kR * P::kAccPitch;
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[n][e];
      x += __shfl_xor_sync(QKV_FULL_MASK, x, 4);
      x += __shfl_xor_sync(QKV_FULL_MASK, x, 8);
      x += __shfl_xor_sync(QKV_FULL_MASK, x, 16);
      const int r = 8 * n + 2 * t + e;
      if (g == 0) *reinterpret_cast<float4*>(ref + (warp * kR + r) * 4) = make_float4(m[n][e], dM[n][e], x, 0.f);
#pragma unroll
      for (int j = 0; j < 2 * kVW; ++j)
        *reinterpret_cast<float2*>(sums + (warp * kR + r) * P::kAccPitch + g * (D / 8) + 2 * j) = make_float2(acc[n][j][e], acc[n][j][e + 2]);
    }
  __syncthreads();
  const int n_rows = r_end - r0;
  for (int x = threadIdx.x; x < n_rows * (D / 4); x += kWarps * 32) {
    const int r = x / (D / 4), c = 4 * (x % (D / 4));
    float4 q[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) q[w] = *reinterpret_cast<const float4*>(ref + (w * kR + r) * 4);
    float mt = kNone;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mt = max_or_nan(mt, q[w].x);
    float dMt = -0.5f * kNone + (kNone - mt);              // (as of a warp that has seen nothing)
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      q[w].x -= mt;
      q[w].y += q[w].x;
      dMt = max_or_nan(dMt, q[w].y);
    }
    float lt = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(sums + (w * kR + r) * P::kAccPitch + c);
      lt = fmaf(q[w].z, ex2(q[w].x), lt);
      const float f = ex2(q[w].y - dMt);
      o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y); o.z = fmaf(y.z, f, o.z); o.w = fmaf(y.w, f, o.w);
    }
    const int rr = r0 + r;
    if (a.n_splits == 1) {
      store_out8(a, s, h, rr, c, o, dMt, lt);
    } else if (a.in_cluster) {
      float* own = reinterpret_cast<float*>(smem + P::kOwn);
      *reinterpret_cast<float4*>(own + r * D + c) = o;
      if (c == 0) *reinterpret_cast<float4*>(own + kR * D + r * 4) = make_float4(mt, dMt, lt, 0.f);
    } else {
      const int64_t slot = part_row8(a, s, seq, h, rr) * a.n_splits + blockIdx.y;
      *reinterpret_cast<float4*>(a.part + slot * D + c) = o;
      if (c == 0) *reinterpret_cast<float4*>(a.ref + slot * 4) = make_float4(mt, dMt, lt, 0.f);
    }
  }
  if (a.in_cluster) {                                      // the splits of these rows are one cluster: joined through shared memory
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int parts = end > a.chunk ? static_cast<int>((end + a.chunk - 1) / a.chunk) : 1;
    float* own = reinterpret_cast<float*>(smem + P::kOwn);
    for (int x = blockIdx.y * (kWarps * 32) + threadIdx.x; x < n_rows * (D / 4); x += a.n_splits * (kWarps * 32)) {
      const int r = x / (D / 4), c = 4 * (x % (D / 4));
      float4 q[kMostCluster], y[kMostCluster];
#pragma unroll
      for (int p = 0; p < kMostCluster; ++p) {
        const float* theirs = cluster.map_shared_rank(own, p < parts ? p : 0);
        q[p] = p < parts ? *reinterpret_cast<const float4*>(theirs + kR * D + r * 4) : make_float4(kNone, -0.5f * kNone, 0.f, 0.f);
        y[p] = *reinterpret_cast<const float4*>(theirs + r * D + c);
      }
      float mt = kNone, lt = 0.f;
#pragma unroll
      for (int p = 0; p < kMostCluster; ++p) mt = max_or_nan(mt, q[p].x);
      float dMt = -0.5f * kNone + (kNone - mt);
#pragma unroll
      for (int p = 0; p < kMostCluster; ++p) {
        q[p].y += q[p].x - mt;
        dMt = max_or_nan(dMt, q[p].y);
      }
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < kMostCluster; ++p) {
        if (p >= parts) continue;
        lt = fmaf(q[p].z, ex2(q[p].x - mt), lt);
        const float f = ex2(q[p].y - dMt);
        o.x = fmaf(y[p].x, f, o.x); o.y = fmaf(y[p].y, f, o.y); o.z = fmaf(y[p].z, f, o.z); o.w = fmaf(y[p].w, f, o.w);
      }
      store_out8(a, s, h, r0 + r, c, o, dMt, lt);
    }
    cluster.sync();                                        // nobody leaves while others read
  }
  leave();
}

// Parts of a row joined: lane = four coordinates (D / 4 lanes).  A warp joins one row, or (by_token, where rows are many and their
// parts few) kTogether query heads of a token, all of whose loads are in flight at once.
constexpr int kTogether = 4;

template <int D, int R>
__global__ void __launch_bounds__(128) paged8_merge_kernel(Attn8Args a) {
  constexpr int kU = R > 1 ? 1 : 2, kP = R > 1 ? 4 : 8;    // a lane's parts (the prefill kernel makes up to 32); parts in flight
  const int lane = threadIdx.x & 31, c = 4 * lane;
  const uint32_t job = blockIdx.x * 4 + (threadIdx.x >> 5), chunk = static_cast<uint32_t>(a.chunk);      // (32 bits: divisions of 64 took most of the time)
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  int seq, h, rr, rows_here = 1;
  int64_t row0;                                            // among the partial results
  Span8 s;
  if (R > 1) {
    const uint32_t hq = a.Hkv * a.G, groups = (hq + R - 1) / R, tok = job / groups, head = (job - tok * groups) * R;
    if (tok >= (a.starts ? a.total_q : static_cast<int64_t>(a.n_seq) * a.q_len)) return;
    if (a.starts) {                                        // the last sequence that starts at or in front of it: 32 at a time
      int lo = 0, n = a.n_seq;
      while (n > 1) {
        const int step = (n + 31) / 32, k = lane * step;
        const uint32_t in = __ballot_sync(QKV_FULL_MASK, k < n && a.starts[lo + (k < n ? k : 0)] <= static_cast<int64_t>(tok));
        const int skip = in ? (__popc(in) - 1) * step : 0;
        lo += skip;
        n = min(step, n - skip);
      }
      seq = lo;
    } else {
      seq = static_cast<int>(tok / static_cast<uint32_t>(a.q_len));
    }
    s = span8(a, seq);
    if (tok < s.tok0 || tok - s.tok0 >= s.q_len) return;
    h = head / a.G;
    rr = static_cast<int>(tok - s.tok0) * a.G + head % a.G;
    rows_here = min(static_cast<uint32_t>(R), hq - head);
    row0 = static_cast<int64_t>(tok) * hq + head;
  } else {
    const uint32_t head = job / static_cast<uint32_t>(a.most_rows);
    if (head >= static_cast<int64_t>(a.n_seq) * a.Hkv) return;
    rr = static_cast<int>(job - head * a.most_rows);
    seq = static_cast<int>(head / a.Hkv);
    h = static_cast<int>(head - seq * static_cast<uint32_t>(a.Hkv));
    s = span8(a, seq);
    row0 = job;
  }
  const int rows = a.G * s.q_len;
  if (rr >= rows || rows > a.most_rows || rows <= a.few_rows) return;
  // (rows of a token are of one tile or of neighbours, whose last tokens differ: the parts are counted for each)
  const int in_head = rr % a.G, first = rr - in_head;      // head h * G + in_head of the token, then the next ones (of the next KV heads, too)
  float4 q[R][kU];
  float mt[R], dMt[R], lt[R];
  int parts[R], most = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = first + (in_head + r) % a.G, te = min((row / a.tile_rows + 1) * a.tile_rows, rows);
    const uint32_t end = static_cast<uint32_t>(visible8(a, s, (te - 1) / a.G));
    parts[r] = r < rows_here ? (end > chunk ? static_cast<int>((end + chunk - 1) / chunk) : 1) : 0;
    most = max(most, parts[r]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int u = 0; u < kU; ++u)
      q[r][u] = lane + 32 * u < parts[r] ? *reinterpret_cast<const float4*>(a.ref + ((row0 + r) * a.n_splits + lane + 32 * u) * 4) : make_float4(kNone, -0.5f * kNone, 0.f, 0.f);
  float4 y[R][kP];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < kP; ++k)
        y[r][k] = c < D && p0 + k < parts[r] ? __ldcs(reinterpret_cast<const float4*>(a.part + ((row0 + r) * a.n_splits + p0 + k) * D + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  fetch(0);
  float4 o[R];
  // lanes that hold parts: the first ones, a power of two
  const int width = most > 16 ? 32 : (most > 8 ? 16 : (most > 4 ? 8 : (most > 2 ? 4 : 2)));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mt[r] = q[r][0].x;
    if (kU > 1) mt[r] = max_or_nan(mt[r], q[r][kU - 1].x);
  }
#pragma unroll 1
  for (int x = width >> 1; x > 0; x >>= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) mt[r] = max_or_nan(mt[r], __shfl_xor_sync(QKV_FULL_MASK, mt[r], x));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mt[r] = __shfl_sync(QKV_FULL_MASK, mt[r], 0);
#pragma unroll
    for (int u = 0; u < kU; ++u) q[r][u].y += q[r][u].x - mt[r];
    dMt[r] = q[r][0].y;
    if (kU > 1) dMt[r] = max_or_nan(dMt[r], q[r][kU - 1].y);
  }
#pragma unroll 1
  for (int x = width >> 1; x > 0; x >>= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) dMt[r] = max_or_nan(dMt[r], __shfl_xor_sync(QKV_FULL_MASK, dMt[r], x));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    dMt[r] = __shfl_sync(QKV_FULL_MASK, dMt[r], 0);
    lt[r] = 0.f;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      lt[r] = fmaf(q[r][u].z, ex2(q[r][u].x - mt[r]), lt[r]);
      q[r][u].w = ex2(q[r][u].y - dMt[r]);
    }
    o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll 1
  for (int x = width >> 1; x > 0; x >>= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) lt[r] += __shfl_xor_sync(QKV_FULL_MASK, lt[r], x);
#pragma unroll
  for (int r = 0; r < R; ++r) lt[r] = __shfl_sync(QKV_FULL_MASK, lt[r], 0);
  for (int p0 = 0;;) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < kP; ++k) {
        const float f = __shfl_sync(QKV_FULL_MASK, p0 + k < 32 ? q[r][0].w : q[r][kU - 1].w, (p0 + k) & 31);
        o[r].x = fmaf(y[r][k].x, f, o[r].x); o[r].y = fmaf(y[r][k].y, f, o[r].y); o[r].z = fmaf(y[r][k].z, f, o[r].z); o[r].w = fmaf(y[r][k].w, f, o[r].w);
      }
    p0 += kP;
    if (p0 >= most) break;
    fetch(p0);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int in = in_head + r;
    if (c < D && r < rows_here) store_out8(a, s, h + in / a.G, first + in % a.G, c, o[r], dMt[r], lt[r]);
  }
}

// How a call is carried out.  Sequences of few rows (query tokens x query heads of a KV head) go to the split kernel, those of
// more to the prefill kernel where it exists (head size 64 and 128, 16-bit queries).  us, split / prefill, 16 sequences of 16384
// tokens: 8 KV heads of 128: 48 rows 350 / 520, 64 rows 444 / 525, 96 rows 647 / 533; 4 of 64: 64 rows 160 / 220, 96 rows 222 / 220, 128
// rows 272 / 181; 64 x 1024 tokens: 64 rows 157 / 155 and 53 / 69, 96 rows 229 / 157 and 73 / 69.  In a ragged batch the
// split kernel has CTAs for the most rows of every sequence, which mostly end at once: 63 single tokens and a
// piece of 1985 over 4096 tokens 340 us with CTAs for 32 rows, 352 for 64.
constexpr int kFewRows = 64, kFewRagged = 32;

struct Plan8 { int ng, tile_rows, row_tiles, most_rows, n_splits; bool cluster; int64_t chunk, part_rows; size_t ws; };

// `rows_used`: rows that sequences mostly have.
Plan8 plan_split(int n_seq, int Hkv, int most_rows, int rows_used, int64_t max_kv_len, int d) {
  Plan8 p{};
  p.most_rows = most_rows;
  p.ng = rows_used > 8 ? 2 : 1;                            // groups of eight rows in a CTA (16 fp32 rows a head: 236 us in one, 288 in two)
  p.row_tiles = (p.most_rows + 8 * p.ng - 1) / (8 * p.ng);
  const int tiles_used = (rows_used + 8 * p.ng - 1) / (8 * p.ng);
  // Tokens of a split.  What fits one wave of resident CTAs is cut into one (each at least a step of its four warps); more
  // is cut five times finer than a wave, so that the last CTAs to run, and sequences of different lengths, leave little
  // of the chip idle.  Measured, 32 x 8 heads x 32768 tokens: 16384 tokens 440 us, 8192 384, 4096 367, 2048 376, 1024 404;
  // 8 heads x 1000: 64 tokens 11.6 us, 128 11.2, 512 13.7; 32 x 8 x 1277 in one split (256 CTAs of 444) 24 us, in two (512) 31.
  const int64_t wave = 3 * kNumSMs, per = (static_cast<int64_t>(n_seq) * Hkv * tiles_used * max_kv_len + wave - 1) / wave;
  const int64_t used = static_cast<int64_t>(n_seq) * Hkv * tiles_used, room = resident(d, p.ng) * kNumSMs;
  const int64_t one = used > 0 && used <= room ? (max_kv_len + room / used - 1) / (room / used) : max_kv_len;      // tokens, with which it is one wave
  p.chunk = per <= 2048 ? (one <= 2048 ? one : per) : (per / 5 < 1024 ? 1024 : (per / 5 > 4096 ? 4096 : per / 5));
  if (p.chunk < 128) p.chunk = 128;
  // Rows for more than eight waves need no splits (fp32, 8 KV heads of 128: 8192 x 4 rows 4702 us in two, 4382 whole).
  if (used > 8 * wave) p.chunk = max_kv_len > 0 ? max_kv_len : 1;
  // Few rows over a short cache: the splits of a row tile are one cluster, whose CTAs join their sums through shared memory:
  // no second launch and no workspace (8 heads x 1000 tokens 12.0 -> 10.3 us, 8 x 4 heads of 64 x 1277 12.1 -> 10.9).  Above 2048
  // tokens the one launch speaks for it, not the time (in a graph, 8 heads of 128, joined in a cluster / by a second launch: 2000
  // tokens 10.3 / 10.3 us, 3000 12.3 / 11.5, 4096 12.3 / 12.3; two sequences of 4096 14.4 / 12.3; 4 heads of 64, 4096 12.0 / 10.3).  Not where
  // there are CTAs for more than two an SM: a cluster is held up by its longest split and by those that have nothing
  // (32 x 8 x up to 1278 in two splits 39 -> 48 us for the whole step).
  const int64_t items = static_cast<int64_t>(n_seq) * Hkv * p.row_tiles;
  const int64_t finest = max_kv_len <= 4096 && items * kMostCluster <= 2 * kNumSMs ? kMostCluster : 64;
  if (p.chunk < (max_kv_len + finest - 1) / finest) p.chunk = (max_kv_len + finest - 1) / finest;
  p.chunk = (p.chunk + 127) / 128 * 128;
  p.n_splits = static_cast<int>((max_kv_len + p.chunk - 1) / p.chunk);
  if (p.n_splits < 1) p.n_splits = 1;
  p.part_rows = static_cast<int64_t>(n_seq) * Hkv * p.most_rows;
  p.cluster = p.n_splits > 1 && p.n_splits <= kMostCluster && items * p.n_splits <= 2 * kNumSMs;
  p.ws = p.n_splits > 1 && !p.cluster ? static_cast<size_t>(p.part_rows) * p.n_splits * (d + 4) * sizeof(float) : 0;
  return p;
}

// `tokens`: query tokens of all sequences, of which a ragged batch may have a few that are long (counted as if they were one).
Plan8 plan_prefill(int n_seq, int Hkv, int G, int q_len, bool ragged, int64_t tokens, int64_t max_kv_len, int d) {
  Plan8 p{};
  p.most_rows = G * q_len;
  auto ctas_of = [&](int rows) { return (ragged ? (tokens * G + rows - 1) / rows : static_cast<int64_t>(n_seq) * ((p.most_rows + rows - 1) / rows)) * Hkv; };
  p.tile_rows = prefill8_rows(d);
  // Fewer rows in a CTA where SMs are idle and the cache is short (a long one is better split).  us, full CTAs / fewer rows: one sequence,
  // 4 KV heads of 64, 8 query heads each: 1024 tokens 51 / 34, 512 30 / 22, 64 over 4096 39 / 30, 512 over 8192 94 / 158; 8 heads of
  // 128, 4 query heads each: 512 tokens 24.7 / 23.6, 256 over 2048 37 / 39, 512 over 8192 106 / 154; ragged, 15 and 512 over 1024 51 / 57.
  if (!ragged && max_kv_len <= (d == 64 ? 4096 : 1024))
    while (p.tile_rows > 128 && ctas_of(p.tile_rows / 2) <= kNumSMs) p.tile_rows /= 2;
  p.row_tiles = (p.most_rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t ctas = ctas_of(p.tile_rows);
  int64_t splits = ctas > 0 ? kNumSMs / ctas : 1;
  // What leaves SMs idle is split over its tokens, into parts of at least 512 (one sequence, 8 KV heads of 128, bf16: 32 x 4 rows
  // over 4096 tokens 30 us, 81 whole, 30 at 256 tokens, 37 at 1024; 512 x 4 over 8192 107, 164 whole).  In a ragged batch of at least 2048, and where the
  // SMs are enough for no more than two, those only from 8192 tokens on, because other sequences use those SMs too and the join is not free: 15 single tokens
  // and a piece of 512 over 1024 tokens 50 us whole, 61 in parts of 512; 31 and 512 over 4096 118 whole, 137 in two; 15 and 256 over
  // 4096 114 whole, 83 in parts of 2048; 3 and 512 over 8192 180 whole, 122 in two.  Where a batch has one request, or a few, those
  // SMs are idle and this is too cautious (one piece, ragged / the same rows dense: 8 heads of 128, 200 x 4 rows over 3500 98 / 43 us,
  // 512 x 4 over 8000 166 / 105; 4 heads of 64, 64 x 8 over 3500 122 / 29): such a batch is better given as a dense call.
  if (ragged && splits == 2 && max_kv_len < 8192) splits = 1;
  const int64_t most = max_kv_len / (ragged ? 2048 : 512);
  if (splits > most) splits = most;
  if (splits > 32) splits = 32;
  if (splits < 1) splits = 1;
  p.chunk = (max_kv_len + splits - 1) / splits;
  p.chunk = (p.chunk + 127) / 128 * 128;
  if (p.chunk < 128) p.chunk = 128;
  p.n_splits = static_cast<int>((max_kv_len + p.chunk - 1) / p.chunk);
  if (p.n_splits < 1) p.n_splits = 1;
  p.part_rows = tokens * Hkv * G;
  p.ws = p.n_splits > 1 ? static_cast<size_t>(p.part_rows) * p.n_splits * (d + 4) * sizeof(float) : 0;
  return p;
}

struct Route8 { bool split, prefill; Plan8 s, p; size_t ws; };

Route8 route8(int n_seq, int Hkv, int G, int q_len, bool ragged, int64_t tokens, int64_t max_kv_len, int d, int dtype) {
  Route8 r{};
  const int rows = G * q_len;
  const int few = ragged ? kFewRagged : kFewRows;
  r.prefill = rows > few && dtype != QKV_F32 && (d == 64 || d == 128);
  r.split = !r.prefill || ragged;                          // (it clears the rows of no sequence, too)
  if (r.split) r.s = plan_split(n_seq, Hkv, r.prefill ? few : rows, r.prefill ? G : rows, r.prefill && G > few ? 0 : max_kv_len, d);
  if (r.prefill) r.p = plan_prefill(n_seq, Hkv, G, q_len, ragged, tokens, max_kv_len, d);
  r.ws = r.s.ws + r.p.ws;                                  // they overlap: each has a place of its own
  return r;
}

// A launch: as a programmatic dependent of the one in front of it (`early`), in clusters of `cluster` CTAs along y.
int launch_as(void (*kernel)(Attn8Args), dim3 grid, int threads, size_t smem, const Attn8Args& a, bool early, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (early) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = 1;
    attr[cfg.numAttrs].val.clusterDim.y = cluster;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? check_launch() : QKV_ELAUNCH;
}

template <int D>
int launch_merge(const Attn8Args& a, cudaStream_t st) {
  if (a.n_splits == 1 || a.in_cluster) return QKV_OK;
  const int64_t rows = a.by_token ? (a.starts ? a.total_q : static_cast<int64_t>(a.n_seq) * a.q_len) * ((a.Hkv * a.G + kTogether - 1) / kTogether)
                                  : static_cast<int64_t>(a.n_seq) * a.Hkv * a.most_rows;      // a warp each
  if (rows > 0x7fffffffLL) return QKV_EDIM;
  return launch_as(a.by_token ? paged8_merge_kernel<D, kTogether> : paged8_merge_kernel<D, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, a, true, 1, st);
}

template <int D, int CODE, int KIND, int NG>
int launch_split(const Attn8Args& a, int64_t items, cudaStream_t st) {
  using P = Split<D, NG>;
  constexpr auto kernel = paged8_split_kernel<D, CODE, KIND, NG>;
  if (const int rc = allow_smem<kernel>(P::kSmem)) return rc;
  // Behind the prefill kernel of the same call, which it shares nothing with, it starts as soon as that one's CTAs have.
  if (const int rc = launch_as(kernel, dim3(static_cast<unsigned>(items), a.n_splits), kWarps * 32, P::kSmem, a, a.behind_prefill != 0, a.in_cluster ? a.n_splits : 1, st))
    return rc;
  return launch_merge<D>(a, st);
}

template <int D, int CODE, int KIND>
int launch_groups(const Attn8Args& a, int ng, int64_t items, cudaStream_t st) {
  return ng == 2 ? launch_split<D, CODE, KIND, 2>(a, items, st) : launch_split<D, CODE, KIND, 1>(a, items, st);
}
template <int D, int CODE>
int launch_types(const Attn8Args& a, int ng, int64_t items, cudaStream_t st) {
  return a.dtype == QKV_F32 ? launch_groups<D, CODE, kF32>(a, ng, items, st)
       : a.dtype == QKV_F16 ? launch_groups<D, CODE, kF16>(a, ng, items, st) : launch_groups<D, CODE, kBF16>(a, ng, items, st);
}
template <int D>
int launch_codes(const Attn8Args& a, int ng, int64_t items, cudaStream_t st) {
  return a.p.code == QKV_E4M3 ? launch_types<D, p8::kE4M3>(a, ng, items, st) : launch_types<D, p8::kInt8>(a, ng, items, st);
}

bool sizes_ok(int n_seq, int Hq, int Hkv, int q_len, int64_t max_kv_len) {
  return n_seq >= 0 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && q_len >= 0 && max_kv_len >= 0 && max_kv_len <= 0x7fffffffLL - 64 &&
         static_cast<int64_t>(Hq) * (q_len > 0 ? q_len : 1) <= 0x7fffffffLL;
}

}  // namespace
}  // namespace qkv

using namespace qkv;

extern "C" size_t qkv_attention_paged8_workspace_bytes(int n_seq, int Hq, int Hkv, int q_len, int ragged, int64_t total_q,
                                                       int64_t max_kv_len, int d, int q_dtype) {
  if (!sizes_ok(n_seq, Hq, Hkv, q_len, max_kv_len) || n_seq == 0 || q_len == 0 || total_q < 0) return 0;
  return route8(n_seq, Hkv, Hq / Hkv, q_len, ragged != 0, ragged ? total_q : static_cast<int64_t>(n_seq) * q_len, max_kv_len, d, q_dtype).ws;
}

extern "C" int qkv_attention_paged8(const void* q, int q_dtype, const int64_t* q_strides, qkv_pages8_t pages,
                                    const int32_t* block_table, int64_t table_stride, int max_blocks, const int32_t* seq_lens,
                                    const int32_t* query_starts, int64_t total_q, int n_seq, int Hq, int q_len, int64_t max_kv_len,
                                    float scale, int causal, void* out, const int64_t* out_strides, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  return qkv_attention_paged8_from(q, q_dtype, q_strides, pages, block_table, table_stride, max_blocks, seq_lens, query_starts, total_q, nullptr,
                                   n_seq, Hq, q_len, max_kv_len, scale, causal, out, out_strides, workspace, workspace_bytes, stream);
}

extern "C" int qkv_attention_paged8_from(const void* q, int q_dtype, const int64_t* q_strides, qkv_pages8_t pages,
                                         const int32_t* block_table, int64_t table_stride, int max_blocks, const int32_t* seq_lens,
                                         const int32_t* query_starts, int64_t total_q, const int32_t* start_lens, int n_seq, int Hq,
                                         int q_len, int64_t max_kv_len, float scale, int causal, void* out, const int64_t* out_strides,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !q_strides || !block_table || !seq_lens || !out || !out_strides) return QKV_ENULL;
  if (q_dtype != QKV_F32 && q_dtype != QKV_BF16 && q_dtype != QKV_F16) return QKV_EDTYPE;
  if (const int rc = check_pages8(pages)) return rc;
  if (!sizes_ok(n_seq, Hq, pages.Hkv, q_len, max_kv_len) || max_blocks < 1 || table_stride < max_blocks || total_q < 0) return QKV_EDIM;
  const int item = q_dtype == QKV_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) return QKV_EALIGN;
  for (int i = 0; i < 3; ++i)
    if ((q_strides[i] * item & 15) || (out_strides[i] * item & 15)) return QKV_EALIGN;
  if (n_seq == 0 || q_len == 0) return QKV_OK;
  Attn8Args a{};
  a.q = q;
  a.dtype = q_dtype;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = q_strides[i];
    a.o_stride[i] = out_strides[i];
  }
  a.p = pages;
  a.table = block_table;
  a.table_stride = table_stride;
  a.seq_lens = seq_lens;
  a.starts = query_starts;
  a.total_q = total_q;
  a.first = start_lens;
  a.n_seq = n_seq;
  a.Hkv = pages.Hkv;
  a.G = Hq / pages.Hkv;
  a.q_len = q_len;
  const int64_t room = static_cast<int64_t>(max_blocks) * pages.block_size;
  a.max_kv_len = max_kv_len < room ? max_kv_len : room;
  a.causal = causal != 0;
  a.scale = scale;
  a.out = out;
  a.bs_shift = (pages.block_size & (pages.block_size - 1)) == 0 ? __builtin_ctz(pages.block_size) : -1;
  const Route8 r = route8(n_seq, a.Hkv, a.G, q_len, query_starts != nullptr, query_starts ? total_q : static_cast<int64_t>(n_seq) * q_len,
                          max_kv_len, pages.d, q_dtype);
  if (r.ws > workspace_bytes || (r.ws > 0 && !workspace)) return QKV_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15u) return QKV_EALIGN;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto with = [&](const Plan8& p, size_t at) {
    Attn8Args b = a;
    b.row_tiles = p.row_tiles;
    b.most_rows = p.most_rows;
    b.n_splits = p.n_splits;
    b.chunk = p.chunk;
    b.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + at);
    b.ref = b.part + static_cast<size_t>(p.part_rows) * p.n_splits * pages.d;
    return b;
  };
  Attn8Args p = with(r.p, r.s.ws), b = with(r.s, 0);
  if (r.prefill) {
    p.tile_rows = r.p.tile_rows;
    p.by_token = 1;
    p.few_rows = r.split ? kFewRagged : 0;
    if (static_cast<int64_t>(n_seq) * a.Hkv > 0x7fffffffLL || p.row_tiles > 65535) return QKV_EDIM;
    if (const int rc = launch_prefill8(p, st)) return rc;
  }
  if (r.split) {
    b.tile_rows = 8 * r.s.ng;
    b.in_cluster = r.s.cluster;
    b.behind_prefill = r.prefill;
    const int64_t items = static_cast<int64_t>(n_seq) * a.Hkv * r.s.row_tiles;
    if (items > 0x7fffffffLL) return QKV_EDIM;
    int rc;
    switch (pages.d) {
      case 32: rc = launch_codes<32>(b, r.s.ng, items, st); break;
      case 64: rc = launch_codes<64>(b, r.s.ng, items, st); break;
      case 96: rc = launch_codes<96>(b, r.s.ng, items, st); break;
      default: rc = launch_codes<128>(b, r.s.ng, items, st); break;
    }
    if (rc) return rc;
  }
  if (!r.prefill) return QKV_OK;
  return pages.d == 64 ? launch_merge<64>(p, st) : launch_merge<128>(p, st);
}
