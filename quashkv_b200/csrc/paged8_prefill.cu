// Attention of many query rows over 8-bit pages on the fifth-generation tensor cores: head_dim 64 and 128, queries of 16 bits.
// Formulas as in paged8_attention.cu.
//
// A CTA holds 256 query rows of one (sequence, KV head), a row being a query token and one of the head's query heads, as
// two row tiles of 128 (the M of an MMA), and goes over tokens in tiles of 128:
//   warps 9-11   bring the codes of a tile from their pages (cp.async) and turn them into fp16 operands in the swizzled
//                order of the tensor core; both K and V as they lie in memory, a row a token: the scores read K with the
//                inner dimension contiguous, the second product reads V with the outer one contiguous, so nothing is
//                transposed
//   warp 8       one thread issues every MMA: scores of a row tile into tensor memory, and weights (tensor memory) times V
//                into an accumulator that stays in tensor memory over the whole sequence
//   warps 0-7    a thread per query row: scores of a tile from tensor memory, softmax, weights as fp16 in their place
// The tensor core works for one row tile while the softmax of the other runs.  Rows hold two whole-number reference
// exponents as in the split kernel, which rise only when a score passes them by 2^4; only then is the accumulator
// rescaled (exactly), by the row's own thread.
//
// Precision: codes are exact in fp16, 16-bit queries too (scaled by a power of two per row); weights are rounded to
// fp16 once, 2^-12 on average of each, which is less than the rounding of the output (2^-9 or, fp16, as much), and the sum of weights is
// fp32 of the unrounded ones.
//
// Bound by the chain of one tile: scores (512 cycles of the tensor core), 128 exponentials a thread (1024 cycles of a
// quarter's unit), second product.
//
// Every wait is bounded; one that runs out is counted (qkv_tensor_core_timeouts) and makes the CTA's rows NaN.
#include <math.h>
#include <stdlib.h>

#include "paged8_attention.cuh"
#include "umma.cuh"

namespace qkv {

namespace {

constexpr int kTok = 128, kRowsT = 128, kStages = 2, kMetaSlots = 4, kGroups = kTok / 16;
constexpr float kNone = -1e30f, kSlack = 4.f, kLift = 10.f;
__device__ unsigned int g_prefill8_timeouts = 0;

struct TileMeta { float ks[kGroups], ex[kGroups], mant[kGroups]; uint32_t bad; uint32_t pad[7]; };   // per group of 16 tokens
static_assert(sizeof(TileMeta) % 16 == 0, "read as 16-byte words");

template <int D> struct Pf8 {
  static constexpr int kQBytes = kRowsT * D * 2, kOpBytes = kTok * D * 2, kRawBytes = kTok * D;
  static constexpr int kUnits = kRawBytes / 512;           // 32 chunks of 16 codes
  static constexpr size_t kSmem = 2 * kQBytes + 2 * kStages * kOpBytes + 2 * kRawBytes + kMetaSlots * sizeof(TileMeta) + 256;
  static_assert(kSmem <= 232448, "shared memory of one CTA");
  static constexpr int kO = 256;                           // tensor memory: scores at 0 and 128, sums at 256 and 256 + 128
};

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
      "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
      "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),
      "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.shared::cta.b64 t, [%0];\n\t}\n" ::"r"(umma::smem_u32(bar)) : "memory");
}

// B operand with its outer dimension contiguous (V as it lies in memory), 128-byte swizzle: 64 outer elements are a row of
// 128 bytes, eight inner steps are 1024 bytes apart, the next 64 outer elements `outer_bytes`.
__device__ __forceinline__ uint64_t smem_desc_outer(uint32_t smem_addr, uint32_t outer_bytes) {
  return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(outer_bytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
constexpr uint32_t kOuterB = 1u << 16;                     // instruction descriptor: operand B has its outer dimension contiguous

template <int D, int CODE>
__global__ void __launch_bounds__(384, 1) paged8_prefill_kernel(Attn8Args a) {
  using P = Pf8<D>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* q_s = smem;                                               // [2]
  unsigned char* k_s = q_s + 2 * P::kQBytes;                               // [kStages]
  unsigned char* v_s = k_s + kStages * P::kOpBytes;                        // [kStages]
  unsigned char* raw_s = v_s + kStages * P::kOpBytes;                      // codes of one K and one V tile
  TileMeta* meta = reinterpret_cast<TileMeta*>(raw_s + 2 * P::kRawBytes);  // [kMetaSlots]
  uint64_t* bars = reinterpret_cast<uint64_t*>(meta + kMetaSlots);
  uint64_t* k_full = bars;                  // [2] 96 threads have stored their part
  uint64_t* v_full = bars + 2;              // [2]
  uint64_t* k_free = bars + 4;              // [2] its MMAs have read it
  uint64_t* v_free = bars + 6;              // [2]
  uint64_t* s_full = bars + 8;              // [2] scores of a row tile; everything issued before has ended, too
  uint64_t* p_ready = bars + 10;            // [2] queries (phase 0), then weights of tile j (phase j + 1)
  uint64_t* o_full = bars + 12;             // [2] all sums
  uint64_t* m_full = bars + 14;             // [4] scales of a tile
  uint64_t* drain = bars + 18;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 19);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  const int h = blockIdx.x % a.Hkv, seq = blockIdx.x / a.Hkv;
  const Span8 s = span8(a, seq);
  const int rows = a.G * s.q_len, r0 = (gridDim.y - 1 - blockIdx.y) * 2 * kRowsT;      // long rows first
  if (r0 >= rows || rows <= a.few_rows) return;
  const int r_end = min(r0 + 2 * kRowsT, rows), nt = r_end - r0 > kRowsT ? 2 : 1;
  const int64_t seen = visible8(a, s, (r_end - 1) / a.G);
  const int64_t begin = static_cast<int64_t>(blockIdx.z) * a.chunk, stop = min(seen, begin + a.chunk);
  if (begin > 0 && begin >= seen) return;
  const int n = stop > begin ? static_cast<int>((stop - begin + kTok - 1) / kTok) : 0;

  if (tid == 0) {
    for (int i = 0; i < 19; ++i) umma::mbar_init(bars + i, i < 4 ? 96 : (i == 10 || i == 11 ? kRowsT : 1));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    *dead = 0;
  }
  if (warp == 0) umma::tmem_alloc(tmem_slot, 512);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) {                        // bounded; false once anything ran out
    if (*dead) return false;
    if (umma::mbar_wait(bar, parity)) return true;
    *dead = 1;
    atomicAdd(&g_prefill8_timeouts, 1u);
    return false;
  };
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(QKV_FULL_MASK, wait(bar, parity)) != 0; };

  if (warp >= 8) {
    // 384 threads start with 168 registers; 256 x 200 + 128 x 104 = 384 x 168
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n");
    if (warp == 8) {
      if (lane == 0) {
        // ---- MMAs ----
        constexpr uint32_t id_s = umma::instr_desc(umma::kFmtF16, 128, kTok), id_o = umma::instr_desc(umma::kFmtF16, 128, D) | kOuterB;
        auto scores = [&](int t, int j) {
          const uint32_t qa = umma::smem_u32(q_s + t * P::kQBytes), ka = umma::smem_u32(k_s + (j % kStages) * P::kOpBytes);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma::mma_f16(tmem + kTok * t, umma::smem_desc_sw128(qa + (k >> 2) * (kRowsT * 128) + (k & 3) * 32),
                          umma::smem_desc_sw128(ka + (k >> 2) * (kTok * 128) + (k & 3) * 32), id_s, k != 0);
          umma::commit(s_full + t);
          if (t == nt - 1) umma::commit(k_free + j % kStages);
        };
        auto values = [&](int t, int j) {
          const uint32_t va = umma::smem_u32(v_s + (j % kStages) * P::kOpBytes);
#pragma unroll
          for (int k = 0; k < kTok / 16; ++k)
            umma::mma_f16_ts(tmem + P::kO + 128 * t, tmem + kTok * t + 8 * k, smem_desc_outer(va + k * 2048, kTok * 128), id_o, j != 0 || k != 0);
          if (t == nt - 1) umma::commit(v_free + j % kStages);
        };
        bool ok = true;
        for (int t = 0; t < nt && ok; ++t) ok = wait(p_ready + t, 0);
        if (n > 0 && ok && (ok = wait(k_full, 0))) {
          umma::fence_after_sync();
          for (int t = 0; t < nt; ++t) scores(t, 0);
        }
        for (int j = 0; j < n && ok; ++j)
          for (int t = 0; t < nt && ok; ++t) {
            if (!(ok = wait(p_ready + t, (j + 1) & 1))) break;
            if (t == 0 && !(ok = wait(v_full + j % kStages, (j / kStages) & 1))) break;
            if (a.test_drop_mma && (blockIdx.x | blockIdx.y | blockIdx.z) == 0 && t == 0 && j == 1) continue;      // test hook
            umma::fence_after_sync();
            values(t, j);
            if (j + 1 == n) {
              umma::commit(o_full + t);
            } else {
              if (t == 0 && !(ok = wait(k_full + (j + 1) % kStages, ((j + 1) / kStages) & 1))) break;
              umma::fence_after_sync();
              scores(t, j + 1);
            }
          }
        if (!ok) {                          // whatever was issued has ended before tensor memory is given back
          umma::commit(drain);
          umma::mbar_wait(drain, 0);
        }
      }
    } else {
      // ---- codes to operands ----
      // Unit u of a tile (32 chunks of 16 codes): block u / 16 of 64 coordinates, group (u / 2) % 8 of 16 tokens, eight of
      // whose tokens are four lanes' each.  This warp has units w, w + 3, ...
      const int w = warp - 9, sub = lane >> 2, c = lane & 3;
      const int32_t* row = a.table + seq * a.table_stride;
      const uint8_t* k_head = a.p.k_codes + h * a.p.k_stride[1];
      const uint8_t* v_head = a.p.v_codes + h * a.p.v_stride[1];
      const uint32_t to0 = sub * 128 + (((2 * c) ^ sub) << 4), to1 = sub * 128 + (((2 * c + 1) ^ sub) << 4);
      // group `lane` (of the first eight) of tile j: its page, the offset inside it, its scales
      auto page_of = [&](int j) -> int {
        const int64_t tok = begin + static_cast<int64_t>(j) * kTok + 16 * (lane & 7);
        if (tok >= stop) return -1;
        const int id = row[a.bs_shift >= 0 ? tok >> a.bs_shift : tok / a.p.block_size];
        return id >= 0 && id < a.p.num_blocks ? id : -1;
      };
      auto offset_of = [&](int j) -> int {
        const int64_t tok = begin + static_cast<int64_t>(j) * kTok + 16 * (lane & 7);
        return static_cast<int>(a.bs_shift >= 0 ? tok & ((1 << a.bs_shift) - 1) : tok % a.p.block_size);
      };
      auto issue = [&](const uint8_t* head, const int64_t* stride, unsigned char* dst, int j, int id, int off) {
#pragma unroll 4
        for (int u = w; u < P::kUnits; u += 3) {
          const int g = (u >> 1) & 7, in = 8 * (u & 1) + sub;
          const int pg = __shfl_sync(QKV_FULL_MASK, id, g), at = __shfl_sync(QKV_FULL_MASK, off, g);
          const bool there = pg >= 0 && begin + static_cast<int64_t>(j) * kTok + 16 * g + in < s.len;
          const uint8_t* src = head + (there ? pg : 0) * stride[0] + (there ? (at + in) * stride[2] + (u >> 4) * 64 + 16 * c : 0);
          cp_async16(dst + u * 512 + lane * 16, src, there ? 16 : 0);      // what is not there is zeros
        }
        cp_async_commit();
      };
      auto convert = [&](const unsigned char* src, unsigned char* dst) {
#pragma unroll 4
        for (int u = w; u < P::kUnits; u += 3) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + u * 512 + lane * 16);
          const uint32_t y[4] = {p8::biased<CODE>(x.x), p8::biased<CODE>(x.y), p8::biased<CODE>(x.z), p8::biased<CODE>(x.w)};
          unsigned char* to = dst + (u >> 4) * (kTok * 128) + (u & 15) * 1024;
          *reinterpret_cast<uint4*>(to + to0) = make_uint4(p8::halves_low<CODE>(y[0]), p8::halves_high<CODE>(y[0]), p8::halves_low<CODE>(y[1]), p8::halves_high<CODE>(y[1]));
          *reinterpret_cast<uint4*>(to + to1) = make_uint4(p8::halves_low<CODE>(y[2]), p8::halves_high<CODE>(y[2]), p8::halves_low<CODE>(y[3]), p8::halves_high<CODE>(y[3]));
        }
        umma::fence_smem_to_async();
      };
      auto scale_of = [&](const float* sc, const int64_t* stride, int id) { return id < 0 ? 0.f : sc[id * stride[0] + h * stride[1]]; };
      unsigned char* raw_k = raw_s;
      unsigned char* raw_v = raw_s + P::kRawBytes;
      int id = n > 0 ? page_of(0) : -1, id1 = n > 1 ? page_of(1) : -1;
      if (n > 0) {
        issue(k_head, a.p.k_stride, raw_k, 0, id, offset_of(0));
        issue(v_head, a.p.v_stride, raw_v, 0, id, offset_of(0));
      }
      float ks = scale_of(a.p.k_scales, a.p.ks_stride, id), vs = scale_of(a.p.v_scales, a.p.vs_stride, id);
      for (int j = 0; j < n; ++j) {
        const int st = j % kStages;
        const uint32_t par = ((j / kStages) & 1) ^ 1;
        const int id2 = j + 2 < n ? page_of(j + 2) : -1;
        cp_async_wait<1>();                                // this thread's chunks of K
        if (j >= kStages && !wait_all(k_free + st, par)) break;
        if (w == 0) {
          TileMeta* mt = meta + j % kMetaSlots;            // (read last by the softmax of tile j - 4, long over)
          if (lane < kGroups) {
            const uint32_t bits = __float_as_uint(vs);
            const int e = static_cast<int>((bits >> 23) & 255u);
            mt->ks[lane] = ks;
            mt->ex[lane] = e ? static_cast<float>(e - 127) : kNone;
            mt->mant[lane] = e ? (e == 255 ? vs : __uint_as_float((bits & 0x807fffffu) | 0x3f800000u)) : 0.f;
          }
          const uint32_t bad = __ballot_sync(QKV_FULL_MASK, lane < kGroups && id < 0);
          if (lane == 0) mt->bad = bad;
          __syncwarp();
          if (lane == 0) arrive(m_full + j % kMetaSlots);
        }
        convert(raw_k, k_s + st * P::kOpBytes);
        arrive(k_full + st);
        const int off1 = offset_of(j + 1);
        if (j + 1 < n) issue(k_head, a.p.k_stride, raw_k, j + 1, id1, off1); else cp_async_commit();
        ks = scale_of(a.p.k_scales, a.p.ks_stride, id1);
        vs = scale_of(a.p.v_scales, a.p.vs_stride, id1);
        cp_async_wait<1>();                                // this thread's chunks of V
        if (j >= kStages && !wait_all(v_free + st, par)) break;
        convert(raw_v, v_s + st * P::kOpBytes);
        arrive(v_full + st);
        if (j + 1 < n) issue(v_head, a.p.v_stride, raw_v, j + 1, id1, off1); else cp_async_commit();
        id = id1;
        id1 = id2;
      }
      cp_async_wait<0>();
    }
  } else {
    // ---- a query row per thread ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;\n");
    const int t = warp >> 2, r = r0 + tid;
    if (t < nt) {
      const bool live = r < r_end;
      const uint32_t my = tmem + kTok * t + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
      float unit;                                          // score (base 2) per unit of the product
      {
        const int64_t at = live ? s.q_row0 + static_cast<int64_t>(r / a.G) * a.q_stride[1] + static_cast<int64_t>(h * a.G + r % a.G) * a.q_stride[2] : 0;
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float v[32];
          if (live) load_row8<32>(a.q, a.dtype, at + c, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, live ? fabsf(v[i]) : 0.f);
        }
        const float up = scale_to8<13>(mx), sg = a.scale < 0.f ? -up : up;      // (a negative scale turns the query round)
        unit = fabsf(a.scale) * 1.4426950408889634f * inverse8(up);
        unsigned char* dst = q_s + t * P::kQBytes;
        const int row = tid & 127;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float v[32];
          if (live) load_row8<32>(a.q, a.dtype, at + c, v);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = live ? pack_half2(v[8 * k + 2 * e] * sg, v[8 * k + 2 * e + 1] * sg) : 0u;
            *reinterpret_cast<uint4*>(dst + umma::sw128_offset(row, c + 8 * k, kRowsT)) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
        umma::fence_smem_to_async();
        arrive(p_ready + t);
      }
      // last token that this row sees, relative to `begin`
      const int lim = live ? static_cast<int>(max(min(visible8(a, s, r / a.G) - begin, a.chunk), static_cast<int64_t>(0))) - 1 : -1;
      float m = kNone, M = 0.5f * kNone, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        if (!(ok = wait_all(s_full + t, j & 1) && wait_all(m_full + j % kMetaSlots, (j / kMetaSlots) & 1))) break;
        umma::fence_after_sync();
        uint32_t x[2][64];
        umma::tmem_ld64_issue(my, x[0]);
        umma::tmem_ld64_issue(my + 64, x[1]);
        const TileMeta& mt = meta[j % kMetaSlots];
        float f[kGroups], ex[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          f[g] = mt.ks[g] * unit;
          ex[g] = mt.ex[g];
        }
        const uint32_t bad = mt.bad;
        const int left = lim - j * kTok;                   // tokens 0 .. left of the tile are visible
        const bool masked = __any_sync(QKV_FULL_MASK, left < kTok - 1) || bad != 0;
        umma::tmem_ld64_wait(x[0]);
        umma::tmem_ld64_wait(x[1]);
        float tm = -INFINITY, tM = -INFINITY;
        if (masked) {
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int k = 16 * g + i;
              uint32_t& y = x[k >> 6][k & 63];
              const float v = (k > left || ((bad >> g) & 1u)) ? -INFINITY : __uint_as_float(y) * f[g];
              y = __float_as_uint(v);
              top = fmaxf(top, v);
            }
            tm = fmaxf(tm, top);
            tM = fmaxf(tM, top + ex[g]);
            f[g] = 1.f;
          }
        } else {
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 16; ++i) top[i & 1] = fmaxf(top[i & 1], __uint_as_float(x[(16 * g + i) >> 6][(16 * g + i) & 63]));
            const float v = fmaxf(top[0], top[1]) * f[g];
            tm = fmaxf(tm, v);
            tM = fmaxf(tM, v + ex[g]);
          }
        }
        const bool rise = tm > m + kSlack || tM > M + (kLift + kSlack);
        if (__any_sync(QKV_FULL_MASK, rise)) {             // scores of this tile are there, so the sums of the one before are
          const float m1 = fmaxf(m, ceilf(tm)), M1 = fmaxf(M, ceilf(tM) - kLift);
          l *= ex2(m - m1);
          const float alpha = ex2(M - M1);
          m = m1;
          M = M1;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              umma::tmem_ld32(my + (P::kO + c), o);        // the sums of row tile t are kO columns behind its scores
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st32(my + (P::kO + c), o);
            }
          }
        }
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t wt[32];
#pragma unroll
          for (int g4 = 0; g4 < 4; ++g4) {
            const int g = 4 * hf + g4;
            const float up = mt.mant[g] * ex2(fminf(m + ex[g] - M, 120.f));
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float p0 = ex2(fmaf(__uint_as_float(x[hf][16 * g4 + i]), f[g], -m));
              const float p1 = ex2(fmaf(__uint_as_float(x[hf][16 * g4 + i + 1]), f[g], -m));
              ls[i & 2] += p0;
              ls[(i & 2) + 1] += p1;
              wt[8 * g4 + i / 2] = pack_half2(p0 * up, p1 * up);
            }
          }
          if (masked) {                                    // a page of NaN weighs nothing where it is not seen
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
              const int k = 64 * hf + i;
              const bool z0 = k > left || ((bad >> (k >> 4)) & 1u), z1 = k + 1 > left || ((bad >> (k >> 4)) & 1u);
              wt[i / 2] &= (z0 ? 0u : 0xffffu) | (z1 ? 0u : 0xffff0000u);
            }
          }
          tmem_st32(my + 32 * hf, wt);
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        umma::tmem_st_wait();
        umma::fence_before_sync();
        arrive(p_ready + t);
      }
      if (ok && n > 0) {
        ok = wait_all(o_full + t, 0);
        umma::fence_after_sync();
      }
      if (!ok) l = __int_as_float(0x7fc00000);             // (a wait that ran out: NaN)
      const int64_t slot = part_row8(a, s, seq, h, r) * a.n_splits + blockIdx.z;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (ok && n > 0) {
          umma::tmem_ld32(my + (P::kO + c), o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = ok ? 0u : 0x7fc00000u;
        }
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 y = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
          if (a.n_splits == 1) store_out8(a, s, h, r, c + e, y, m, M, l);
          else *reinterpret_cast<float4*>(a.part + slot * D + c + e) = y;
        }
      }
      if (live && a.n_splits > 1) *reinterpret_cast<float4*>(a.ref + slot * 4) = make_float4(m, M, l, 0.f);
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == 0) umma::tmem_dealloc(tmem, 512);
}

template <int D, int CODE>
int launch(const Attn8Args& a, dim3 grid, cudaStream_t st) {
  auto kernel = paged8_prefill_kernel<D, CODE>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Pf8<D>::kSmem)) != cudaSuccess) return QKV_ELAUNCH;
  kernel<<<grid, 384, Pf8<D>::kSmem, st>>>(a);
  return check_launch();
}

}  // namespace

unsigned int prefill8_timeouts() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_prefill8_timeouts, sizeof(v));
  return v;
}

int launch_prefill8(const Attn8Args& a_in, cudaStream_t st) {
  Attn8Args a = a_in;
  const char* e = getenv("QUASHKV_B200_TEST_DROP_MMA");
  a.test_drop_mma = e && e[0] == '1';
  const dim3 grid(static_cast<unsigned>(a.n_seq) * a.Hkv, a.row_tiles, a.n_splits);
  if (a.p.d == 64) return a.p.code == QKV_E4M3 ? launch<64, p8::kE4M3>(a, grid, st) : launch<64, p8::kInt8>(a, grid, st);
  return a.p.code == QKV_E4M3 ? launch<128, p8::kE4M3>(a, grid, st) : launch<128, p8::kInt8>(a, grid, st);
}

}  // namespace qkv
