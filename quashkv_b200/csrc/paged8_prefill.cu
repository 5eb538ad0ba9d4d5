// Attention of many query rows over 8-bit pages on the fifth-generation tensor cores: head_dim 64 and 128, queries of 16 bits.
// Formulas as in paged8_attention.cu.
//
// A CTA holds query rows of one (sequence, KV head), a row being a query token and one of the head's query heads, as row
// tiles of 128 (the M of an MMA), and goes over tokens: operands in tiles of 128, scores in tiles of 128 or 64 (below).
//   softmax warps   a thread per query row: scores of a tile from tensor memory, softmax, weights as fp16 in their place
//   one MMA warp    one of its threads issues every MMA: scores of a row tile into tensor memory, and weights (tensor
//                   memory) times V into an accumulator that stays in tensor memory over the whole sequence
//   converters      bring the codes of a tile from their pages (cp.async) and turn them into fp16 operands in the swizzled
//                   order of the tensor core; both K and V as they lie in memory, a row a token: the scores read K with the
//                   inner dimension contiguous, the second product reads V with the outer one contiguous, so nothing is
//                   transposed
// The tensor core works for one row tile while the softmax of the others runs.  Rows hold two whole-number reference
// exponents as in the split kernel, which rise only when a score passes them by 4; only then is the accumulator
// rescaled (exactly), by the row's own thread.
//
// Precision: codes are exact in fp16, 16-bit queries too (scaled by a power of two per row); weights are rounded to
// fp16 once, 2^-11 of each at most: an eighth of what the output's own rounding takes with bf16 queries, and as much as that with fp16
// ones, whose weights the split kernel holds as hi + lo (a second product here).  The sum of weights is fp32 of the unrounded ones.
//
// Bound by the chain of a row tile: its scores, its softmax, its weights times V, none of which can overlap another of
// the same row tile, since scores and weights share their columns.  At head_dim 128 a round of 128 tokens takes about
// 4400 cycles: 2900 of softmax (two warps on a quarter of the SM, whose exponentials alone take 2048) and 1400 of tensor core
// and hand-over.  512 columns of tensor memory are two row tiles of 128 scores and 128 sums.  At head_dim 64 they are
// four of 64 and 64, which lets another row tile's softmax run meanwhile: 130 -> 100 us at 8 x 1024 tokens, 32 heads.
// Measured (causal, bf16, e4m3): 2 x 4096 tokens, 32 heads of 128 over 8: 362-374 us by the box, 735-760 TFLOP/s; 8 x 1024, 32
// heads of 64 over 4: 103 us, 334 TFLOP/s counted over visible pairs.
// Slower at head_dim 128: score tiles of 64 tokens in two buffers each; two threads a row (490 us); rows read twice from
// tensor memory in place of held in registers (470); arithmetic on single numbers in place of pairs (386).
//
// Every wait is bounded; one that runs out is counted (qkv_tensor_core_timeouts) and makes the CTA's rows NaN.
#include <math.h>
#include <stdlib.h>

#include "paged8_attention.cuh"
#include "umma.cuh"

namespace qkv {

namespace {

constexpr int kTok = 128, kRowsT = 128, kStages = 2, kMetaSlots = 4, kGroups = kTok / 16;
// Weights reach 2^15 and the largest is at least 2^9, as in the split kernel: half of fp16's least step is 2^-34 of it, so the many small
// weights of a long cache keep their sum.  (References that rise by 14 and a largest of 1/2 lose weights below 2^-25 of it: 2 x 4096 tokens
// 349 us where this took 362, 8 x 1024 of 64 100 and 101, but weights of 2^-26 beside one came to nothing, however many.)
constexpr float kNone = -3e38f, kSlack = 4.f, kLift = 10.f;
// A score is at most 128 x 448 x 2^14 (below 2^30) times its factor: with factors up to this one they stay below 2^22 and references in fp32
// are exact.  Tiles of larger ones are done with more care (`huge` below).
constexpr float kPlainFactor = 1.f / 256.f;
__device__ unsigned int g_prefill8_timeouts = 0;

struct TileMeta { float ks[kGroups], ex[kGroups], mant[kGroups]; uint32_t bad; float ks_most; uint32_t pad[6]; };   // per group of 16 tokens
static_assert(sizeof(TileMeta) % 16 == 0, "read as 16-byte words");

template <int D> struct Pf8 {
  static constexpr int kQBytes = kRowsT * D * 2, kOpBytes = kTok * D * 2, kRawBytes = kTok * D;
  static constexpr int kUnits = kRawBytes / 512;           // 32 chunks of 16 codes
  // Row tiles, and tokens of a score tile: what 512 columns of tensor memory hold, scores at kSub t and sums at 256 + D t.
  // Four row tiles of 64 tokens keep more softmax warps at work than two of 128, where the sums leave room for them.
  static constexpr int NT = D == 64 ? 4 : 2, kSub = D == 64 ? 64 : 128, kRowsC = NT * kRowsT;
  static constexpr int kConverters = D == 64 ? 3 : 7;      // warps that turn codes into operands
  static constexpr int kSoft = 4 * NT, kThreads = 32 * (kSoft + 1 + kConverters);
  // Registers of a softmax thread and of the others: within what the CTA starts with (640 threads of 96, 512 of 128).
  static constexpr int kSoftRegs = D == 64 ? 104 : 192, kOtherRegs = 64, kStartRegs = D == 64 ? 96 : 128;
  static_assert(32 * (kSoft * kSoftRegs + (1 + kConverters) * kOtherRegs) <= kThreads * kStartRegs, "setmaxnreg would wait for ever");
  static constexpr size_t kSmem = NT * kQBytes + 2 * kStages * kOpBytes + 2 * kRawBytes + kMetaSlots * sizeof(TileMeta) + 256;
  static_assert(kSmem <= 232448, "shared memory of one CTA");
  static constexpr int kO = 256;
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

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {      // and its wait
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
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

// Waits for a phase; a thread that finds it incomplete sleeps until it ends, for at most a millisecond at a time (polling took
// more issue slots than the work).  Gives up after about 0.2 s, or once another wait of the CTA has.
__device__ __forceinline__ bool sleep_on(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
               : "=r"(ok) : "r"(umma::smem_u32(bar)), "r"(parity), "r"(1000000u) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* dead) {
  const long long t0 = clock64();
  while (!*dead) {
    if (sleep_on(bar, parity)) return true;
    if (clock64() - t0 > 400000000LL) {
      *dead = 1;
      atomicAdd(&g_prefill8_timeouts, 1u);
    }
  }
  return false;
}

__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(one));
  return one != 0;
}

// Two fp32 numbers in one register pair.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float2 both(uint64_t x) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(d.x), "=f"(d.y) : "l"(x));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint32_t ex2v(uint32_t x) {      // keeps its place in the order of the source
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(__uint_as_float(x)));
  return __float_as_uint(y);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A ragged batch as one row of tiles: a sequence's first one is its rows' place among all, in tiles, plus its number, which
// leaves each room enough for its own (ceil(b - a) <= floor(b) - floor(a) + 1).
__device__ __forceinline__ int first_tile(const Attn8Args& a, int seq, int rows) {
  const int64_t tok = min(static_cast<int64_t>(max(a.starts[seq], 0)), a.total_q);
  return static_cast<int>(tok * a.G / rows) + seq;
}
// The last sequence whose first tile is not behind `tile` (or 0), by a warp: 32 at a time.
__device__ __forceinline__ int owner_of(const Attn8Args& a, int tile, int rows) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = a.n_seq;
  while (n > 1) {
    const int step = (n + 31) / 32, k = lane * step;
    const uint32_t in = __ballot_sync(QKV_FULL_MASK, k < n && first_tile(a, lo + (k < n ? k : 0), rows) <= tile);
    const int skip = in ? (__popc(in) - 1) * step : 0;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// Where row r of a CTA's (sequence, KV head) lies in the queries or the output, in elements.
__device__ __forceinline__ int64_t row_at(const Attn8Args& a, int64_t row0, const int64_t* stride, int h, int r) {
  const int tok = r / a.G;
  return row0 + tok * stride[1] + (h * a.G + r - tok * a.G) * stride[2];
}

// The 32 query rows of a warp as fp16 operands, each scaled by a power of two (and turned round for a negative scale of the
// scores): D / 8 lanes fetch a row.  Returns the score in base 2 that one unit of a product stands
// for in the lane's own row.
template <int D, bool BF16>
__device__ __forceinline__ float stage_queries(const Attn8Args& a, const Span8& s, int h, int first, int r_end, unsigned char* dst, int row0) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, sub = lane / kLanes, c = lane % kLanes;
  auto values = [](uint32_t x) {
    return BF16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&x));
  };
  // (cp.async, because the little that is left of L1 beside the operands holds up loads that pass through it)
  const int64_t mine = row_at(a, s.q_row0, a.q_stride, h, first + lane < r_end ? first + lane : first);
#pragma unroll 4
  for (int i = 0; i < kLanes; ++i) {
    const int k = kRows * i + sub;
    const int64_t at = __shfl_sync(QKV_FULL_MASK, mine, k);
    cp_async16(dst + umma::sw128_offset(row0 + k, 8 * c, kRowsT), static_cast<const uint16_t*>(a.q) + at + 8 * c, first + k < r_end ? 16 : 0);
  }
  cp_async_commit();
  cp_async_wait<0>();
  // Each step for all rows, so that none waits for the one before.  A thread turns the chunks that it copied.
  float mx[kLanes];
  auto chunk = [&](int i) { return reinterpret_cast<uint4*>(dst + umma::sw128_offset(row0 + kRows * i + sub, 8 * c, kRowsT)); };
#pragma unroll
  for (int i = 0; i < kLanes; ++i) {
    const uint4 w = *chunk(i);
    const float2 v0 = values(w.x), v1 = values(w.y), v2 = values(w.z), v3 = values(w.w);
    mx[i] = max3(max3(fabsf(v0.x), fabsf(v0.y), fabsf(v1.x)), max3(fabsf(v1.y), fabsf(v2.x), fabsf(v2.y)), fmaxf(fabsf(v3.x), fabsf(v3.y)));
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1)
#pragma unroll
    for (int i = 0; i < kLanes; ++i) mx[i] = fmaxf(mx[i], __shfl_xor_sync(QKV_FULL_MASK, mx[i], o));
  float unit = 0.f;
#pragma unroll
  for (int i = 0; i < kLanes; ++i) {
    const float up = scale_to8<13>(mx[i]), sg = a.scale < 0.f ? -up : up;
    const uint4 w = *chunk(i);
    const uint32_t y[4] = {w.x, w.y, w.z, w.w};
    uint32_t x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = values(y[e]);
      x[e] = pack_half2(v.x * sg, v.y * sg);
    }
    *chunk(i) = make_uint4(x[0], x[1], x[2], x[3]);
    const float u = __shfl_sync(QKV_FULL_MASK, up, lane % kRows * kLanes);
    if (lane / kRows == i) unit = fabsf(a.scale) * 1.4426950408889634f * inverse8(u);
  }
  return unit;
}

// PACKED: a ragged batch's tiles behind one another.
template <int D, int CODE, bool PACKED>
__global__ void __launch_bounds__(Pf8<D>::kThreads, 1) paged8_prefill_kernel(Attn8Args a) {
  using P = Pf8<D>;
  extern __shared__ __align__(1024) unsigned char smem[];
  constexpr int NT = P::NT, kSub = P::kSub, kParts = kTok / kSub, kConverters = P::kConverters, kSoft = P::kSoft;
  unsigned char* q_s = smem;                                               // [NT]
  unsigned char* k_s = q_s + NT * P::kQBytes;                               // [kStages]
  unsigned char* v_s = k_s + kStages * P::kOpBytes;                        // [kStages]
  unsigned char* raw_s = v_s + kStages * P::kOpBytes;                      // codes of one K and one V tile
  TileMeta* meta = reinterpret_cast<TileMeta*>(raw_s + 2 * P::kRawBytes);  // [kMetaSlots]
  uint64_t* bars = reinterpret_cast<uint64_t*>(meta + kMetaSlots);
  uint64_t* k_full = bars;                  // [2] every converter thread has stored its part
  uint64_t* v_full = bars + 2;              // [2]
  uint64_t* k_free = bars + 4;              // [2] its MMAs have read it
  uint64_t* v_free = bars + 6;              // [2]
  uint64_t* m_full = bars + 8;              // [4] scales of a tile
  uint64_t* p_ready = bars + 12;            // [NT] queries (phase 0), then weights of score tile i (phase i + 1)
  uint64_t* s_full = p_ready + NT;          // [NT] scores of a row tile; everything issued before has ended, too
  uint64_t* o_full = s_full + NT;           // [NT] all sums
  uint64_t* drain = o_full + NT;
  constexpr int kBars = 13 + 3 * NT;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  const int order = gridDim.y - 1 - blockIdx.y, h = blockIdx.x % a.Hkv;      // long rows first
  const int most = PACKED ? P::kRowsC : a.tile_rows;        // rows of a CTA
  const int seq = PACKED ? owner_of(a, order, P::kRowsC) : blockIdx.x / a.Hkv;
  const Span8 s = span8(a, seq);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int rows = a.G * s.q_len, r0 = (PACKED ? order - first_tile(a, seq, P::kRowsC) : order) * most;
  if ((PACKED && r0 < 0) || r0 >= rows || rows <= a.few_rows) return;
  const int r_end = min(r0 + most, rows), nt = (r_end - r0 + kRowsT - 1) / kRowsT;
  const int64_t seen = visible8(a, s, (r_end - 1) / a.G);
  const int64_t begin = static_cast<int64_t>(blockIdx.z) * a.chunk, stop = min(seen, begin + a.chunk);
  if (begin > 0 && begin >= seen) return;
  const int n_sub = stop > begin ? static_cast<int>((stop - begin + kSub - 1) / kSub) : 0;      // score tiles of kSub tokens
  const int n = (n_sub + kParts - 1) / kParts;                                                // operand tiles of kTok

  if (tid == 0) {
    for (int i = 0; i < kBars; ++i) umma::mbar_init(bars + i, i < 4 ? 32 * kConverters : (i >= 12 && i < 12 + NT ? kRowsT : 1));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    *dead = 0;
  }
  if (warp == 0) umma::tmem_alloc(tmem_slot, 512);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  // (all 512 columns of tensor memory are this CTA's: addresses start at 0)
  auto wait = [&](uint64_t* bar, uint32_t parity) {                        // bounded; false when it, or another one, ran out
    return sleep_on(bar, parity) || wait_on(bar, parity, dead);
  };
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(QKV_FULL_MASK, wait(bar, parity)) != 0; };

  if (warp >= kSoft) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(P::kOtherRegs));
    if (warp == kSoft) {
      // ---- MMAs: the warp goes through this as one, one of its threads issues ----
      constexpr uint32_t id_s = umma::instr_desc(umma::kFmtF16, 128, kSub), id_o = umma::instr_desc(umma::kFmtF16, 128, D) | kOuterB;
      const bool leader = elect_one();
      const uint64_t q_desc = umma::smem_desc_sw128(umma::smem_u32(q_s)), k_desc = umma::smem_desc_sw128(umma::smem_u32(k_s));
      const uint64_t v_desc = smem_desc_outer(umma::smem_u32(v_s), kTok * 128);
      auto scores = [&](int t, int i) {     // score tile i: part i % kParts of operand tile i / kParts
        const int st = (i / kParts) % kStages, part = i % kParts;
        const uint64_t qd = q_desc + t * (P::kQBytes >> 4), kd = k_desc + ((st * P::kOpBytes + part * (kSub * 128)) >> 4);
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma::mma_f16(kSub * t, qd + (((k >> 2) * (kRowsT * 128) + (k & 3) * 32) >> 4), kd + (((k >> 2) * (kTok * 128) + (k & 3) * 32) >> 4), id_s, k != 0);
          umma::commit(s_full + t);
          if (t == nt - 1 && part == kParts - 1) umma::commit(k_free + st);
        }
        __syncwarp();
      };
      auto values = [&](int t, int i) {
        const int st = (i / kParts) % kStages, part = i % kParts;
        const uint64_t vd = v_desc + ((st * P::kOpBytes + part * (kSub * 128)) >> 4);
        if (leader) {
#pragma unroll
          for (int k = 0; k < kSub / 16; ++k)
            umma::mma_f16_ts(P::kO + D * t, kSub * t + 8 * k, vd + (k * 2048 >> 4), id_o, i != 0 || k != 0);
          if (t == nt - 1 && part == kParts - 1) umma::commit(v_free + st);
          if (i + 1 == n_sub) umma::commit(o_full + t);
        }
        __syncwarp();
      };
      bool ok = true;
      for (int t = 0; t < nt && ok; ++t) ok = wait_all(p_ready + t, 0);
      if (n > 0 && ok && (ok = wait_all(k_full, 0))) {
        umma::fence_after_sync();
        for (int t = 0; t < nt; ++t) scores(t, 0);
      }
      for (int i = 0; i < n_sub && ok; ++i) {
        // the operands are there long before the weights
        const int j = i / kParts, j1 = (i + 1) / kParts;
        if (i % kParts == 0) ok = wait_all(v_full + j % kStages, (j / kStages) & 1);
        if (ok && j1 != j && i + 1 < n_sub) ok = wait_all(k_full + j1 % kStages, (j1 / kStages) & 1);
        for (int t = 0; t < nt && ok; ++t) {
          if (!(ok = wait_all(p_ready + t, (i + 1) & 1))) break;
          if (a.test_drop_mma && (blockIdx.x | blockIdx.y | blockIdx.z) == 0 && t == 0 && i == 1) continue;      // test hook
          umma::fence_after_sync();
          values(t, i);
          if (i + 1 < n_sub) scores(t, i + 1);
        }
      }
      if (!ok) {                            // whatever was issued has ended before tensor memory is given back
        if (leader) umma::commit(drain);
        for (int i = 0; i < 400 && !sleep_on(drain, 0); ++i) {}
      }
    } else {
      // ---- codes to operands ----
      // Unit u of a tile (32 chunks of 16 codes): block u / 16 of 64 coordinates, group (u / 2) % 8 of 16 tokens, eight of
      // whose tokens are four lanes' each.  This warp has units w, w + kConverters, ...  A thread converts the chunks that it copied.
      const int w = warp - kSoft - 1, sub = lane >> 2, c = lane & 3;
      constexpr int kMine = (P::kUnits + kConverters - 1) / kConverters;
      const int32_t* row = a.table + seq * a.table_stride;
      const uint32_t to0 = sub * 128 + (((2 * c) ^ sub) << 4), to1 = sub * 128 + (((2 * c + 1) ^ sub) << 4);
      // group `lane` (of the first eight) of tile j: its page and the offset inside it
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
      // The group's first byte: its address is computed once, by one lane, and handed round.
      auto group_at = [&](const uint8_t* codes, const int64_t* stride, int id, int off) -> uint64_t {
        return id < 0 ? 0 : reinterpret_cast<uint64_t>(codes + id * stride[0] + h * stride[1] + off * stride[2]);
      };
      auto issue = [&](uint64_t group, const uint8_t* any, int64_t stride, unsigned char* dst, int j) {
        const int64_t held = s.len - begin - static_cast<int64_t>(j) * kTok;
        const int valid = held < kTok ? static_cast<int>(held) : kTok;
        const uint64_t mine = sub * stride + 16 * c;
        uint64_t at[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) at[i] = __shfl_sync(QKV_FULL_MASK, group, ((w + kConverters * i) >> 1) & 7);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int u = w + kConverters * i;
          if (u < P::kUnits) {
            const bool there = at[i] != 0 && 8 * (u & 15) + sub < valid;
            const uint64_t src = at[i] + mine + ((u & 1) ? 8 * stride : 0) + (u >> 4) * 64;
            cp_async16(dst + u * 512 + lane * 16, there ? reinterpret_cast<const uint8_t*>(src) : any, there ? 16 : 0);      // else zeros
          }
        }
        cp_async_commit();
      };
      auto convert = [&](const unsigned char* src, unsigned char* dst) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int u = w + kConverters * i;
          if (u < P::kUnits) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + u * 512 + lane * 16);
            const uint32_t y[4] = {p8::biased<CODE>(x.x), p8::biased<CODE>(x.y), p8::biased<CODE>(x.z), p8::biased<CODE>(x.w)};
            unsigned char* to = dst + (u >> 4) * (kTok * 128) + (u & 15) * 1024;
            *reinterpret_cast<uint4*>(to + to0) = make_uint4(p8::halves_low<CODE>(y[0]), p8::halves_high<CODE>(y[0]), p8::halves_low<CODE>(y[1]), p8::halves_high<CODE>(y[1]));
            *reinterpret_cast<uint4*>(to + to1) = make_uint4(p8::halves_low<CODE>(y[2]), p8::halves_high<CODE>(y[2]), p8::halves_low<CODE>(y[3]), p8::halves_high<CODE>(y[3]));
          }
        }
        umma::fence_smem_to_async();
      };
      auto scale_of = [&](const float* sc, const int64_t* stride, int id) { return id < 0 ? 0.f : sc[id * stride[0] + h * stride[1]]; };
      unsigned char* raw_k = raw_s;
      unsigned char* raw_v = raw_s + P::kRawBytes;
      int id = n > 0 ? page_of(0) : -1, id1 = n > 1 ? page_of(1) : -1;
      if (n > 0) {
        issue(group_at(a.p.k_codes, a.p.k_stride, id, offset_of(0)), a.p.k_codes, a.p.k_stride[2], raw_k, 0);
        issue(group_at(a.p.v_codes, a.p.v_stride, id, offset_of(0)), a.p.v_codes, a.p.v_stride[2], raw_v, 0);
      }
      float ks = scale_of(a.p.k_scales, a.p.ks_stride, id), vs = scale_of(a.p.v_scales, a.p.vs_stride, id);
      for (int j = 0; j < n; ++j) {
        const int st = j % kStages;
        const uint32_t par = ((j / kStages) & 1) ^ 1;
        const int id2 = j + 2 < n ? page_of(j + 2) : -1, off1 = offset_of(j + 1);
        const uint64_t k1 = group_at(a.p.k_codes, a.p.k_stride, id1, off1), v1 = group_at(a.p.v_codes, a.p.v_stride, id1, off1);
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
          const uint32_t most = __reduce_max_sync(QKV_FULL_MASK, lane < kGroups && ks == ks ? __float_as_uint(ks) : 0u);      // (0 or more)
          if (lane == 0) { mt->bad = bad; mt->ks_most = __uint_as_float(most); }
          __syncwarp();
          if (lane == 0) arrive(m_full + j % kMetaSlots);
        }
        convert(raw_k, k_s + st * P::kOpBytes);
        arrive(k_full + st);
        if (j + 1 < n) issue(k1, a.p.k_codes, a.p.k_stride[2], raw_k, j + 1); else cp_async_commit();
        ks = scale_of(a.p.k_scales, a.p.ks_stride, id1);
        vs = scale_of(a.p.v_scales, a.p.vs_stride, id1);
        cp_async_wait<1>();                                // this thread's chunks of V
        if (j >= kStages && !wait_all(v_free + st, par)) break;
        convert(raw_v, v_s + st * P::kOpBytes);
        arrive(v_full + st);
        if (j + 1 < n) issue(v1, a.p.v_codes, a.p.v_stride[2], raw_v, j + 1); else cp_async_commit();
        id = id1;
        id1 = id2;
      }
      cp_async_wait<0>();
    }
  } else {
    // ---- a query row per thread ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(P::kSoftRegs));
    const int t = warp >> 2, r = r0 + tid;
    if (t < nt) {
      const bool live = r < r_end;
      const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16, my = kSub * t + lanes, sums = P::kO + D * t + lanes;
      float unit;
      {
        const int row0 = 32 * (warp & 3), first = r0 + t * kRowsT + row0;
        unit = a.dtype == QKV_BF16 ? stage_queries<D, true>(a, s, h, first, r_end, q_s + t * P::kQBytes, row0)
                                   : stage_queries<D, false>(a, s, h, first, r_end, q_s + t * P::kQBytes, row0);
        umma::fence_smem_to_async();
        arrive(p_ready + t);
        // An infinity among the queries (2^115 is beyond what any number gives): the row is NaN in any case, and not `huge`.
        if (unit > fabsf(a.scale) * (1.4426950408889634f * 0x1.8p114f)) unit = 0.f;
      }
      // last token that this row sees, relative to `begin`
      const int lim = live ? static_cast<int>(max(min(visible8(a, s, r / a.G) - begin, a.chunk), static_cast<int64_t>(0))) - 1 : -1;
      float m = kNone, M = 0.5f * kNone, l = 0.f;
      // From the row's first tile on whose scores may be far from 0: products are rounded before a reference
      // is taken from them, so that none passes it, and M is held as M - m, which stays exact where m + 1 is no number any more.
      bool ok = true, huge = false;
      constexpr int kG = kSub / 16;
      for (int i = 0; i < n_sub; ++i) {
        const int j = i / kParts, g0 = i % kParts * kG;    // groups g0 .. of operand tile j
        if (i % kParts == 0 && !(ok = wait_all(m_full + j % kMetaSlots, (j / kMetaSlots) & 1))) break;
        // factors of the scores, and of the weights as long as the references stay: while the scores come about
        const TileMeta& mt = meta[j % kMetaSlots];
        float f[kG], ex[kG], up[kG];
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          f[g] = mt.ks[g0 + g] * unit;
          ex[g] = mt.ex[g0 + g];
        }
        auto factors = [&] {
#pragma unroll
          for (int g = 0; g < kG; ++g) up[g] = mt.mant[g0 + g] * ex2(fminf((huge ? 0.f : m) + ex[g] - M, 120.f));
        };
        if (!huge && mt.ks_most * unit > kPlainFactor) {
          huge = true;
          M -= m;
        }
        factors();
        const uint32_t bad = (mt.bad >> g0) & ((1u << kG) - 1u);
        if (!(ok = wait_all(s_full + t, i & 1))) break;
        umma::fence_after_sync();
        uint32_t x[kSub / 64][64];
        const int left = lim - i * kSub;                   // tokens 0 .. left of the tile are visible
        const bool masked = __any_sync(QKV_FULL_MASK, left < kSub - 1 || huge) || bad != 0;
#pragma unroll
        for (int hf = 0; hf < kSub / 64; ++hf) umma::tmem_ld64_issue(my + 64 * hf, x[hf]);
#pragma unroll
        for (int hf = 0; hf < kSub / 64; ++hf) umma::tmem_ld64_wait(x[hf]);
        float tm = -INFINITY, tM = -INFINITY;
        if (masked) {
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int k = 16 * g + e;
              uint32_t& y = x[k >> 6][k & 63];
              const float v = (k > left || ((bad >> g) & 1u)) ? -INFINITY : __uint_as_float(y) * f[g];
              y = __float_as_uint(v);
              top = fmaxf(top, v);
            }
            tm = fmaxf(tm, top);
            tM = fmaxf(tM, top + ex[g]);
            f[g] = 1.f;
            if (huge) up[g] = top;                         // (factors come anew below)
          }
        } else {
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            auto at = [&](int e) { return __uint_as_float(x[(16 * g + e) >> 6][(16 * g + e) & 63]); };
            float top[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e] = max3(at(3 * e), at(3 * e + 1), at(3 * e + 2));
            const float v = max3(max3(top[0], top[1], top[2]), max3(top[3], at(12), at(13)), fmaxf(at(14), at(15))) * f[g];
            tm = fmaxf(tm, v);
            tM = fmaxf(tM, v + ex[g]);
          }
        }
        const bool rise = tm > m + kSlack || tM > M + (kLift + kSlack) || huge;
        if (__any_sync(QKV_FULL_MASK, rise)) {     // scores of this tile are there, so the sums of the one before are
          const float m1 = fmaxf(m, ceilf(tm));
          if (huge) {
            M += m - m1;
            tM = -INFINITY;
#pragma unroll
            for (int g = 0; g < kG; ++g) tM = fmaxf(tM, up[g] - m1 + ex[g]);
          }
          const float M1 = fmaxf(M, ceilf(tM) - kLift);
          l *= ex2(m - m1);
          const float alpha = ex2(M - M1);
          m = m1;
          M = M1;
          factors();
          if (i > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld16(sums + c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              umma::tmem_st16(sums + c, o);
            }
          }
        }
        // Sixteen tokens at a time in three steps (argument, exponential, product and rounding), one step apart, so that the
        // exponentials, of which a scheduler starts one in eight cycles, have the other steps' instructions between them.
        uint64_t ls[2] = {0, 0};
        const uint64_t low = pair(-m, -m);
        uint32_t wt[32];
        auto el = [&](int k) -> uint32_t& { return x[k >> 6][k & 63]; };
        auto argument = [&](int k) {
          const float fg = f[k >> 4];
          const float2 e = both(fma2(pair(__uint_as_float(el(k)), __uint_as_float(el(k + 1))), pair(fg, fg), low));
          el(k) = __float_as_uint(e.x);
          el(k + 1) = __float_as_uint(e.y);
        };
        auto weigh = [&](int k) {
          const float u = up[k >> 4];
          const uint64_t p = pair(__uint_as_float(el(k)), __uint_as_float(el(k + 1)));
          ls[(k >> 1) & 1] = add2(ls[(k >> 1) & 1], p);
          const float2 w = both(mul2(p, pair(u, u)));
          wt[(k & 63) >> 1] = pack_half2(w.x, w.y);
        };
        auto store = [&](int hf) {
          if (masked) {                                    // a page of NaN weighs nothing where it is not seen
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
              const int k = 64 * hf + i;
              const bool gone = (bad >> (k >> 4)) & 1u;
              wt[i / 2] &= (k > left || gone ? 0u : 0xffffu) | (k + 1 > left || gone ? 0u : 0xffff0000u);
            }
          }
          tmem_st32(my + 32 * hf, wt);
        };
#pragma unroll
        for (int e = 0; e < 16; e += 2) argument(e);
#pragma unroll
        for (int g = 0; g <= kG; ++g) {
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            if (g < kG) el(16 * g + e) = ex2v(el(16 * g + e));
            if (g + 1 < kG) argument(16 * (g + 1) + e);
            if (g < kG) el(16 * g + e + 1) = ex2v(el(16 * g + e + 1));
            if (g > 0) weigh(16 * (g - 1) + e);
          }
          if (g == 4) store(0);
          if (g == 8) store(1);
        }
        const float2 l2 = both(add2(ls[0], ls[1]));
        l += l2.x + l2.y;
        umma::tmem_st_wait();
        umma::fence_before_sync();
        arrive(p_ready + t);
      }
      if (ok && n_sub > 0) {
        ok = wait_all(o_full + t, 0);
        umma::fence_after_sync();
      }
      if (!ok) l = __int_as_float(0x7fc00000);             // (a wait that ran out: NaN)
      // Rows leave through the place of the queries, so that D / 8 lanes write a row.  At D = 128 a warp's place there holds
      // rows of other warps' queries, too: only behind o_full, which every product that reads them and so every warp's
      // queries are in front of.  Where nothing was summed, or a wait ran out, a thread writes its row by itself.
      const int64_t slot = part_row8(a, s, seq, h, live ? r : 0) * a.n_splits + blockIdx.z;
      const float dM = huge ? M : M - m;
      const Unit8 by = unit8(dM, l);                       // a row that has seen nothing is zeros
      unsigned char* rows_s = q_s + t * P::kQBytes + 32 * (warp & 3) * (2 * D);
      const bool summed = ok && n_sub > 0;                 // (the same for all of a warp)
      if (!summed && a.n_splits == 1 && live) {
        uint4* at = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row_at(a, s.o_row0, a.o_stride, h, r));
        const uint32_t x = ok ? 0u : 0x7fff7fffu;          // (NaN in both types)
#pragma unroll 1
        for (int c = 0; c < D / 8; ++c) at[c] = make_uint4(x, x, x, x);
      }
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (summed) {
          umma::tmem_ld32(sums + c, o);
        } else if (a.n_splits == 1) {
          break;
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = ok ? 0u : 0x7fc00000u;
        }
        if (a.n_splits > 1) {
          if (!live) continue;
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(a.part + slot * D + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          continue;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float v0 = __uint_as_float(o[e + 2 * k]) * by.x * by.y, v1 = __uint_as_float(o[e + 2 * k + 1]) * by.x * by.y;
            const __nv_bfloat162 z = __floats2bfloat162_rn(v0, v1);
            y[k] = a.dtype == QKV_BF16 ? *reinterpret_cast<const uint32_t*>(&z) : pack_half2(v0, v1);
          }
          *reinterpret_cast<uint4*>(rows_s + lane * (2 * D) + ((((c + e) >> 3) ^ (lane & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
      if (summed && a.n_splits == 1) {
        constexpr int kLanes = D / 8, kRows = 32 / kLanes;
        const int64_t mine = row_at(a, s.o_row0, a.o_stride, h, live ? r : r0);
        __syncwarp();
#pragma unroll 8
        for (int i = 0; i < kLanes; ++i) {
          const int k = kRows * i + lane / kLanes, c = lane % kLanes;
          const int64_t at = __shfl_sync(QKV_FULL_MASK, mine, k);
          const uint4 y = *reinterpret_cast<const uint4*>(rows_s + k * (2 * D) + ((c ^ (k & 7)) << 4));
          if (r - lane + k < r_end) *(reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) + c) = y;
        }
      }
      if (live && a.n_splits > 1) *reinterpret_cast<float4*>(a.ref + slot * 4) = make_float4(m, dM, l, 0.f);
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == 0) umma::tmem_dealloc(*tmem_slot, 512);
}

template <int D, int CODE, bool PACKED>
int launch_as_is(const Attn8Args& a, dim3 grid, cudaStream_t st) {
  constexpr auto kernel = paged8_prefill_kernel<D, CODE, PACKED>;
  if (const int rc = allow_smem<kernel>(Pf8<D>::kSmem)) return rc;
  kernel<<<grid, Pf8<D>::kThreads, Pf8<D>::kSmem, st>>>(a);
  return check_launch();
}
template <int D, int CODE>
int launch(const Attn8Args& a, dim3 grid, bool packed, cudaStream_t st) {
  return packed ? launch_as_is<D, CODE, true>(a, grid, st) : launch_as_is<D, CODE, false>(a, grid, st);
}

}  // namespace

unsigned int prefill8_timeouts() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_prefill8_timeouts, sizeof(v));
  return v;
}

int prefill8_rows(int d) { return d == 64 ? Pf8<64>::kRowsC : Pf8<128>::kRowsC; }

int launch_prefill8(const Attn8Args& a_in, cudaStream_t st) {
  Attn8Args a = a_in;
  const char* e = getenv("QUASHKV_B200_TEST_DROP_MMA");
  a.test_drop_mma = e && e[0] == '1';
  // A ragged batch is one row of tiles where that is fewer than the most rows for each sequence, whose CTAs have mostly nothing.
  const int64_t tiles = a.total_q * a.G / a.tile_rows + a.n_seq;
  const bool packed = a.starts && tiles < static_cast<int64_t>(a.n_seq) * a.row_tiles && tiles <= 65535;
  const dim3 grid(static_cast<unsigned>(packed ? 1 : a.n_seq) * a.Hkv, static_cast<unsigned>(packed ? tiles : a.row_tiles), a.n_splits);
  if (a.p.d == 64) return a.p.code == QKV_E4M3 ? launch<64, p8::kE4M3>(a, grid, packed, st) : launch<64, p8::kInt8>(a, grid, packed, st);
  return a.p.code == QKV_E4M3 ? launch<128, p8::kE4M3>(a, grid, packed, st) : launch<128, p8::kInt8>(a, grid, packed, st);
}

}  // namespace qkv
