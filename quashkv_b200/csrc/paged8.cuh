// Pages of a KV cache held in 8 bits: what the kernels that fill and read them share.
//
// Codes are e4m3 or int8; both are exact in fp16, so a code becomes an fp16 matrix operand without a rounding.
#pragma once

#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"

namespace qkv {
namespace p8 {

constexpr int kE4M3 = QKV_E4M3, kInt8 = QKV_INT8;

// Largest code, and 2^e of the range around it: a scale is 2^(exponent of the largest magnitude - kTopExp), or the next
// power of two where its mantissa is above that of the largest code (1.75 x 2^8 and 1.984375 x 2^6).
template <int CODE> struct Code;
template <> struct Code<kE4M3> { static constexpr int kTopExp = 8; static constexpr uint32_t kTopMant = 0x600000u; };
template <> struct Code<kInt8> { static constexpr int kTopExp = 6; static constexpr uint32_t kTopMant = 0x7e0000u; };
constexpr int kLeastExp = -120;            // least exponent of a scale: it and its inverse stay normal numbers

// Least power of two s (at least 2^-120) with top <= largest code * s; 0 for top = 0, NaN where top is not finite.
template <int CODE>
__host__ __device__ __forceinline__ float scale_for(float top) {
  union { float f; uint32_t u; } x;
  x.f = top;
  if (top == 0.f) return 0.f;
  if ((x.u & 0x7f800000u) == 0x7f800000u) { x.u = 0x7fc00000u; return x.f; }
  int e = static_cast<int>(x.u >> 23) - 127 - Code<CODE>::kTopExp + ((x.u & 0x7fffffu) > Code<CODE>::kTopMant ? 1 : 0);
  if (e < kLeastExp) e = kLeastExp;
  x.u = static_cast<uint32_t>(e + 127) << 23;
  return x.f;
}

// Slot of position `pos` of a sequence whose row of the block table is `row`: -1 outside the table or in a block with a
// negative number.
__host__ __device__ __forceinline__ int64_t slot_of(const int32_t* row, int max_blocks, int block_size, int64_t pos) {
  if (pos < 0) return -1;
  const int64_t blk = pos / block_size;
  if (blk >= max_blocks) return -1;
  const int64_t id = row[blk];
  return id < 0 ? -1 : id * block_size + pos % block_size;
}

#ifdef __CUDACC__
// Two e4m3 or int8 codes in the low 16 bits of x as a pair of fp16 values.
template <int CODE> __device__ __forceinline__ uint32_t halves_low(uint32_t x);
template <> __device__ __forceinline__ uint32_t halves_low<kE4M3>(uint32_t x) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}\n" : "=r"(d) : "r"(x));
  return d;
}
// int8: a byte u = code + 128 under 0x64 is the fp16 number 1024 + u; 1152 less is the code.  The caller has flipped the
// sign bits (`biased`).
__device__ __forceinline__ uint32_t minus_1152(uint32_t h) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <> __device__ __forceinline__ uint32_t halves_low<kInt8>(uint32_t x) {
  return minus_1152(__byte_perm(x, 0x64646464u, 0x4140));
}
template <int CODE> __device__ __forceinline__ uint32_t halves_high(uint32_t x);
template <> __device__ __forceinline__ uint32_t halves_high<kE4M3>(uint32_t x) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}\n" : "=r"(d) : "r"(x));
  return d;
}
template <> __device__ __forceinline__ uint32_t halves_high<kInt8>(uint32_t x) {
  return minus_1152(__byte_perm(x, 0x64646464u, 0x4342));
}
// A word of four codes as the conversions above want it.
template <int CODE> __device__ __forceinline__ uint32_t biased(uint32_t w) { return CODE == kInt8 ? w ^ 0x80808080u : w; }

// Four values as four codes: rounded to nearest, ties to even, saturating; int8 stays within -127 .. 127.
template <int CODE> __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d);
template <> __device__ __forceinline__ uint32_t encode4<kE4M3>(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}\n" : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
template <> __device__ __forceinline__ uint32_t encode4<kInt8>(float a, float b, float c, float d) {
  // x + 1.5 * 2^23 has the integer nearest to x (ties to even) in its low byte for |x| <= 127
  const float m = 12582912.f;
  const uint32_t lo = __byte_perm(__float_as_uint(a + m), __float_as_uint(b + m), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(c + m), __float_as_uint(d + m), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
template <int CODE> __device__ __forceinline__ float4 decode4(uint32_t w) {
  const uint32_t x = biased<CODE>(w), l = halves_low<CODE>(x), h = halves_high<CODE>(x);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&l)), b = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return make_float4(a.x, a.y, b.x, b.y);
}
#endif

}  // namespace p8

// Allows a kernel `smem` bytes of dynamic shared memory on the current device: once for each device, since the call costs
// as much host time as a launch.
template <auto kernel>
int allow_smem(size_t smem) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (smem <= 48 * 1024) return QKV_OK;
  if (cudaGetDevice(&dev) != cudaSuccess) return QKV_ELAUNCH;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return QKV_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) return QKV_ELAUNCH;
  done.fetch_or(bit, std::memory_order_relaxed);
  return QKV_OK;
}

// What the entry points check of a pool before anything is launched.
inline int check_pages8(const qkv_pages8_t& p) {
  if (!p.k_codes || !p.v_codes || !p.k_scales || !p.v_scales) return QKV_ENULL;
  if (p.code != QKV_E4M3 && p.code != QKV_INT8) return QKV_EDTYPE;
  if ((p.d != 32 && p.d != 64 && p.d != 96 && p.d != 128) || p.Hkv < 1 || p.Hkv > 65535 || p.num_blocks < 1 || p.num_blocks > 0x7fffffffLL ||
      p.block_size < 16 || p.block_size % 16 != 0) return QKV_EDIM;
  if ((reinterpret_cast<uintptr_t>(p.k_codes) | reinterpret_cast<uintptr_t>(p.v_codes)) & 15u) return QKV_EALIGN;
  if ((reinterpret_cast<uintptr_t>(p.k_scales) | reinterpret_cast<uintptr_t>(p.v_scales)) & 3u) return QKV_EALIGN;
  for (int i = 0; i < 3; ++i)
    if (((p.k_stride[i] | p.v_stride[i]) & 15) || p.k_stride[i] < 0 || p.v_stride[i] < 0) return QKV_EALIGN;
  for (int i = 0; i < 2; ++i)
    if (p.ks_stride[i] < 0 || p.vs_stride[i] < 0) return QKV_EARG;
  return QKV_OK;
}

}  // namespace qkv
