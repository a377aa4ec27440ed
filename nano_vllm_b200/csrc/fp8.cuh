// The 8-bit K/V cache: e4m3 codes and one scale for every 16 slots of a block and KV head.
//
// A code c of slot s, head h stands for value(c) * scale[s / 256][h][s % 256 / 16].  Scales that the stores write are powers
// of two: a floating-point code loses nothing by that (the same four significant bits in every binade, 448 / 2^-6 from end to
// end), the quotient x / scale is exact, so that a row is rounded once, by its code, and a group whose scale has to grow is
// coded anew without a second rounding except of values that fall below 2^-6 of the new scale.  Readers take any finite scale from
// 0 on; their results below 2^-126 may be zero.
#pragma once

#include "common.cuh"

namespace nvllm {

constexpr int kScaleGroup = NVLLM_SCALE_GROUP;        // slots that share a scale
constexpr int kGroups = kBlockSize / kScaleGroup;     // scales of a block and head
constexpr int kMinExponent = -64, kMaxExponent = 120;  // of a scale that a store writes: 448 * 2^120 is the first beyond bf16
static_assert(kScaleGroup == 16 && kGroups == 16, "a half warp holds a group's rows or a block's scales");

// Argument checks shared by the entry points that take such a cache.
inline int check_fp8_planes(const char* who, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                            int32_t num_kv_heads, int32_t head_dim, int64_t num_blocks) {
  if (head_dim != 64 && head_dim != 128) return fail(NVLLM_E_GEOMETRY, "%s: head_dim=%d unsupported (64 or 128)", who, head_dim);
  if (num_kv_heads <= 0) return fail(NVLLM_E_GEOMETRY, "%s: Hkv=%d must be positive", who, num_kv_heads);
  if (num_blocks <= 0 || num_blocks > 0x7fffffffLL / kBlockSize)
    return fail(NVLLM_E_GEOMETRY, "%s: num_blocks=%lld must be positive and its slots fit 32 bits", who, (long long)num_blocks);
  if (!k_cache || !v_cache || !k_scale || !v_scale) return fail(NVLLM_E_NULL, "%s: NULL pointer argument", who);
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scale) || !aligned16(v_scale))
    return fail(NVLLM_E_ALIGN, "%s: cache and scale pointers must be 16-byte aligned", who);
  return NVLLM_OK;
}

#ifdef __CUDACC__

// Two values to two codes, `lo` in the low byte: nearest, ties to even, beyond 448 to 448, NaN to 0x7f.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_of_f16x2(uint32_t x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(x));
  return r;
}
// Two codes (the low or the high half of x) to f16, exactly: every e4m3 value is one of f16.
__device__ __forceinline__ uint32_t f16x2_of_low(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_of_high(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float2 float2_of_f16x2(uint32_t x) {
  float2 r;
  asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(x));
  return r;
}

__device__ __forceinline__ uint2 ld_shared8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared8(uint32_t a, const uint2& v) {
  asm volatile("st.shared.v2.u32 [%0], {%1,%2};\n" ::"r"(a), "r"(v.x), "r"(v.y) : "memory");
}

// What sums over V are held in stays between these, whatever the scales: so does its reciprocal, which the build's fast arithmetic
// flushes to zero behind 2^126, as it does subnormal operands.
constexpr float kLargestUnit = 0x1p126f;
// a * b with subnormal operands as they are.
__device__ __forceinline__ float mul_subnormal(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Largest magnitude (as bf16 bits) of two bf16 and `m`, infinities and NaN left out.
__device__ __forceinline__ uint32_t max_finite2(uint32_t m, uint32_t x) {
  x &= 0x7fff7fffu;
  return __vmaxu2(m, x & ~__vcmpgeu2(x, 0x7f807f80u));
}
// The larger of the magnitudes of two bf16, twice; the sign bits are anything.  NaN wins.
__device__ __forceinline__ uint32_t max_magnitude(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Exponent of the smallest scale s that takes a magnitude of these bf16 bits: |x| <= 448 s, 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(uint32_t bf16_bits) {
  const int e = static_cast<int>(bf16_bits >> 7) - 127 - 8 + ((bf16_bits & 0x7fu) > 0x60u);
  return max(kMinExponent, e);
}
// Exponent of a scale read from memory, of the next power of two if it is none.
__device__ __forceinline__ int exponent_of(float scale) {
  const uint32_t b = __float_as_uint(scale);
  return min(kMaxExponent, max(kMinExponent, static_cast<int>(b >> 23 & 255u) - 127 + ((b & 0x7fffffu) != 0)));
}

// Four bf16 over a scale of 1 / inv to four codes; what is not finite becomes NaN (e4m3 has no infinities).
__device__ __forceinline__ uint32_t encode4(const uint2& x, float inv) {
  float y[4] = {__uint_as_float(x.x << 16) * inv, __uint_as_float(x.x & 0xffff0000u) * inv, __uint_as_float(x.y << 16) * inv,
                __uint_as_float(x.y & 0xffff0000u) * inv};
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = fabsf(y[i]) <= 448.f ? y[i] : NAN;
  return e4m3x2(y[0], y[1]) | e4m3x2(y[2], y[3]) << 16;
}
// The same of finite values, inv = 2^-e twice in bf16 (a power of two leaves all bits of a bf16 product).  A magnitude below 2^9
// times 2^-112 has in bf16 the exponent that it has in f16 without, its bits three places further right (subnormal ones too;
// of those f16 has more bits, which only values below 2^-14 have, and they are zeros in e4m3).  The signs go around: this takes
// five instructions of the integer unit for four values, which is what bounds the store; by way of fp32 it were nine.
__device__ __forceinline__ uint32_t encode4_finite(const uint2& x, uint32_t inv) {
  auto code2 = [&](uint32_t v) {
    uint32_t y, z;
    unsigned short c;
    asm("{.reg .b32 m; abs.bf16x2 m, %1; mul.rn.bf16x2 %0, m, %2;}" : "=r"(y) : "r"(v), "r"(inv));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(z) : "r"(y), "r"(0x07800780u));  // 2^-112, twice
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(z * 8));
    return static_cast<uint32_t>(c);
  };
  return __byte_perm(code2(x.x), code2(x.y), 0x5410) | (__byte_perm(x.x, x.y, 0x7531) & 0x80808080u);
}
// Four codes whose scale changes by `ratio` <= 1.
__device__ __forceinline__ uint32_t recode4(uint32_t c, float ratio) {
  const float2 a = float2_of_f16x2(f16x2_of_low(c)), b = float2_of_f16x2(f16x2_of_high(c));
  return e4m3x2(a.x * ratio, a.y * ratio) | e4m3x2(b.x * ratio, b.y * ratio) << 16;
}

#endif  // __CUDACC__
}  // namespace nvllm
