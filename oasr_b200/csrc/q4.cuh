// The 4-bit form of cached keys and values.
//
// A row of D values (one token, one head) is D / 32 groups with a scale each.  The scale is the group's largest magnitude
// over 7, rounded UP to five significant bits, so that codes stay in [-7, 7]; a code has at most three significant bits, so
// code * scale has at most eight and is exact in bf16 and in fp16: every reader, in whatever order it multiplies, works with
// the same values, and a 16-bit operand of the tensor cores holds them without a further rounding.  The coarser scale costs
// at most 1 / 16 of a step (3 % of a step on average).
//
// Order in memory: the row's 32-bit word j holds the eight dims of octet j / G of group j % G (G = D / 32), dim i of the
// octet in bits 4 i .. 4 i + 3 as code + 8.  Four lanes that each take G consecutive words then hold one octet of every
// group, which is what an MMA step over a single group wants.
#pragma once
#include "common.cuh"

namespace ob {
namespace q4 {

template <typename T> struct Limits;
// the largest five-bit scale whose 7-fold is finite, and a floor that keeps the scale a normal, exact five-bit number
template <> struct Limits<__half> { static constexpr float kMin = 0x1p-20f, kMax = 9216.f; };
template <> struct Limits<__nv_bfloat16> { static constexpr float kMin = 0x1p-120f, kMax = 0x1.2p125f; };

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN wins: a group with a NaN gets a NaN scale
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ float scale_of(float amax) {
  if (!(amax == amax)) return amax;
  const uint32_t up = (__float_as_uint(__fdiv_rn(amax, 7.f)) + 0x7FFFFu) & ~0x7FFFFu;
  return fminf(fmaxf(__uint_as_float(up), Limits<T>::kMin), Limits<T>::kMax);
}

// rint(x / scale) of eight values as nibbles, exactly (ties to even), without a division each: the product with an approximate
// reciprocal is within 2^-18 of the quotient, so its rounding is off by one at most, and where it is, or where the quotient lies
// halfway, the remainder x - c scale says so, which is exact (a code and a scale have eight bits together, and it is at most half a
// scale).
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float scale) {
  constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: adding it rounds to whole numbers, ties to even, into the low bits
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
  const int half = __float_as_int(0.5f * scale);
  int c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fmaf(x[i], inv, kMagic);
    const float d = fmaf(kMagic - t, scale, x[i]);
    c[i] = __float_as_int(t) - __float_as_int(kMagic);
    // further than half a step, or exactly half a step from an odd number: the neighbour
    if (fabsf(d) > __int_as_float(half - (c[i] & 1))) c[i] += d < 0.f ? -1 : 1;
  }
  if (!(scale < Limits<T>::kMax)) {      // a scale at its limit: what is beyond saturates (and a NaN scale has some code)
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = min(max(c[i], -7), 7);
  }
  uint32_t w = 0x88888888u;
#pragma unroll
  for (int i = 0; i < 8; ++i) w += static_cast<uint32_t>(c[i]) << (4 * i);
  return w;
}

// word of octet o (dims 8 o .. 8 o + 7), and the octet of word j
__device__ __forceinline__ int word_of_octet(int o, int groups) { return (o & 3) * groups + (o >> 2); }
__device__ __forceinline__ int octet_of_word(int j, int groups) { return (j % groups) * 4 + j / groups; }

}  // namespace q4
}  // namespace ob
