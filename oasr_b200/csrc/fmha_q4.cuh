// What the kernels of attention over 4-bit pages share: arguments, and codes as 16-bit operands of the tensor cores.
#pragma once
#include "common.cuh"

namespace ob {
namespace fmha_q4 {

struct Args {
  void* out;
  const void* q;
  const uint32_t *k_codes, *v_codes;
  const void *k_scales, *v_scales;
  const int32_t *block_table, *seqlens, *seqstarts, *q_lens;
  int64_t qs_b, qs_h, qs_t, os_b, os_h, os_t;
  int64_t blocks_per_seq, block_size, num_blocks;
  int B, H, Hkv, Tq, causal;
  float scale_log2;
};

// Attention of long chunks (fmha_q4_prompt.cu): tensor memory, 256 query rows a block.
int run_prompt(const Args& a, int head_dim, int dtype, cudaStream_t stream);

constexpr float kEmpty = -3e38f;   // a maximum below every score: differences to it overflow to -inf or are zero, never NaN

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t bf162_bits(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); }
// two 16-bit values (the low halves or the high halves of two words) as one
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

constexpr uint32_t kLow = 0x000f000fu, kSecond = 0x00f000f0u, kMagic16 = 0x64006400u;   // 1024 in fp16

// (w & mask) | magic in one instruction
__device__ __forceinline__ uint32_t behind(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}

// A code behind a magic exponent (a 4-bit number under the bits of 1024 is 1024 + n, and one subtraction takes 1024 off) is the
// conversion of Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale
// Production" (2022); the constants follow from the formats.
// The codes n - 8 of two keys (one in each half) at bits 0..3 / 4..7, in fp16 and exact: behind an exponent where a step is 1 / 16.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return half2_bits(__hsub2(as_half2(behind(w, kLow, kMagic16)), as_half2(0x64086408u))); }   // (1024 + n) - 1032
__device__ __forceinline__ uint32_t second_codes(uint32_t w) {                                                                                           // (1024 + 16 n) / 16 - 72
  return half2_bits(__hfma2(as_half2(behind(w, kSecond, kMagic16)), as_half2(0x2c002c00u), as_half2(0xd480d480u)));
}

// Codes times scales as operands.  `low` / `second`: the codes of two keys (one in each half) at bits 0..3 / 4..7, times the
// keys' scales; `steep`: what second() wants for the scales.
template <typename T>
struct Op;
template <>
struct Op<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t low(uint32_t w, uint32_t scale) {   // ((128 + n) - 136) s
    const __nv_bfloat162 v = __hsub2(as_bf162(behind(w, kLow, 0x43004300u)), as_bf162(0x43084308u));
    return bf162_bits(__hmul2(v, as_bf162(scale)));
  }
  static __device__ __forceinline__ uint32_t steep(uint32_t scale) { return bf162_bits(__hmul2(as_bf162(scale), as_bf162(0x40804080u))); }   // 4 s: finite
  static __device__ __forceinline__ uint32_t second(uint32_t w, uint32_t steep) {   // (n 2^-129 2^127 - 2) 4 s
    const __nv_bfloat162 v = __hfma2(as_bf162(w & kSecond), as_bf162(0x7f007f00u), as_bf162(0xc000c000u));
    return bf162_bits(__hmul2(v, as_bf162(steep)));
  }
  static __device__ __forceinline__ float low_f(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float high_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return bf162_bits(__floats2bfloat162_rn(lo, hi)); }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Op<__half> {
  static __device__ __forceinline__ uint32_t low(uint32_t w, uint32_t scale) { return half2_bits(__hmul2(as_half2(low_codes(w)), as_half2(scale))); }
  static __device__ __forceinline__ uint32_t steep(uint32_t scale) { return scale; }
  static __device__ __forceinline__ uint32_t second(uint32_t w, uint32_t scale) { return half2_bits(__hmul2(as_half2(second_codes(w)), as_half2(scale))); }
  static __device__ __forceinline__ float low_f(uint32_t w) { return __low2float(as_half2(w)); }
  static __device__ __forceinline__ float high_f(uint32_t w) { return __high2float(as_half2(w)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return half2_bits(__floats2half2_rn(lo, hi)); }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

}  // namespace fmha_q4
}  // namespace ob
