// Attention over 4-bit pages (q4.cuh):
//
//   out[r] = sum_j softmax_j(scale q_r . k_j) v_j      over start <= j < len, and with `causal` j <= len - q_len + t
//
// Query row t of sequence b stands at position len[b] - q_len[b] + t, so one rule serves a single token, a chunk and a whole
// prompt whose keys are in the pages already.  A row that sees nothing, and rows t >= q_len[b], are zeros.
//
// First form: a warp per query row.  32 keys at a time: a lane scores a key, the warp shares maximum and sum, and each lane
// adds up D / 32 dims of the output.
#include "common.cuh"
#include "q4.cuh"
#include "sm100_ptx.cuh"

namespace ob {
namespace {

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

template <typename T, int D>
__global__ void __launch_bounds__(128) fmha_q4_kernel(const Args a) {
  constexpr int G = D / 32, W = D / 8;
  __shared__ float sq[4][D];
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (row >= static_cast<int64_t>(a.B) * a.H * a.Tq) return;
  const int64_t b = row / (static_cast<int64_t>(a.H) * a.Tq);
  const int h = static_cast<int>(row / a.Tq % a.H), t = static_cast<int>(row % a.Tq), hk = h / (a.H / a.Hkv);
  const T* q = static_cast<const T*>(a.q) + b * a.qs_b + h * a.qs_h + t * a.qs_t;
  T* out = static_cast<T*>(a.out) + b * a.os_b + h * a.os_h + t * a.os_t;
  const int q_len = a.q_lens ? min(a.q_lens[b], a.Tq) : a.Tq;
  int64_t end = min(static_cast<int64_t>(a.seqlens[b]), a.blocks_per_seq * a.block_size);
  const int64_t start = a.seqstarts ? max(a.seqstarts[b], 0) : 0;
  if (a.causal) end = min(end, static_cast<int64_t>(a.seqlens[b]) - q_len + t + 1);
  if (t >= q_len) end = 0;
  for (int d = lane; d < D; d += 32) sq[warp][d] = Elem<T>::to_f(q[d]);
  __syncwarp();
  float o[G] = {}, m = -INFINITY, l = 0.f;
  for (int64_t j0 = start; j0 < end; j0 += 32) {
    const int64_t j = j0 + lane;
    int64_t base = -1;
    float s = -INFINITY;
    if (j < end) {
      const int64_t page = a.block_table[b * a.blocks_per_seq + j / a.block_size];
      if (page >= 0 && page < a.num_blocks) base = (page * a.Hkv + hk) * a.block_size + j % a.block_size;
    }
    if (base >= 0) {
      s = 0.f;
      for (int w = 0; w < W; ++w) {
        const int oct = q4::octet_of_word(w, G);
        const uint32_t word = a.k_codes[base * W + w];
        const float ks = Elem<T>::to_f(static_cast<const T*>(a.k_scales)[base * G + oct / 4]);
        for (int i = 0; i < 8; ++i) s = fmaf(sq[warp][oct * 8 + i], q4::value_of(word, i, ks), s);
      }
      s *= a.scale_log2;
    }
    const float mn = fmaxf(m, warp_max(s));
    if (mn == -INFINITY) continue;
    const float p = exp2f(s - mn), f = exp2f(m - mn);
    m = mn;
    l = fmaf(l, f, warp_sum(p));
    for (int g = 0; g < G; ++g) o[g] *= f;
    for (int i = 0; i < 32; ++i) {
      const float pi = __shfl_sync(0xffffffffu, p, i);
      const int64_t at = __shfl_sync(0xffffffffu, base, i);
      if (at < 0) continue;
      for (int g = 0; g < G; ++g) {   // dim 32 g + lane
        const uint32_t word = a.v_codes[at * W + q4::word_of_octet(g * 4 + lane / 8, G)];
        o[g] = fmaf(pi, q4::value_of(word, lane % 8, Elem<T>::to_f(static_cast<const T*>(a.v_scales)[at * G + g])), o[g]);
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  for (int g = 0; g < G; ++g) out[g * 32 + lane] = Elem<T>::from_f(o[g] * inv);
}

}  // namespace
}  // namespace ob

extern "C" int oasr_b200_fmha_q4(void* out, const int64_t* out_strides, const void* q, const int64_t* q_strides, const void* k_codes,
                                 const void* k_scales, const void* v_codes, const void* v_scales, const int32_t* block_table,
                                 const int32_t* seqlens, const int32_t* seqstarts, const int32_t* q_lens, int64_t blocks_per_seq,
                                 int64_t block_size, int64_t num_blocks, int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t D,
                                 double scale, int causal, int dtype, void* stream) {
  using namespace ob;
  OB_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && Tq >= 0 && D > 0 && blocks_per_seq >= 0 && num_blocks > 0, OASR_ERR_INVALID, "fmha_q4: bad shape");
  OB_REQUIRE(H % Hkv == 0, OASR_ERR_INVALID, "fmha_q4: H (%lld) must be divisible by H_kv (%lld)", (long long)H, (long long)Hkv);
  OB_REQUIRE(D == 64 || D == 128, OASR_ERR_UNSUPPORTED, "fmha_q4: head_dim %lld is not supported (64 and 128 are)", (long long)D);
  OB_REQUIRE(block_size > 0 && block_size % 16 == 0, OASR_ERR_UNSUPPORTED, "fmha_q4: the block size must be a multiple of 16 (got %lld)",
             (long long)block_size);
  OB_REQUIRE(B <= 65535 && H <= 65535 && Tq <= 0x7fffff && blocks_per_seq * block_size <= 0x7fffffff, OASR_ERR_INVALID,
             "fmha_q4: batch, head count or length too large");
  if (B == 0 || Tq == 0) return OASR_OK;
  OB_REQUIRE(out && out_strides && q && q_strides && k_codes && k_scales && v_codes && v_scales && block_table && seqlens, OASR_ERR_INVALID,
             "fmha_q4: null pointer argument");
  for (int i = 0; i < 3; ++i)
    OB_REQUIRE(out_strides[i] % 8 == 0 && q_strides[i] % 8 == 0, OASR_ERR_ALIGN, "fmha_q4: strides must be multiples of 8 elements");
  OB_REQUIRE(is_aligned(out, 16) && is_aligned(q, 16) && is_aligned(k_codes, 16) && is_aligned(v_codes, 16) && is_aligned(k_scales, 16) &&
                 is_aligned(v_scales, 16),
             OASR_ERR_ALIGN, "fmha_q4: operands must be 16-byte aligned");
  const Args a{out, q, static_cast<const uint32_t*>(k_codes), static_cast<const uint32_t*>(v_codes), k_scales, v_scales, block_table, seqlens,
               seqstarts, q_lens, q_strides[0], q_strides[1], q_strides[2], out_strides[0], out_strides[1], out_strides[2], blocks_per_seq,
               block_size, num_blocks, static_cast<int>(B), static_cast<int>(H), static_cast<int>(Hkv), static_cast<int>(Tq), causal != 0,
               static_cast<float>(scale * 1.4426950408889634)};
  const dim3 grid(static_cast<unsigned>((B * H * Tq + 3) / 4));
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int {
    launch_pdl(D == 64 ? fmha_q4_kernel<T_, 64> : fmha_q4_kernel<T_, 128>, grid, dim3(128), 0, static_cast<cudaStream_t>(stream), a);
    return check_launch("fmha_q4 launch");
  });
}
