// Norms of queries and keys for each head with the position rotation, and the same on the way into the paged cache.
//
//   n(x) = x * rsqrt(mean(x^2) + eps) * w                         per head row, skipped without a weight
//   y_a  = x_a cos - x_b sin,  y_b = x_b cos + x_a sin            pairs (a, b) of the first R dims: (i, i + R / 2), or (2 i, 2 i + 1)
//
// cos | sin come from an fp32 table row per position.  All arithmetic is fp32; on the way to 4-bit codes the products and sums of
// the rotation are rounded one by one (no contraction), so that a code is a matter of the formula alone.
//
// A lane owns a unit of 16 dims: the two octets whose dims pair up (u and u + R / 16), or two neighbouring octets where pairs
// are neighbours or nothing is rotated.  So a lane reads what it writes and nothing else (rows may be turned in place), and the
// row sum is a shuffle over D / 16 lanes.  Tokens are the fast index of the grid, so that the lanes of a warp have one kind of row
// (queries, keys, values); heads as the fast index took 96 instead of 87 us for the case below.  No load waits for another but the
// position table's for the position.
//
// Everything is read once and written once.  B200: 16384 tokens, 32 + 8 heads of 128, norms and rotation, 75 us (344 MB, 4.6 TB/s, 0.70 of
// the copy rate; 0.61 of the issue slots); 20016 frames of 48 heads of 128 of which half are padding, into 4-bit pages, 106 us, bound by
// instructions (0.76 of the issue slots: an exact code costs some 15); calls of a few tokens by their launch.
#include "common.cuh"
#include "fmha_q4.cuh"
#include "q4.cuh"
#include "sm100_ptx.cuh"

namespace ob {
namespace {

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    const Pack<T> v = ld128(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f(v.v[i]);
  } else {
    const Pack<T> v = ld128(p), w = ld128(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v.v[i], x[4 + i] = w.v[i];
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    Pack<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.v[i] = Elem<T>::from_f(x[i]);
    st128(p, v);
  } else {
    Pack<T> v, w;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.v[i] = x[i], w.v[i] = x[4 + i];
    st128(p, v);
    st128(p + 4, w);
  }
}

// The two octets of unit u; `units` of them are rotated.
template <bool kInter>
__device__ __forceinline__ int2 unit_octets(int u, int rotated) {
  return (!kInter && u < rotated) ? make_int2(u, u + rotated) : make_int2(2 * u, 2 * u + 1);
}

struct Turn {
  float c[8], s[8];
};

__device__ __forceinline__ Turn load_turn(const float* row, int half, int u) {
  Turn t;
  load8(row + u * 8, t.c);
  load8(row + half + u * 8, t.s);
  return t;
}

template <bool kInter, bool kRounded>
__device__ __forceinline__ void rotate(float (&a)[8], float (&b)[8], const Turn& t) {
  auto turn = [](float& x, float& y, float c, float s) {
    const float nx = kRounded ? __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)) : fmaf(x, c, -y * s);
    y = kRounded ? __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s)) : fmaf(y, c, x * s);
    x = nx;
  };
  if constexpr (kInter) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      turn(a[2 * i], a[2 * i + 1], t.c[i], t.s[i]);
      turn(b[2 * i], b[2 * i + 1], t.c[4 + i], t.s[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(a[i], b[i], t.c[i], t.s[i]);
  }
}

// The two octets of a lane in a row, as loaded.
template <typename T>
struct Unit {
  static constexpr int kPacks = 8 / Elem<T>::kVec;
  Pack<T> a[kPacks], b[kPacks];
  __device__ __forceinline__ void load(const T* row, int2 oct) {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) a[i] = ld128(row + oct.x * 8 + i * Elem<T>::kVec), b[i] = ld128(row + oct.y * 8 + i * Elem<T>::kVec);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) *reinterpret_cast<uint4*>(&a[i]) = *reinterpret_cast<uint4*>(&b[i]) = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void values(float (&xa)[8], float (&xb)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      xa[i] = Elem<T>::to_f(a[i / Elem<T>::kVec].v[i % Elem<T>::kVec]);
      xb[i] = Elem<T>::to_f(b[i / Elem<T>::kVec].v[i % Elem<T>::kVec]);
    }
  }
};

// x * rsqrt(mean(x^2) + eps) * w over the `lanes` lanes of a row; every lane of the warp calls it, idle ones with zeros, and rows
// that are not normed (a NaN weight does not reach a row that has no position) with `on` false.
template <typename T>
__device__ __forceinline__ void norm_row(float (&a)[8], float (&b)[8], const Unit<T>& w, bool on, int lanes, float inv_d, float eps) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
  for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (!on) return;
  const float r = rsqrtf(fmaf(sum, inv_d, eps));
  float wa[8], wb[8];
  w.values(wa, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = a[i] * r * wa[i], b[i] = b[i] * r * wb[i];
}

struct QkArgs {
  void *q_out, *k_out;
  const void *q, *k, *q_weight, *k_weight;
  const float* table;
  const void* positions;
  int64_t table_rows, tokens, qs_n, qs_h, ks_n, ks_h, qo_n, qo_h, ko_n, ko_h;
  int half, heads, kv_heads, q_chunks, units, lanes, lane_shift, pos_i64;
  float inv_d, eps;
};

// A lane takes one head, or two neighbouring ones (HB) that share weights, cosines and sines.
template <typename T, bool kInter, int HB>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : HB == 1 ? 4 : 3) qk_norm_rope_kernel(const QkArgs a) {
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const uint32_t group = static_cast<uint32_t>((static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> a.lane_shift);   // fewer than 2^31
  const int u = threadIdx.x & (a.lanes - 1);
  const uint32_t tokens = static_cast<uint32_t>(a.tokens), at32 = group / tokens;
  const int64_t n = group - at32 * tokens;
  const int at = static_cast<int>(at32);
  const bool is_q = at < a.q_chunks;
  const int head = (is_q ? at : at - a.q_chunks) * HB;
  const int heads = u < a.units ? (is_q ? a.heads : a.kv_heads) - head : 0;   // <= 0: an idle lane
  const int rotated = a.half / 8;
  const int2 oct = unit_octets<kInter>(u, rotated);
  const T* weight = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
  const int64_t in_stride = is_q ? a.qs_h : a.ks_h, out_stride = is_q ? a.qo_h : a.ko_h;
  const T* src = (is_q ? static_cast<const T*>(a.q) + n * a.qs_n : static_cast<const T*>(a.k) + n * a.ks_n) + head * in_stride;
  T* dst = (is_q ? static_cast<T*>(a.q_out) + n * a.qo_n : static_cast<T*>(a.k_out) + n * a.ko_n) + head * out_stride;
  Unit<T> x[HB], w;
  int64_t pos = -1;
  if (heads > 0) pos = a.pos_i64 ? static_cast<const int64_t*>(a.positions)[n] : static_cast<const int32_t*>(a.positions)[n];
#pragma unroll
  for (int i = 0; i < HB; ++i) {   // none of these waits for the position
    x[i].zero();
    if (i < heads) x[i].load(src + i * in_stride, oct);
  }
  if (weight && heads > 0) w.load(weight, oct);
  const bool known = pos >= 0 && pos < a.table_rows;
  const bool turned = known && u < rotated;
  Turn t;
  if (turned) t = load_turn(a.table + pos * 2 * a.half, a.half, u);
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    float xa[8], xb[8];
    x[i].values(xa, xb);
    if (a.q_weight || a.k_weight) norm_row<T>(xa, xb, w, weight, a.lanes, a.inv_d, a.eps);
    if (turned) rotate<kInter, false>(xa, xb, t);
    if (!known) {                  // no such position: a zero row
#pragma unroll
      for (int j = 0; j < 8; ++j) xa[j] = xb[j] = 0.f;
    }
    if (i < heads) {
      store8(dst + i * out_stride + oct.x * 8, xa);
      store8(dst + i * out_stride + oct.y * 8, xb);
    }
  }
}

struct WriteArgs {
  void *q_out, *k_pool, *v_pool;       // pools: 16-bit rows, or codes
  void *k_scales, *v_scales;           // 4-bit pools only
  const void *q, *k, *v, *q_weight, *k_weight;
  const float* table;
  const int32_t *block_table, *offsets, *rope_offsets, *new_lens;
  int64_t table_rows, B, T, qs_b, qs_h, qs_t, ks_b, ks_h, ks_t, vs_b, vs_h, vs_t, qo_b, qo_h, qo_t;
  int64_t blocks_per_seq, block_size, num_blocks;
  int half, heads, kv_heads, units, lanes, lane_shift, groups;
  float inv_d, eps;
};

// Largest magnitudes of the groups that a lane's two octets lie in.  The rows of a warp may be of different kinds (`pairs`: of
// values, whose groups are always two lanes), and a shuffle names the whole warp: every branch here goes the same way in all of its
// lanes, and lanes choose among the results afterwards.
template <bool kInter>
__device__ __forceinline__ float2 group_max(float ma, float mb, int2 oct, int u, int rotated, int lanes, bool pairs) {
  const float both = q4::max_nan(ma, mb), pair = q4::max_nan(both, __shfl_xor_sync(0xffffffffu, both, 1));
  if (kInter || __all_sync(0xffffffffu, pairs)) return make_float2(pair, pair);   // neighbouring octets: a group is two lanes
  if (rotated % 4 == 0) {                                 // octets u and u + rotated: each in a group of four lanes
    ma = q4::max_nan(ma, __shfl_xor_sync(0xffffffffu, ma, 1));
    mb = q4::max_nan(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
    ma = q4::max_nan(ma, __shfl_xor_sync(0xffffffffu, ma, 2));
    mb = q4::max_nan(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
    return !pairs && u < rotated ? make_float2(ma, mb) : make_float2(pair, pair);
  }
  float r[2];                                             // a group holds octets of both kinds: ask each octet's lane
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int first = (s ? oct.y : oct.x) & ~3;
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = first + j;
      const bool split = o < 2 * rotated;
      const int lane = split ? (o < rotated ? o : o - rotated) : o >> 1;
      const bool slot_b = split ? o >= rotated : (o & 1);
      const float va = __shfl_sync(0xffffffffu, ma, lane, lanes), vb = __shfl_sync(0xffffffffu, mb, lane, lanes);
      m = q4::max_nan(m, slot_b ? vb : va);
    }
    r[s] = m;
  }
  return pairs ? make_float2(pair, pair) : make_float2(r[0], r[1]);
}

__device__ __forceinline__ float octet_max(const float (&x)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = q4::max_nan(m, fabsf(x[i]));
  return m;
}

template <typename T>
__device__ __forceinline__ void store_q4(uint32_t* codes, T* scales, const float (&x)[8], int o, float amax, int groups) {
  const float s = q4::scale_of<T>(amax);
  codes[q4::word_of_octet(o, groups)] = q4::codes_of<T>(x, s);
  if ((o & 3) == 0) scales[o >> 2] = Elem<T>::from_f(s);
}

// Head rows of one frame: the queries' (into q_out), then the keys' and the values' (into their page).
template <typename T, bool kInter, bool kQ4>
__global__ void __launch_bounds__(256, 4) write_kv_rope_kernel(const WriteArgs a) {
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const uint32_t group = static_cast<uint32_t>((static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> a.lane_shift);   // fewer than 2^31
  const int u = threadIdx.x & (a.lanes - 1);
  const uint32_t frames = static_cast<uint32_t>(a.B * a.T), index32 = group / frames, frame = group - index32 * frames, T32 = static_cast<uint32_t>(a.T);
  const int64_t b = frame / T32, t = frame - static_cast<uint32_t>(b) * T32;
  const int index = static_cast<int>(index32);
  const int kind = index < a.heads ? 0 : index < a.heads + a.kv_heads ? 1 : 2;
  const int head = index - (kind > 0 ? a.heads : 0) - (kind > 1 ? a.kv_heads : 0);
  const bool mine = index < a.heads + 2 * a.kv_heads && u < a.units;
  const int rotated = a.half / 8;
  const int2 oct = kind == 2 ? make_int2(2 * u, 2 * u + 1) : unit_octets<kInter>(u, rotated);   // values are not rotated
  const T* weight = static_cast<const T*>(kind == 0 ? a.q_weight : kind == 1 ? a.k_weight : nullptr);
  Unit<T> x, w;
  x.zero();
  bool fresh = false, known = false;
  int64_t page = -1, slot = 0, pos = 0;
  if (mine) {
    fresh = !a.new_lens || t < a.new_lens[b];
    if (fresh) {   // not waiting for the page or the position
      x.load(kind == 0   ? static_cast<const T*>(a.q) + b * a.qs_b + head * a.qs_h + t * a.qs_t
             : kind == 1 ? static_cast<const T*>(a.k) + b * a.ks_b + head * a.ks_h + t * a.ks_t
                         : static_cast<const T*>(a.v) + b * a.vs_b + head * a.vs_h + t * a.vs_t,
             oct);
      if (weight) w.load(weight, oct);
    }
    const int64_t at = static_cast<int64_t>(a.offsets[b]) + t;
    pos = a.rope_offsets ? static_cast<int64_t>(a.rope_offsets[b]) + t : at;
    known = fresh && pos >= 0 && pos < a.table_rows;
    if (fresh && at >= 0) {                             // below 2^32
      const uint32_t size = static_cast<uint32_t>(a.block_size), logical = static_cast<uint32_t>(at) / size;
      slot = static_cast<uint32_t>(at) - logical * size;
      if (logical < a.blocks_per_seq) page = a.block_table[b * a.blocks_per_seq + logical];
    }
    if (page >= a.num_blocks) page = -1;                // outside the table or the pool: dropped, never written
  }
  const bool turned = known && kind != 2 && u < rotated;
  Turn tn;
  if (turned) tn = load_turn(a.table + pos * 2 * a.half, a.half, u);
  float xa[8], xb[8];
  x.values(xa, xb);
  if (a.q_weight || a.k_weight) norm_row<T>(xa, xb, w, weight && fresh, a.lanes, a.inv_d, a.eps);
  if (turned) {
    if (kQ4 && kind == 1) rotate<kInter, true>(xa, xb, tn);
    else rotate<kInter, false>(xa, xb, tn);
  }
  if (!known && kind != 2) {   // no such position: a zero query or key
#pragma unroll
    for (int i = 0; i < 8; ++i) xa[i] = xb[i] = 0.f;
  }
  float2 gmax = make_float2(0.f, 0.f);
  if (kQ4 && __any_sync(0xffffffffu, kind != 0)) gmax = group_max<kInter>(octet_max(xa), octet_max(xb), oct, u, rotated, a.lanes, kind == 2);
  if (!mine) return;
  const int dims = a.units * 16;
  if (kind == 0) {
    T* dst = static_cast<T*>(a.q_out) + b * a.qo_b + head * a.qo_h + t * a.qo_t;
    store8(dst + oct.x * 8, xa);
    store8(dst + oct.y * 8, xb);
  } else if (page >= 0) {
    if constexpr (kQ4) {
      const int64_t row = (page * a.kv_heads + head) * a.block_size + slot;
      uint32_t* codes = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(kind == 1 ? a.k_pool : a.v_pool) + row * (dims / 2));
      T* scales = static_cast<T*>(kind == 1 ? a.k_scales : a.v_scales) + row * a.groups;
      store_q4<T>(codes, scales, xa, oct.x, gmax.x, a.groups);
      store_q4<T>(codes, scales, xb, oct.y, gmax.y, a.groups);
    } else {
      const int64_t row = (page * a.block_size + slot) * a.kv_heads + head;
      T* dst = static_cast<T*>(kind == 1 ? a.k_pool : a.v_pool) + row * dims;
      store8(dst + oct.x * 8, xa);
      store8(dst + oct.y * 8, xb);
    }
  }
}

struct GatherArgs {
  void *k_out, *v_out;
  const uint32_t *k_codes, *v_codes;
  const void *k_scales, *v_scales;
  const int32_t *block_table, *starts;
  int64_t B, Hkv, T, blocks_per_seq, block_size, num_blocks;
  int words, groups, rows, span;
  uint32_t chunks;
};

// The eight values of a word in order; each is one product in T, rounded once where the scale has more than its five bits.
template <typename T>
__device__ __forceinline__ uint4 values_of(uint32_t w, uint32_t scale) {
  using Op = fmha_q4::Op<T>;
  const uint32_t s2 = scale | (scale << 16), s4 = Op::steep(s2), h = w >> 8;
  const uint32_t a = Op::low(w, s2), b = Op::second(w, s4), c = Op::low(h, s2), d = Op::second(h, s4);   // dims (0, 4), (1, 5), (2, 6), (3, 7)
  return make_uint4(fmha_q4::lows(a, b), fmha_q4::lows(c, d), fmha_q4::highs(a, b), fmha_q4::highs(c, d));
}

// out[b, h, i, :] = the values of position starts[b] + i; a word (8 values) of K and of V per thread.  A block takes `span`
// positions of one (b, h), `rows` of them at a time.
template <typename T>
__global__ void __launch_bounds__(256) gather_q4_kernel(const GatherArgs a) {
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const uint32_t bh = blockIdx.x / a.chunks, chunk = blockIdx.x - bh * a.chunks;
  const uint32_t b = bh / static_cast<uint32_t>(a.Hkv), h = bh - b * static_cast<uint32_t>(a.Hkv);
  const int row0 = threadIdx.x / a.words, j = threadIdx.x - row0 * a.words;
  if (row0 >= a.rows) return;
  const int o = q4::octet_of_word(j, a.groups);
  const int64_t start = a.starts ? a.starts[b] : 0;
  const uint32_t size = static_cast<uint32_t>(a.block_size);
  const int64_t end = min(static_cast<int64_t>(chunk + 1) * a.span, a.T);
  for (int64_t i = static_cast<int64_t>(chunk) * a.span + row0; i < end; i += a.rows) {
    const int64_t pos = start + i;
    const uint32_t logical = static_cast<uint32_t>(pos) / size;     // of positions from 0 on, below 2^32
    int64_t page = -1;
    if (pos >= 0 && logical < a.blocks_per_seq) page = a.block_table[b * a.blocks_per_seq + logical];
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (page >= 0 && page < a.num_blocks) {
      const int64_t row = (page * a.Hkv + h) * a.block_size + (static_cast<uint32_t>(pos) - logical * size);
      const uint32_t kw = a.k_codes[row * a.words + j], vw = a.v_codes[row * a.words + j];
      k = values_of<T>(kw, static_cast<const uint16_t*>(a.k_scales)[row * a.groups + (o >> 2)]);
      v = values_of<T>(vw, static_cast<const uint16_t*>(a.v_scales)[row * a.groups + (o >> 2)]);
    }
    const int64_t dst = ((bh * a.T + i) * a.words + o) * 8;
    *reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + dst) = k;
    *reinterpret_cast<uint4*>(static_cast<T*>(a.v_out) + dst) = v;
  }
}

struct Shape {
  int units, lanes, lane_shift;   // lanes: a power of two that holds a row's units
  int64_t blocks;
};
Shape shape_of(int64_t D, int64_t rows) {
  Shape s;
  s.units = static_cast<int>(D / 16);
  s.lanes = 2, s.lane_shift = 1;
  while (s.lanes < s.units) s.lanes <<= 1, ++s.lane_shift;
  s.blocks = (rows * s.lanes + 255) / 256;
  return s;
}

bool strides8(int64_t a, int64_t b, int64_t c) { return a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }

int write_common(bool q4, void* q_out, const int64_t* qo, void* k_pool, void* k_scales, void* v_pool, void* v_scales, const void* q,
                 const int64_t* qs, const void* k, const int64_t* ks, const void* v, const int64_t* vs, const void* q_weight,
                 const void* k_weight, const float* table, int64_t table_rows, int64_t rotary_dim, const int32_t* block_table,
                 const int32_t* offsets, const int32_t* rope_offsets, const int32_t* new_lens, int64_t B, int64_t H, int64_t Hkv,
                 int64_t T, int64_t D, int64_t blocks_per_seq, int64_t block_size, int64_t num_blocks, double eps, int interleaved,
                 int dtype, void* stream) {
  OB_REQUIRE(B >= 0 && T >= 0 && H >= 0 && Hkv > 0 && D > 0 && blocks_per_seq >= 0 && block_size > 0 && num_blocks > 0, OASR_ERR_INVALID,
             "write_kv_rope: bad shape");
  OB_REQUIRE(H + 2 * Hkv <= 65535, OASR_ERR_INVALID, "write_kv_rope: head count too large");
  OB_REQUIRE(D % 16 == 0 && D <= 512, OASR_ERR_UNSUPPORTED, "write_kv_rope: head_dim must be a multiple of 16 up to 512 (got %lld)", (long long)D);
  OB_REQUIRE(!q4 || D % 32 == 0, OASR_ERR_UNSUPPORTED, "write_kv_rope_q4: head_dim must be a multiple of 32 (got %lld)", (long long)D);
  OB_REQUIRE(rotary_dim > 0 && rotary_dim % 16 == 0 && rotary_dim <= D, OASR_ERR_UNSUPPORTED,
             "write_kv_rope: rotary_dim must be a multiple of 16 up to head_dim (got %lld)", (long long)rotary_dim);
  OB_REQUIRE(table_rows > 0, OASR_ERR_INVALID, "write_kv_rope: empty position table");
  if (B == 0 || T == 0) return OASR_OK;
  OB_REQUIRE(k_pool && v_pool && k && v && ks && vs && table && (block_table || blocks_per_seq == 0) && offsets && (!q4 || (k_scales && v_scales)) &&
                 (H == 0 || (q && q_out && qs && qo)),
             OASR_ERR_INVALID, "write_kv_rope: null pointer argument");
  OB_REQUIRE(strides8(ks[0], ks[1], ks[2]) && strides8(vs[0], vs[1], vs[2]) &&
                 (H == 0 || (strides8(qs[0], qs[1], qs[2]) && strides8(qo[0], qo[1], qo[2]))),
             OASR_ERR_ALIGN, "write_kv_rope: strides must be multiples of 8 elements");
  OB_REQUIRE(is_aligned(k_pool, 16) && is_aligned(v_pool, 16) && is_aligned(k, 16) && is_aligned(v, 16) && is_aligned(table, 16) &&
                 (H == 0 || (is_aligned(q, 16) && is_aligned(q_out, 16))) && is_aligned(q_weight, 16) && is_aligned(k_weight, 16),
             OASR_ERR_ALIGN, "write_kv_rope: operands must be 16-byte aligned");
  const Shape s = shape_of(D, B * T * (H + 2 * Hkv));
  OB_REQUIRE(block_size <= 0x7fffffff && B * T * (H + 2 * Hkv) <= 0x7fffff00 && s.blocks <= 0x7fffffff, OASR_ERR_INVALID,
             "write_kv_rope: too many rows for one call");
  static const int64_t kNone[3] = {0, 0, 0};
  if (H == 0) qs = qo = kNone;
  const WriteArgs a{q_out, k_pool, v_pool, k_scales, v_scales, q, k, v, q_weight, k_weight, table, block_table, offsets, rope_offsets, new_lens,
                    table_rows, B, T, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], qo[0], qo[1], qo[2],
                    blocks_per_seq, block_size, num_blocks, static_cast<int>(rotary_dim / 2), static_cast<int>(H), static_cast<int>(Hkv),
                    s.units, s.lanes, s.lane_shift, static_cast<int>(D / 32), 1.f / static_cast<float>(D),
                    static_cast<float>(eps)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(s.blocks));
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int {
    auto kern = q4 ? (interleaved ? write_kv_rope_kernel<T_, true, true> : write_kv_rope_kernel<T_, false, true>)
                   : (interleaved ? write_kv_rope_kernel<T_, true, false> : write_kv_rope_kernel<T_, false, false>);
    launch_pdl(kern, grid, dim3(256), 0, st, a);
    return check_launch("write_kv_rope launch");
  });
}

}  // namespace
}  // namespace ob

extern "C" {

int oasr_b200_qk_norm_rope(void* q_out, void* k_out, const void* q, const void* k, const void* q_weight, const void* k_weight,
                           const float* table, int64_t table_rows, int64_t rotary_dim, const void* positions, int pos_i64, int64_t N,
                           int64_t H, int64_t Hkv, int64_t D, int64_t qs_n, int64_t qs_h, int64_t ks_n, int64_t ks_h, int64_t qo_n,
                           int64_t qo_h, int64_t ko_n, int64_t ko_h, double eps, int interleaved, int dtype, void* stream) {
  using namespace ob;
  OB_REQUIRE(N >= 0 && H > 0 && Hkv >= 0 && D > 0, OASR_ERR_INVALID, "qk_norm_rope: bad shape");
  OB_REQUIRE(H + Hkv <= 65535, OASR_ERR_INVALID, "qk_norm_rope: head count too large");
  OB_REQUIRE(D % 16 == 0 && D <= 512, OASR_ERR_UNSUPPORTED, "qk_norm_rope: head_dim must be a multiple of 16 up to 512 (got %lld)", (long long)D);
  OB_REQUIRE(rotary_dim > 0 && rotary_dim % 16 == 0 && rotary_dim <= D, OASR_ERR_UNSUPPORTED,
             "qk_norm_rope: rotary_dim must be a multiple of 16 up to head_dim (got %lld)", (long long)rotary_dim);
  OB_REQUIRE(table_rows > 0, OASR_ERR_INVALID, "qk_norm_rope: empty position table");
  if (N == 0) return OASR_OK;
  OB_REQUIRE(q && q_out && table && positions && (Hkv == 0 || (k && k_out)), OASR_ERR_INVALID, "qk_norm_rope: null pointer argument");
  const int64_t e = dtype == OASR_DT_F32 ? 4 : 8;
  OB_REQUIRE(qs_n % e == 0 && qs_h % e == 0 && ks_n % e == 0 && ks_h % e == 0 && qo_n % e == 0 && qo_h % e == 0 && ko_n % e == 0 && ko_h % e == 0,
             OASR_ERR_ALIGN, "qk_norm_rope: strides must be multiples of 16 bytes");
  OB_REQUIRE(is_aligned(q, 16) && is_aligned(k, 16) && is_aligned(q_out, 16) && is_aligned(k_out, 16) && is_aligned(table, 16) &&
                 is_aligned(q_weight, 16) && is_aligned(k_weight, 16) && is_aligned(positions, pos_i64 ? 8 : 4),
             OASR_ERR_ALIGN, "qk_norm_rope: operands must be 16-byte aligned");
  // two heads a lane where that leaves every SM eight blocks
  const int batch = shape_of(D, N * ((H + Hkv) / 2)).blocks >= static_cast<int64_t>(sm_count()) * 8 ? 2 : 1;
  const int64_t q_chunks = (H + batch - 1) / batch, chunks = q_chunks + (Hkv + batch - 1) / batch;
  const Shape s = shape_of(D, N * chunks);
  OB_REQUIRE(N * chunks <= 0x7fffff00 && s.blocks <= 0x7fffffff, OASR_ERR_INVALID, "qk_norm_rope: too many rows for one call");
  const QkArgs a{q_out, k_out, q, k, q_weight, k_weight, table, positions, table_rows, N, qs_n, qs_h, ks_n, ks_h, qo_n, qo_h, ko_n, ko_h,
                 static_cast<int>(rotary_dim / 2), static_cast<int>(H), static_cast<int>(Hkv), static_cast<int>(q_chunks), s.units, s.lanes, s.lane_shift, pos_i64, 1.f / static_cast<float>(D), static_cast<float>(eps)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return OB_DISPATCH_FLOAT(dtype, T_, [&]() -> int {
    auto kern = batch == 2 ? (interleaved ? qk_norm_rope_kernel<T_, true, 2> : qk_norm_rope_kernel<T_, false, 2>)
                           : (interleaved ? qk_norm_rope_kernel<T_, true, 1> : qk_norm_rope_kernel<T_, false, 1>);
    launch_pdl(kern, dim3(static_cast<unsigned>(s.blocks)), dim3(256), 0, st, a);
    return check_launch("qk_norm_rope launch");
  });
}

int oasr_b200_write_kv_rope(void* q_out, const int64_t* q_out_strides, void* k_pool, void* v_pool, const void* q, const int64_t* q_strides,
                            const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, const void* q_weight,
                            const void* k_weight, const float* table, int64_t table_rows, int64_t rotary_dim, const int32_t* block_table,
                            const int32_t* offsets, const int32_t* rope_offsets, const int32_t* new_lens, int64_t B, int64_t H,
                            int64_t Hkv, int64_t T, int64_t D, int64_t blocks_per_seq, int64_t block_size, int64_t num_blocks, double eps,
                            int interleaved, int dtype, void* stream) {
  return ob::write_common(false, q_out, q_out_strides, k_pool, nullptr, v_pool, nullptr, q, q_strides, k, k_strides, v, v_strides, q_weight,
                          k_weight, table, table_rows, rotary_dim, block_table, offsets, rope_offsets, new_lens, B, H, Hkv, T, D,
                          blocks_per_seq, block_size, num_blocks, eps, interleaved, dtype, stream);
}

int oasr_b200_write_kv_rope_q4(void* q_out, const int64_t* q_out_strides, void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                               const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                               const int64_t* v_strides, const void* q_weight, const void* k_weight, const float* table,
                               int64_t table_rows, int64_t rotary_dim, const int32_t* block_table, const int32_t* offsets,
                               const int32_t* rope_offsets, const int32_t* new_lens, int64_t B, int64_t H, int64_t Hkv, int64_t T,
                               int64_t D, int64_t blocks_per_seq, int64_t block_size, int64_t num_blocks, double eps, int interleaved,
                               int dtype, void* stream) {
  return ob::write_common(true, q_out, q_out_strides, k_codes, k_scales, v_codes, v_scales, q, q_strides, k, k_strides, v, v_strides, q_weight,
                          k_weight, table, table_rows, rotary_dim, block_table, offsets, rope_offsets, new_lens, B, H, Hkv, T, D,
                          blocks_per_seq, block_size, num_blocks, eps, interleaved, dtype, stream);
}

int oasr_b200_paged_kv_gather_q4(void* k_out, void* v_out, const void* k_codes, const void* k_scales, const void* v_codes,
                                 const void* v_scales, const int32_t* block_table, const int32_t* starts, int64_t B, int64_t Hkv, int64_t T,
                                 int64_t D, int64_t blocks_per_seq, int64_t block_size, int64_t num_blocks, int dtype, void* stream) {
  using namespace ob;
  OB_REQUIRE(B >= 0 && T >= 0 && Hkv > 0 && D > 0 && blocks_per_seq >= 0 && block_size > 0 && num_blocks > 0, OASR_ERR_INVALID,
             "paged_kv_gather_q4: bad shape");
  OB_REQUIRE(D % 32 == 0 && D <= 512, OASR_ERR_UNSUPPORTED, "paged_kv_gather_q4: head_dim must be a multiple of 32 up to 512 (got %lld)", (long long)D);
  if (B == 0 || T == 0) return OASR_OK;
  OB_REQUIRE(k_out && v_out && k_codes && k_scales && v_codes && v_scales && (block_table || blocks_per_seq == 0), OASR_ERR_INVALID,
             "paged_kv_gather_q4: null pointer argument");
  OB_REQUIRE(is_aligned(k_out, 16) && is_aligned(v_out, 16) && is_aligned(k_codes, 16) && is_aligned(v_codes, 16), OASR_ERR_ALIGN,
             "paged_kv_gather_q4: operands must be 16-byte aligned");
  OB_REQUIRE(T <= 0x7fffffff && block_size <= 0x7fffffff, OASR_ERR_INVALID, "paged_kv_gather_q4: too long");
  const int words = static_cast<int>(D / 8), rows = 256 / words;
  const int span = rows * 4;   // four rounds a block where the sequence is that long
  const int64_t chunks = (T + span - 1) / span, grid = B * Hkv * chunks;
  OB_REQUIRE(grid <= 0x7fffffff, OASR_ERR_INVALID, "paged_kv_gather_q4: too many rows for one call");
  const GatherArgs a{k_out, v_out, static_cast<const uint32_t*>(k_codes), static_cast<const uint32_t*>(v_codes), k_scales, v_scales, block_table, starts,
                     B, Hkv, T, blocks_per_seq, block_size, num_blocks, words, static_cast<int>(D / 32), rows, span, static_cast<uint32_t>(chunks)};
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int {
    launch_pdl(gather_q4_kernel<T_>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, static_cast<cudaStream_t>(stream), a);
    return check_launch("paged_kv_gather_q4 launch");
  });
}

}  // extern "C"
