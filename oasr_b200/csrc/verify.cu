// Which drafted tokens stand against the target's probabilities, from given random numbers, and the token behind them:
//
//   n = 0;  p = softmax(logits[n] / temperature)
//   for the children c of n in order, x = drafts[c]:     accepted iff  u_c q(x) < p(x)  (then n = c, and from the start);
//                                                        p <- max(p - q, 0), normalised
//   none accepted: the token is the first whose cumulative p passes u_0.
//
// q is the distribution that the children of n were drawn from (draft_probs[n]), or 1 at x where drafts are taken as chosen.  A
// temperature of zero puts all of p on the first maximum.  Whoever drafted, the tokens are distributed as the target alone would give them.
//
// The answer is whole numbers, so what decides is computed in 64 bits: weights e^(l / temperature) to some 2^-31, their sums in an order that follows
// from the batch, the vocabulary and the type (the number of warps that share a row), so that a call repeats itself.
// They come out of a table of 2^(i / 256) and a polynomial of degree 3 for the rest (the method of Tang, "Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic", 1989).  Weights are taken relative to logits of 0: 64 bits reach 2^250 above and 2^500 below; rows
// that lie elsewhere are taken again relative to their maximum.
// Bound by the walk: a node's rows are read, summed and decided before the next one's address is known (16 trees of 48 over 131071 bf16 logits: 15.0 us,
// floor 1.3; 32 chains of 8 with their own probabilities over 65537 fp32 logits: 34.2 us, floor 3.8).  That is this kernel's choice: only which row comes
// next depends on the decisions.  All rows of all nodes would take 31 us at the first of these, but 10 at the second and 0.02 at 3 chains of 5 over 5002
// (12.1 us).
// p and q unnormalised: with k children rejected  p_k = max(p - beta_k q, 0) / Pi_k,  Pi_k the sum of the numerators, beta_1 = 1 and
// beta_{k+1} = beta_k + Pi_k.  Where Pi_k has become so small that the next difference would be one of roundings, p_k takes p's place and it begins anew.
// With q = 1 at x a rejection takes x's weight out of the sum.
//
// A cluster of blocks walks one sequence's tree and reads the rows on the accepted path only; every warp owns a run of the vocabulary.  Per
// node: a pass over the row, the warps' sums to every block of the cluster, and every warp takes the same decision from them.  The warp whose
// run has the drawn token walks through it again.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "sm100_ptx.cuh"
#include "smem_limit.cuh"

namespace ob {
namespace verify {
namespace {

constexpr int kMaxWarps = 16, kMaxCluster = 8, kSlots = kMaxWarps * kMaxCluster, kTable = 256, kCopies = 16, kMaxNodes = 1024, kVec = 8;

struct Args {
  int32_t *tokens, *path, *counts;
  const void* logits;
  const float* probs;
  const int32_t *drafts, *parents;
  const float *uniforms, *temperatures;
  int64_t ls_b, ls_n, ps_b, ps_n, parents_b;   // strides: logits, draft probabilities, parents of a sequence (0: one tree for all)
  int B, T, V;
  float temperature;
  uint32_t two12, two21;   // 2^12 and 2^21 as numbers that the compiler does not know: products with them are no shifts (see near_zero)
};

// 2^((i - 1/2) / 256) less i 2^12 in its upper word, so that k 2^12 added there gives table[k mod 256] 2^(k div 256)
struct Table {
  uint64_t e[kTable];
  constexpr Table() : e() {
    for (int i = 0; i < kTable; ++i) {
      const double x = (i - 0.5) * (0.69314718055994530942 / kTable);
      double sum = 1., term = 1.;
      for (int n = 1; n < 24; ++n) term = term * x / n, sum += term;
      // the bits of a number of [1/2, 2)
      const bool low = sum < 1.;
      e[i] = (static_cast<uint64_t>(low ? 1022 : 1023) << 52) + static_cast<uint64_t>((low ? 2. * sum : sum) * 4503599627370496. - 4503599627370496.) - (static_cast<uint64_t>(i) << 44);
    }
  }
};
__device__ constexpr Table g_table{};

// The table lies there 16 times: half a warp reads 16 entries of 8 bytes at a time, each lane from banks of its own.  What the warps of a cluster
// tell one another about a row (a number and a whole number each) is held twice, in turn: a barrier lies between a use and the next
// writing of the same one.  Behind it: stages of rejections, parents, drafts, uniforms, first child and next sibling of T nodes.
struct Shared {
  double table[kTable][kCopies];
  double sum[2][kSlots];
  int id[2][kSlots];
  int stages[kMaxWarps];   // each warp's count of them
};

// e^((l - ref) / temperature).  A row that lies around zero has ref 0; then the multiple of 2^(1 / 256) and the rest f come from fp32 operations
// (a product is exact inside its sum, and the rest is small), and 2^(f / 256) is the 64-bit number 1 + G 2^-31 with G out of the low bits of an fp32
// sum: one 64-bit multiply-add a weight.  Both 64-bit numbers are put together by integer multiply-adds: logic and shifts, half as fast, were 0.94
// busy (65537 logits by four blocks: 6.3k clocks).  Any other row takes it in 64 bits throughout.
struct Weigher {
  const double* table;   // the lane's copy
  double rate, ref;      // 256 log2(e) / temperature
  float rate_hi, rate_lo, lo, hi;   // logits below lo have no weight, logits above hi are out of range
  uint32_t two12, two21;
  bool centered;

  __device__ __forceinline__ void relative_to(float r, bool centered_) {
    ref = r;
    centered = centered_;
    rate_hi = static_cast<float>(rate), rate_lo = static_cast<float>(rate - static_cast<double>(rate_hi));
    lo = static_cast<float>(fmax(ref - 500. * kTable / rate, static_cast<double>(-FLT_MAX)));   // rounded away from ref by at most as much again
    hi = static_cast<float>(fmin(ref + 250. * kTable / rate, static_cast<double>(FLT_MAX)));
  }
  // the weight of lo <= l <= hi, ref 0, in two factors: table[k mod 256] 2^(k div 256), entries for half a step less, and 2^((f + 1/2) / 256)
  __device__ __forceinline__ void near_zero(float l, double& v, double& d) const {
    constexpr float kMagic = 12582912.f, kUnit = 1.f / 256.f;   // 1.5 * 2^23 and 2^-8: low bits of a sum with them are whole numbers
    constexpr double kStep = 0.6931471805599453 / kTable, kHalf = kStep / 2, kRoot = 1 + kHalf * (1 + kHalf / 2 * (1 + kHalf / 3 * (1 + kHalf / 4)));   // 2^(1 / 512)
    constexpr float c0 = static_cast<float>(kUnit + (kRoot - 1)), c1 = static_cast<float>(kRoot * kStep), c2 = static_cast<float>(kRoot * kStep * kStep / 2),
                    c3 = static_cast<float>(kRoot * kStep * kStep * kStep / 6);
    const float t = fmaf(l, rate_hi, kMagic);
    const float f = fmaf(l, rate_lo, fmaf(l, rate_hi, kMagic - t));   // in [-1/2, 1/2]
    const uint32_t k = __float_as_uint(t), g = __float_as_uint(fmaf(fmaf(fmaf(f, c3, c2), f, c1), f, c0));
    v = scaled(k);
    constexpr uint64_t kOne = (uint64_t(0x3ff00000) << 32) - (uint64_t(0x3b800000) << 21);
    uint64_t r;
    asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(g), "r"(two21), "l"(kOne));
    d = __longlong_as_double(r);
  }
  __device__ __forceinline__ double scaled(uint32_t k) const {   // (of k only the low 20 bits matter: 1.5 2^23 has none there)
    const double e = table[(k & (kTable - 1)) * kCopies];
    uint32_t hi_word;
    asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(hi_word) : "r"(k), "r"(two12), "r"(__double2hiint(e)));
    return __hiloint2double(hi_word, __double2loint(e));
  }
  __device__ __forceinline__ double near_zero(float l) const {
    double v, d;
    near_zero(l, v, d);
    return v * d;
  }
  __device__ __forceinline__ double far(float l) const {
    constexpr double kMagic = 6755399441055744.;   // 1.5 * 2^52
    constexpr double c1 = 0.6931471805599453 / kTable, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
    const double x = static_cast<double>(fminf(l, hi)) - ref;
    const double t = fma(x, rate, kMagic);
    const double f = fma(x, rate, -(t - kMagic)) + 0.5;
    return scaled(__double2loint(t)) * fma(fma(fma(f, c3, c2), f, c1), f, 1.);
  }
  __device__ __forceinline__ double operator()(float l) const;
};
static_assert(kTable == 256, "the exponent is what is above 8 bits");
// Out of line (instructions that a block runs once come from memory, and there are enough of them), by value (a struct whose address is taken
// lives there too).
__device__ __noinline__ double far_weight(const double* table, double rate, double ref, float hi, uint32_t two12, float l) {
  return Weigher{table, rate, ref, 0.f, 0.f, 0.f, hi, two12, 0, false}.far(l);
}
__device__ __forceinline__ double Weigher::operator()(float l) const {
  if (!(l >= lo)) return 0.;
  return centered ? near_zero(fminf(l, hi)) : far_weight(table, rate, ref, hi, two12, l);
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan64(double v) {   // sums of the lanes up to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += w;
  }
  return v;
}

// A row of logits in vectors of eight that start on a boundary of 16 bytes: vector j has tokens first(j) .. first(j) + 7, those outside
// [0, V) at -inf.
template <typename T>
struct Vec {
  Pack<T> p[kVec / Elem<T>::kVec];
  __device__ __forceinline__ T& operator[](int i) { return p[i / Elem<T>::kVec].v[i % Elem<T>::kVec]; }
  __device__ __forceinline__ const T& operator[](int i) const { return p[i / Elem<T>::kVec].v[i % Elem<T>::kVec]; }
  __device__ __forceinline__ float operator()(int i) const { return Elem<T>::to_f((*this)[i]); }
};
// The largest of many logits (NaN where there is one) and logits raised to a least one, two 16-bit ones an instruction.  That one lies between kLeast
// and -kFinest (see verify_kernel): the type has it to its full precision there (fp16: above its subnormal numbers), and the rates, 1.3e5 over it, fit fp32.
template <typename T>
struct Range;
template <>
struct Range<float> {
  static constexpr float kLeast = -FLT_MAX, kFinest = 1e-32f;
  float lo, top = -INFINITY;
  __device__ __forceinline__ explicit Range(float l) : lo(l) {}
  __device__ __forceinline__ void note(const Vec<float>& x) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(x[i]));
  }
  __device__ __forceinline__ void take(Vec<float>& x) {
    note(x);
#pragma unroll
    for (int i = 0; i < kVec; ++i) x[i] = fmaxf(x[i], lo);
  }
  __device__ __forceinline__ float largest() const { return top; }
};
template <typename T, typename T2>
struct Range16 {
  T2 lo, top;
  __device__ __forceinline__ explicit Range16(float l) {
    lo.x = lo.y = Elem<T>::from_f(l);
    top.x = top.y = Elem<T>::from_f(-INFINITY);
  }
  __device__ __forceinline__ void note(const Vec<T>& x) {
#pragma unroll
    for (int i = 0; i < kVec; i += 2) top = __hmax2_nan(top, *reinterpret_cast<const T2*>(&x[i]));
  }
  __device__ __forceinline__ void take(Vec<T>& x) {
    note(x);
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
      T2& v = *reinterpret_cast<T2*>(&x[i]);
      v = __hmax2(v, lo);
    }
  }
  __device__ __forceinline__ float largest() const {
    const float a = Elem<T>::to_f(top.x), b = Elem<T>::to_f(top.y);
    return a != a ? a : b != b ? b : fmaxf(a, b);
  }
};
template <>
struct Range<__half> : Range16<__half, __half2> {
  using Range16::Range16;
  static constexpr float kLeast = -65504.f, kFinest = 6.103515625e-5f;
};
template <>
struct Range<__nv_bfloat16> : Range16<__nv_bfloat16, __nv_bfloat162> {
  using Range16::Range16;
  static constexpr float kLeast = -3.3895314e38f, kFinest = 1e-32f;
};
template <typename T>
struct Row {
  const T* p;
  int V, skew;
  __device__ __forceinline__ Row(const T* p_, int V_) : p(p_), V(V_), skew(static_cast<int>(reinterpret_cast<uintptr_t>(p_) % 16 / sizeof(T))) {}
  __device__ __forceinline__ int vectors() const { return (V + skew + kVec - 1) / kVec; }
  __device__ __forceinline__ int first(int j) const { return j * kVec - skew; }
  __device__ __forceinline__ Vec<T> load(int j) const {
    const int v0 = first(j);
    Vec<T> v;
    if (v0 >= 0 && v0 + kVec <= V) {
#pragma unroll
      for (int i = 0; i < kVec / Elem<T>::kVec; ++i) v.p[i] = ld128(p + v0 + i * Elem<T>::kVec);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = v0 + i >= 0 && v0 + i < V ? p[v0 + i] : Elem<T>::from_f(-INFINITY);
    }
    return v;
  }
  // the draft's probabilities of the same tokens
  __device__ __forceinline__ void load_probs(const float* q, int j, float (&x)[kVec]) const {
    const int v0 = first(j);
    if (v0 >= 0 && v0 + kVec <= V && (reinterpret_cast<uintptr_t>(q + v0) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < kVec; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(q + v0 + i);
        x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) x[i] = v0 + i >= 0 && v0 + i < V ? q[v0 + i] : 0.f;
    }
  }
  // f(j, logits) for this lane's vectors j0 + lane, j0 + lane + 32, ... below j1, kBatch loads at a time
  template <int kBatch, typename F>
  __device__ __forceinline__ void each(int j0, int j1, F&& f) const {
    int j = j0 + static_cast<int>(threadIdx.x & 31);
#pragma unroll 1
    for (; j + 32 * (kBatch - 1) < j1; j += 32 * kBatch) {
      Vec<T> x[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) x[i] = load(j + 32 * i);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) f(j + 32 * i, x[i]);
    }
    if constexpr (kBatch > 1) {
#pragma unroll 1
      for (; j < j1; j += 32) {
        Vec<T> x = load(j);
        f(j, x);
      }
    }
  }
};

// The passes over a warp's run [j0, j1) of a row.  Each is a function of its own, with the registers to itself: inlined into the walk through the
// tree the constants of the first were made anew for every logit (37 instructions each in the place of 17).

// What a total of weights around zero has to reach, and a warp's sum to be one: a row's weights down to 2^-300 of its largest count.
constexpr double kLeastTotal = 0x1p-160, kLeastSum = 0x1p-465;

// this lane's sum of weights around zero, NaN where a logit lies outside.  Logits below the range count as ones at its end: 2^-499 or
// less each, of up to 2^27 together less than kLeastSum
template <typename T>
__device__ __noinline__ double sum_near(const Row<T> row, const Weigher weigh, const int j0, const int j1) {
  double s0 = 0., s1 = 0.;
  Range<T> range(weigh.lo);
  row.template each<2>(j0, j1, [&](int, Vec<T>& x) {
    range.take(x);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      double v, d;
      weigh.near_zero(x(i), v, d);
      if (i & 1) s1 = fma(v, d, s1);
      else s0 = fma(v, d, s0);
    }
  });
  return range.largest() <= weigh.hi ? s0 + s1 : NAN;
}

// The same in fp32, 4 instructions a logit in the place of 20.  |log2(weight)| stays below 127, so its product and its factor are off by 2^-17.4 and
// 2^-17.4 at most, the exponential by 2^-22, sums of up to 128 in a row (kMostUnits) by 2^-17: kSlack holds them all.
constexpr double kSlack = 0x1p-15;
constexpr int kMostUnits = 64;   // of a warp: 512 logits a lane, in four sums
template <typename T>
__device__ __noinline__ float sum_fast(const Row<T> row, const float rate, const float hi, const int j0, const int j1) {
  float s[4] = {};
  Range<T> range(-INFINITY);
  row.template each<2>(j0, j1, [&](int, const Vec<T>& x) {
    range.note(x);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      float e;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x(i) * rate));
      s[i & 3] += e;
    }
  });
  return range.largest() <= hi ? (s[0] + s[1]) + (s[2] + s[3]) : NAN;
}

// the largest logit (NaN: there is one) and its first token
struct Largest {
  float l;
  int token;
  __device__ __forceinline__ void take(float v, int w) {
    if (v != v || v > l || (v == l && w < token)) l = l != l ? l : v, token = w;
  }
  __device__ __forceinline__ void of_warp() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) take(__shfl_xor_sync(0xffffffffu, l, o), __shfl_xor_sync(0xffffffffu, token, o));
  }
};
template <typename T>
__device__ __noinline__ Largest largest_of(const Row<T> row, const int j0, const int j1) {
  Largest best{-INFINITY, 0x7fffffff};
  row.template each<1>(j0, j1, [&](int j, const Vec<T>& x) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) best.take(x(i), row.first(j) + i);
  });
  best.of_warp();
  return best;
}

// What rejections have made of p: p = weight inv, then n times p <- max(p - beta q, 0) scale, of each stage's numbers, and at last max(p - beta q, 0) (not
// divided by its sum).  With beta 0 nothing was rejected, and it is the weight as it stands.  The stages lie in shared memory behind what Shared has.
struct Stage {
  double beta, scale;
};
__device__ __forceinline__ double left_in_stages(double p, const double y, const double beta, const int n) {
  extern __shared__ __align__(16) uint8_t smem[];
  const Stage* const stages = reinterpret_cast<const Stage*>(smem + sizeof(Shared));
#pragma unroll 1
  for (int i = 0; i < n; ++i) p = fmax(fma(-stages[i].beta, y, p), 0.) * stages[i].scale;
  return fmax(fma(-beta, y, p), 0.);
}
constexpr double kLeastRest = 0x1p-16;   // a difference of numbers of 53 bits keeps 37 of them: more than weights have

// What is left of eight tokens' weights, with y the draft's probabilities.
template <typename T>
__device__ __forceinline__ void remaining(const Weigher& weigh, const Vec<T>& x, const float (&y)[kVec], double inv, double beta, int stages, double (&w)[kVec]) {
  if (weigh.centered) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) w[i] = weigh.near_zero(fmaxf(x(i), weigh.lo));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) w[i] = weigh(x(i));
  }
  if (beta > 0.) {
    if (stages > 0) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) w[i] = left_in_stages(w[i] * inv, static_cast<double>(y[i]), beta, stages);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) w[i] = fma(w[i], inv, -beta * static_cast<double>(y[i]));
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (!(x(i) >= weigh.lo && w[i] > 0.)) w[i] = 0.;
}
// this lane's sum of it
template <typename T>
__device__ __noinline__ double sum_remaining(const Row<T> row, const Weigher weigh, const int j0, const int j1, const float* q, const double inv, const double beta,
                                              const int stages) {
  double s = 0.;
#pragma unroll 1
  for (int j = j0 + static_cast<int>(threadIdx.x & 31); j < j1; j += 32) {
    const Vec<T> x = row.load(j);
    float y[kVec] = {};
    if (beta > 0.) row.load_probs(q, j, y);
    double w[kVec];
    remaining(weigh, x, y, inv, beta, stages, w);
    s += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  }
  return s;
}

// kDrawn: with the draft's probabilities.  (One kernel for both fetches the instructions of either around the other's: 3 chains of 5 over 5002 logits 13.1 us,
// 12.1 so; 32 drawn chains of 8 over 65537 36.9, 34.2.)
template <typename T, int kWarps, bool kDrawn>
__global__ void __launch_bounds__(kWarps * 32, kMaxWarps / kWarps) verify_kernel(const Args a, const int C) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  Stage* const stages = reinterpret_cast<Stage*>(smem + sizeof(Shared));   // (see left_in_stages)
  int* const parents = reinterpret_cast<int*>(stages + a.T);
  int* const drafts = parents + a.T;
  float* const u = reinterpret_cast<float*>(drafts + a.T);
  int* const first_kid = reinterpret_cast<int*>(u + a.T);   // a.T: none
  int* const sibling = first_kid + a.T;
  int* const token_of = sibling + a.T;                       // what the walk has found so far: stored at the end, as a barrier waits for stores
  int* const node_of = token_of + a.T;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = C > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0, b = static_cast<int>(blockIdx.x) / C;
  constexpr int kThreads = kWarps * 32, kFills = 2 * kTable / kThreads;   // a thread fills half of the copies of so many entries
  uint64_t entry[kFills];                                                 // (stored once the tree's loads are on their way)
#pragma unroll
  for (int i = 0; i < kFills; ++i) entry[i] = g_table.e[(threadIdx.x + i * kThreads) % kTable];
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // waited for before the first word to another block
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int slots = C * kWarps, slot_bits = __ffs(slots) - 1, mine = warp * C + rank;   // in the order of the vocabulary: few runs are dealt to all blocks
  auto row_of = [&](int n) { return Row<T>(static_cast<const T*>(a.logits) + b * a.ls_b + n * a.ls_n, a.V); };
  // A row's vectors in units of 32, as evenly over the warps as units go: the first `more` have one above `each`.
  auto run_of = [&](const Row<T>& row, int& each, int& more, int& j0, int& j1) {
    const int units = (row.vectors() + 31) >> 5;
    each = units >> slot_bits, more = units & (slots - 1);
    j0 = min((mine * each + min(mine, more)) * 32, row.vectors()), j1 = min(j0 + (each + (mine < more)) * 32, row.vectors());
  };
  // elements [e0, e1) of a row of V, towards the L2 cache
  auto ahead = [&](const auto* p, int e0, int e1) {
    const char *at = reinterpret_cast<const char*>(p + max(e0, 0)) + lane * 128, *end = reinterpret_cast<const char*>(p + min(e1, a.V));
#pragma unroll 1
    for (; at < end; at += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
  };
  {
    const Row<T> row = row_of(0);
    int each, more, j0, j1;
    run_of(row, each, more, j0, j1);
    ahead(row.p, row.first(j0), row.first(j1));
  }
  for (int i = threadIdx.x; i < a.T; i += kThreads) {
    parents[i] = a.parents[b * a.parents_b + i];
    drafts[i] = a.drafts[static_cast<int64_t>(b) * a.T + i];
    u[i] = a.uniforms[static_cast<int64_t>(b) * a.T + i];
  }
  const float temperature = a.temperatures ? a.temperatures[b] : a.temperature;
#pragma unroll
  for (int f = 0; f < kFills; ++f) {
    const int item = threadIdx.x + f * kThreads, at = item % kTable;
#pragma unroll
    for (int i = 0; i < kCopies / 2; ++i) sh.table[at][(at + i) % (kCopies / 2) + item / kTable * (kCopies / 2)] = __longlong_as_double(entry[f]);
  }
  const bool greedy = !(temperature > 0.f);
  int32_t* const tokens = a.tokens + static_cast<int64_t>(b) * a.T;
  int32_t* const path = a.path + static_cast<int64_t>(b) * a.T;
  const bool writer = rank == 0 && threadIdx.x == 0;
  __syncthreads();
  for (int i = warp; i < a.T; i += kWarps) {   // a warp per node: its children, from the last one on
    int next = a.T;
#pragma unroll 1
    for (int base = (a.T - 1) & ~31; base + 31 > i; base -= 32) {
      const int k = base + lane;
      const bool is = k > i && k < a.T && parents[k] == i;
      const uint32_t m = __ballot_sync(0xffffffffu, is), above = m & ~((2u << lane) - 1);
      if (is) sibling[k] = above ? base + __ffs(above) - 1 : next;
      if (m) next = base + __ffs(m) - 1;
    }
    if (lane == 0) first_kid[i] = next;
  }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every block of the cluster runs: its shared memory may be written

  int turn = 0;
  auto meet = [&](double sum, int id) {   // all warps' numbers in sum[turn ^ 1], id[turn ^ 1] of every block
    if (C == 1) {
      if (lane == 0) sh.sum[turn][mine] = sum, sh.id[turn][mine] = id;
      __syncthreads();
    } else {
      if (lane < C) {
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(ptx::map_to_cta(&sh.sum[turn][mine], lane)), "d"(sum) : "memory");
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ptx::map_to_cta(&sh.id[turn][mine], lane)), "r"(id) : "memory");
      }
      __syncwarp();
      ptx::cluster_sync();
    }
    turn ^= 1;
  };
  auto sum_all = [&]() {   // of all warps, in an order that is the same everywhere
    double s[kSlots / 32];
#pragma unroll
    for (int i = 0; i < kSlots / 32; ++i) s[i] = i * 32 + lane < slots ? sh.sum[turn ^ 1][i * 32 + lane] : 0.;
    static_assert(kSlots / 32 == 4, "four a lane");
    return warp_sum64((s[0] + s[1]) + (s[2] + s[3]));
  };

  int n = 0, count = 0;
  if (writer) node_of[0] = 0;
  Weigher weigh{&sh.table[0][lane % kCopies], kTable * 1.4426950408889634 / static_cast<double>(temperature), 0., 0.f, 0.f, 0.f, 0.f, a.two12, a.two21, true};
#pragma unroll 1
  for (;;) {
    const Row<T> row = row_of(n);
    const float* const q = kDrawn ? a.probs + b * a.ps_b + n * a.ps_n : nullptr;
    int each, longer, j0, j1;
    run_of(row, each, longer, j0, j1);
    // Children of the node, one a lane, up to 32 at a time.  A lane without one, or whose draft is no token, has token -1.
    const int kid0 = first_kid[n];
    int kid = a.T, kid_token = -1;
    T kid_logit = Elem<T>::from_f(0.f);
    float kid_q = 1.f;
    auto take_kids = [&](int from) {   // -> the first one that is left
      kid = a.T;
      int i = 0;
#pragma unroll 1
      for (; i < 32 && from < a.T; ++i, from = sibling[from])
        if (lane == i) kid = from;
      kid_token = kid < a.T ? drafts[kid] : -1;
      if (kid_token >= a.V || kid_token < 0) kid_token = -1;
      if (kid_token >= 0) {
        kid_logit = row.p[kid_token];
        if (kDrawn) kid_q = q[kid_token];
      }
      return from;
    };
    int more = take_kids(kid0);
    bool several = false;   // more than 32 of them
    if (kid0 < a.T) {   // the row of the child that is tried first, and the draft's, towards the L2 cache while this row is walked through
      ahead(row_of(kid0).p, row.first(j0), row.first(j1));
      if (kDrawn) ahead(q, row.first(j0), row.first(j1));
    }

    auto tell_sum = [&](double s) {
      s = warp_sum64(s);
      meet(s < kLeastSum ? 0. : s, 0);
      return sum_all();
    };

    int accepted = -1, accepted_token = -1, at = 0;
    double total = 0.;
    bool fine = true;
    double kid_w = 0.;
    bool kid_again = false;
    // whether an earlier child had this lane's token
    auto repeated = [&]() {
      bool same = (__match_any_sync(0xffffffffu, kid_token) & ((1u << lane) - 1)) != 0;
      if (several && kid_token >= 0)
        for (int k = kid0; !same && k < kid; k = sibling[k]) same = drafts[k] == kid_token;
      return same;
    };
    weigh.relative_to(0.f, true);
    // (Temperatures of up to 3e-35, fp16 2e-7, or from 1e36, fp16 200, on: weights relative to the row's largest logit, in 64 bits throughout.)
    const bool in_range = !greedy && weigh.lo > Range<T>::kLeast && weigh.lo <= -Range<T>::kFinest;
    if (in_range && kid0 < a.T && more >= a.T && each >= 2 && each < kMostUnits) {
      // ---- a child that is accepted, or refused, by more than what fp32 may be off needs no more than that (runs of less are as fast in 64 bits)
      const float rate = weigh.rate_hi * (1.f / kTable);
      total = tell_sum(sum_fast(row, rate, 120.f / rate, j0, j1));
      if (total >= 0x1p-60) {
        kid_w = kid_token >= 0 ? weigh(Elem<T>::to_f(kid_logit)) : 0.;
        kid_again = repeated();
        const double draw = (kid < a.T ? static_cast<double>(u[kid]) : 0.) * static_cast<double>(kid_q), slack = total * kSlack;
        double rest = total;
#pragma unroll 1
        for (uint32_t todo = __ballot_sync(0xffffffffu, kid_token >= 0); todo; todo &= todo - 1) {
          const int k = __ffs(todo) - 1;
          const double w = !kDrawn && kid_again ? 0. : kid_w;
          if (__shfl_sync(0xffffffffu, draw * (rest + slack) < w, k)) {
            accepted = __shfl_sync(0xffffffffu, kid, k), accepted_token = __shfl_sync(0xffffffffu, kid_token, k);
            break;
          }
          if (kDrawn || __shfl_sync(0xffffffffu, draw * (rest - slack) < w, k)) break;
          rest = fmax(rest - __shfl_sync(0xffffffffu, w, k), 0.);
        }
      }
      total = 0.;
    }
    if (accepted < 0) {
      if (in_range) total = tell_sum(sum_near(row, weigh, j0, j1));
      if (!(total >= kLeastTotal)) {   // greedy, or the row does not lie around zero (or all of a type's numbers do)
        Largest best = largest_of(row, j0, j1);
        meet(best.l, best.token);
        best = {-INFINITY, 0x7fffffff};
        for (int i = lane; i < slots; i += 32) best.take(static_cast<float>(sh.sum[turn ^ 1][i]), sh.id[turn ^ 1][i]);
        best.of_warp();
        fine = fabsf(best.l) < INFINITY;   // there is a distribution
        at = best.token;
        if (fine && !greedy) {
          weigh.relative_to(best.l, false);
          total = tell_sum(sum_remaining<T>(row, weigh, j0, j1, nullptr, 1., 0., 0));
        }
      }
    }
    // ---- the children in turn.  `rest` is Pi (of p unnormalised while nothing is rejected): p is what is left of a weight (max(weight inv - beta q, 0), or
    // that in stages) divided by it.
    double beta = 0., inv = 1., rest = greedy ? 1. : total;
    if (kDrawn && lane == 0) sh.stages[warp] = 0;
    __syncwarp();
    const float q_at = greedy && fine && kDrawn ? q[at] : 0.f;
    auto own_weight = [&]() { return kid_token < 0 ? 0. : greedy ? (kid_token == at ? 1. : 0.) : weigh(Elem<T>::to_f(kid_logit)); };
#pragma unroll 1
    while (accepted < 0 && fine && kid0 < a.T) {
      kid_w = own_weight();
      kid_again = repeated();
      const float kid_u = kid < a.T ? u[kid] : 0.f;
      uint32_t todo = __ballot_sync(0xffffffffu, kid_token >= 0);
#pragma unroll 1
      for (; todo && accepted < 0; todo &= todo - 1) {
        const int k = __ffs(todo) - 1;
        if (kDrawn) {
          const double w = beta > 0. ? left_in_stages(kid_w * inv, static_cast<double>(kid_q), beta, sh.stages[warp]) : kid_w;
          const bool good = static_cast<double>(kid_u) * static_cast<double>(kid_q) * rest < w;
          if (__shfl_sync(0xffffffffu, good, k)) {
            accepted = __shfl_sync(0xffffffffu, kid, k), accepted_token = __shfl_sync(0xffffffffu, kid_token, k);
            break;
          }
          inv = greedy ? 1. : 1. / total;
          if (beta > 0. && rest > 0. && rest < kLeastRest) {   // (every warp writes the same, and reads what it has written)
            const int s = sh.stages[warp];
            __syncwarp();
            stages[s] = Stage{beta, 1. / rest};
            if (lane == 0) sh.stages[warp] = s + 1;
            __syncwarp();
            beta = 0.;
          }
          beta = beta > 0. ? beta + rest : 1.;
          if (greedy) {
            rest = left_in_stages(1., static_cast<double>(q_at), beta, sh.stages[warp]);
          } else {
            meet(warp_sum64(sum_remaining(row, weigh, j0, j1, q, inv, beta, sh.stages[warp])), 0);
            rest = sum_all();
          }
        } else {
          const double w = kid_again ? 0. : kid_w;
          const bool good = static_cast<double>(kid_u) * rest < w;
          if (__shfl_sync(0xffffffffu, good, k)) {
            accepted = __shfl_sync(0xffffffffu, kid, k), accepted_token = __shfl_sync(0xffffffffu, kid_token, k);
            break;
          }
          rest = fmax(rest - __shfl_sync(0xffffffffu, w, k), 0.);
        }
      }
      if (accepted >= 0 || more >= a.T) break;
      several = true;
      more = take_kids(more);
    }
    if (accepted >= 0) {
      if (writer) token_of[count] = accepted_token, node_of[count + 1] = accepted;
      ++count;
      n = accepted;
      continue;
    }
    // ---- the token behind the path
    if (!fine || greedy) {
      if (writer) tokens[count] = fine && rest > 0. ? at : -1;
      break;
    }
    // The warps' sums in the order of the vocabulary, `span` to a lane, without the children's weights where those are out.
    const int span = (slots + 31) / 32;
    double part[kSlots / 32];
    auto take_sums = [&]() {
#pragma unroll
      for (int i = 0; i < kSlots / 32; ++i) part[i] = i < span && lane * span + i < slots ? sh.sum[turn ^ 1][lane * span + i] : 0.;
    };
    take_sums();
    const bool without = !kDrawn && kid0 < a.T;
    auto each_kid = [&](auto&& f) {   // f(token, weight) for every rejected child's token, once
      int further = several ? take_kids(kid0) : a.T;
#pragma unroll 1
      for (;;) {
        if (several) kid_w = own_weight(), kid_again = repeated();
#pragma unroll 1
        for (uint32_t todo = __ballot_sync(0xffffffffu, kid_token >= 0 && !kid_again); todo; todo &= todo - 1) {
          const int k = __ffs(todo) - 1;
          f(__shfl_sync(0xffffffffu, kid_token, k), __shfl_sync(0xffffffffu, kid_w, k));
        }
        if (further >= a.T) break;
        further = take_kids(further);
      }
    };
    // A run that has little but its children's weights (2^-32 of its sum; the differences are off by 2^-35 at most) is summed again without them: a
    // difference of roundings would be a run that has no token to give, or hide one that has.
    bool touched = false, again = false;   // a child's token lies in this warp's run; there are such runs
    if (without) {
      each_kid([&](int token, double w) {
        const int unit = (token + row.skew) / (kVec * 32), split = longer * (each + 1);
        const int owner = unit < split ? unit / (each + 1) : longer + (unit - split) / each;   // (`each` 0: all units lie below the split)
        touched |= owner == mine;
#pragma unroll
        for (int i = 0; i < kSlots / 32; ++i)
          if (owner == lane * span + i && i < span) part[i] = fmax(part[i] - w, 0.);
      });
#pragma unroll
      for (int i = 0; i < kSlots / 32; ++i) {
        const double with = i < span && lane * span + i < slots ? sh.sum[turn ^ 1][lane * span + i] : 0.;
        again |= with > 0. && part[i] <= with * 0x1p-32;
      }
      again = __any_sync(0xffffffffu, again);
    }
#pragma unroll 1
    for (;; again = false) {
      double goal = INFINITY;
      bool here = touched;   // whether this warp walks through its run
      if (!again) {
        const double lane_sum = (part[0] + part[1]) + (part[2] + part[3]), upto = warp_scan64(lane_sum);
        const double all = __shfl_sync(0xffffffffu, upto, 31), target = static_cast<double>(u[0]) * all;
        // the first warp whose cumulative sum passes the target, else the last one with something in it
        const uint32_t past = __ballot_sync(0xffffffffu, lane_sum > 0. && upto > target), some = __ballot_sync(0xffffffffu, lane_sum > 0.);
        const int lane_of = past ? __ffs(past) - 1 : 31 - __clz(some | 1u);
        double before = upto - lane_sum, prefix = 0., last_prefix = 0.;
        int owner = -1, last_owner = -1;
#pragma unroll
        for (int i = 0; i < kSlots / 32; ++i) {
          if (part[i] > 0.) {
            last_owner = lane * span + i, last_prefix = before;
            if (owner < 0 && before + part[i] > target) owner = lane * span + i, prefix = before;
          }
          before += part[i];
        }
        if (owner < 0) owner = last_owner, prefix = last_prefix;
        owner = __shfl_sync(0xffffffffu, owner, lane_of);
        goal = target - __shfl_sync(0xffffffffu, prefix, lane_of);
        here = some && owner == mine;
        if (!some && writer) tokens[count] = -1;
      }
      double passed = 0.;
      if (here) {   // its run once more: 256 logits at a time until the goal is passed
        int last_positive = -1, token = -1;
#pragma unroll 1
        for (int base = j0; base < j1 && token < 0; base += 32) {
          const int j = base + lane;
          double w[kVec] = {};
          if (j < j1) {
            const Vec<T> x = row.load(j);
            float y[kVec] = {};
            if (kDrawn && beta > 0.) row.load_probs(q, j, y);
            remaining(weigh, x, y, inv, kDrawn ? beta : 0., kDrawn && beta > 0. ? sh.stages[warp] : 0, w);
          }
          if (touched)
            each_kid([&](int out, double) {
              const int off = out - row.first(j);
#pragma unroll
              for (int i = 0; i < kVec; ++i)
                if (off == i) w[i] = 0.;
            });
          int last = -1;
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (w[i] > 0.) last = row.first(j) + i;
          const double sum = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])), through = warp_scan64(sum);
          const uint32_t there = __ballot_sync(0xffffffffu, last >= 0 && passed + through > goal), positive = __ballot_sync(0xffffffffu, last >= 0);
          if (there) {
            double run = passed + (through - sum);
            int found = last;   // (sums in another order may fall short of the goal by a rounding)
            bool done = false;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
              run += w[i];
              if (!done && w[i] > 0. && run > goal) found = row.first(j) + i, done = true;
            }
            token = __shfl_sync(0xffffffffu, found, __ffs(there) - 1);
          }
          if (positive) last_positive = __shfl_sync(0xffffffffu, last, 31 - __clz(positive));
          passed += __shfl_sync(0xffffffffu, through, 31);
        }
        if (!again && lane == 0) tokens[count] = token >= 0 ? token : last_positive;
      }
      if (!again) break;
      meet(touched ? passed : sh.sum[turn ^ 1][mine], 0);
      take_sums();
    }
    break;
  }
  if (rank == 0) {
    if (writer) a.counts[b] = count + 1;
    __syncthreads();
    for (int i = threadIdx.x; i < a.T; i += kThreads) {
      if (i != count) tokens[i] = i < count ? token_of[i] : -1;   // (the new token is stored by who found it)
      path[i] = i <= count ? node_of[i] : -1;
    }
  }
}

template <typename T, int kWarps, bool kDrawn>
int launch(const Args& a, const int C, cudaStream_t s) {
  auto bytes = [](int nodes) { return static_cast<int>(sizeof(Shared) + nodes * 44); };
  static SmemLimit limit;
  const cudaError_t e = limit.raise(verify_kernel<T, kWarps, kDrawn>, bytes(kMaxNodes));
  if (e != cudaSuccess) return set_error(OASR_ERR_CUDA, "verify_drafts: shared memory limit: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.B * C));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = bytes(a.T);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = g_pdl ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {static_cast<unsigned>(C), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, verify_kernel<T, kWarps, kDrawn>, a, C);
  return check_launch("verify_drafts launch");
}

template <typename T, bool kDrawn>
int launch(const Args& a, cudaStream_t s) {
  // Blocks of eight warps, two to an SM, and of a cluster as many as fit, as long as each has work for four of its warps.  Long rows of few sequences
  // take blocks of sixteen: every warp decides for itself, and more warps take longer for that (3 chains of 5 over 5002 tokens: 12.6 us with eight, 14.2
  // with sixteen; 32 drawn chains of 8 over 65537: 34.6, 36.7), but a row is walked through in fewer steps (16 trees of 48 over 131071: 21, 16).
  // Clusters of sixteen were no faster.
  const int sms = sm_count(), units = a.V / (32 * kVec);
  int C = 1;
  while (C < kMaxCluster && a.B * C <= sms && units > C * 4) C *= 2;
  if (units > 192 && a.B * kMaxCluster <= sms) return launch<T, 16, kDrawn>(a, C, s);
  return launch<T, 8, kDrawn>(a, C, s);
}

}  // namespace
}  // namespace verify
}  // namespace ob

extern "C" int oasr_b200_verify_drafts(int32_t* tokens, int32_t* path, int32_t* counts, const void* logits, int64_t logits_stride_b,
                                       int64_t logits_stride_n, const int32_t* drafts, const int32_t* parents, int64_t parents_stride,
                                       const float* uniforms, const float* draft_probs, int64_t probs_stride_b, int64_t probs_stride_n,
                                       const float* temperatures, double temperature, int64_t B, int64_t T, int64_t V, int dtype, void* stream) {
  using namespace ob;
  OB_REQUIRE(B >= 0 && T >= 0 && V > 0, OASR_ERR_INVALID, "verify_drafts: bad shape");
  OB_REQUIRE(T <= verify::kMaxNodes, OASR_ERR_UNSUPPORTED, "verify_drafts: trees of up to %d nodes (got %lld)", verify::kMaxNodes, (long long)T);
  OB_REQUIRE(B <= 0xffffff && V <= 0x7ffffff, OASR_ERR_INVALID, "verify_drafts: batch or vocabulary too large");
  if (B == 0 || T == 0) return OASR_OK;
  OB_REQUIRE(tokens && path && counts && logits && drafts && parents && uniforms, OASR_ERR_INVALID, "verify_drafts: null pointer argument");
  OB_REQUIRE(temperatures || std::isfinite(temperature), OASR_ERR_INVALID, "verify_drafts: the temperature must be a finite number");
  OB_REQUIRE(dtype == OASR_DT_F32 || dtype == OASR_DT_F16 || dtype == OASR_DT_BF16, OASR_ERR_DTYPE, "verify_drafts: unsupported dtype id %d", dtype);
  OB_REQUIRE(is_aligned(tokens, 4) && is_aligned(path, 4) && is_aligned(counts, 4) && is_aligned(logits, dtype == OASR_DT_F32 ? 4 : 2) && is_aligned(drafts, 4) &&
                 is_aligned(parents, 4) && is_aligned(uniforms, 4) && is_aligned(draft_probs, 4) && is_aligned(temperatures, 4),
             OASR_ERR_ALIGN, "verify_drafts: operands must be aligned to their elements");
  const verify::Args a{tokens, path, counts, logits, draft_probs, drafts, parents, uniforms, temperatures, logits_stride_b, logits_stride_n, probs_stride_b,
                       probs_stride_n, parents_stride, static_cast<int>(B), static_cast<int>(T), static_cast<int>(V), static_cast<float>(temperature), 1u << 12, 1u << 21};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return OB_DISPATCH_FLOAT(dtype, T_, [&]() -> int { return draft_probs ? verify::launch<T_, true>(a, st) : verify::launch<T_, false>(a, st); });
}
