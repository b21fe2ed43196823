// Log-probs of given tokens, entropy and top alternatives of every row of logits, in one pass over the logits.
//
//   lse = M + log S,  S = sum_j exp(x_j - M);   log p(t) = x_t - lse;   H = log S - (1 / S) sum_j (x_j - M) exp(x_j - M)
//   top k by (value, then lowest index)
//
// Sums run in fp32 and in the log2 domain, d_j = x_j log2(e) - m2 with m2 = M log2(e) rounded: one fused multiply-add a value.
// What the rounding of m2 shifts all of them by is taken out of the two sums afterwards.  Rows whose maximum is beyond 2^20 (a mask
// that leaves nothing, of whatever size) take d_j = (x_j - M) log2(e).
//
// A warp owns up to 32 * NV granules of 16 bytes of one row and holds them in registers: they are read from memory once, and the
// maximum, the sums and the selection all run on that copy.  Selection: the k-th largest of 64 to 128 maxima of parts of the row is a
// lower bound of its k-th largest value, so only what reaches it (a little over k values) goes to a list in shared memory, where
// every lane counts how many are above its own.  Where that is too many (a mask that leaves fewer than k tokens makes the bound the
// mask's value) the list takes what is above the bound, and the lowest indices of the bound's value fill it up.  A row whose list
// still overflows, or that holds a NaN, takes k rounds of a warp-wide maximum over the row instead; the result is the same.
// Larger rows are split over the warps of a block, and over a cluster of blocks where the rows are few: the parts' statistics
// and sorted lists meet in shared memory (the first block's, written through the cluster).
//
// Bound: instructions, not bytes (unpack, multiply-add, clamp, exp2 and two sums a logit).  One B200, bf16, device time of a call
// without and with 8 and 30 alternatives: 8000 rows of 5002 logits 25, 37 and 47 us (bytes alone 12), 2473 of 5876 18, 27 and 33
// us (4.4), 602 of 78300 37, 57 and 73 us (14), 16 of 5002 6, 8 and 10 us.
#include <type_traits>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ob {
namespace {

constexpr int kMaxTop = 32;
constexpr int kList = 192;          // candidates a row can hold
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kFar = -200.f;      // 2^-200 is zero in fp32: the exponent of a masked (-inf) logit, which keeps d * exp2(d) at zero

struct Args {
  float *log_probs, *entropy, *top_log_probs;
  int32_t* top_ids;
  const void *logits, *tokens;
  int64_t rows, stride;
  int vocab, num_tokens, top_k, tokens_i64;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order of the values as unsigned numbers; a NaN ranks above everything, and below all ones: no element's key is the one above
// all keys that a walk through them starts from.
constexpr uint32_t kNan = 0xfffffffeu;
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return kNan;
  const uint32_t b = __float_as_uint(x + 0.f);   // -0 ranks with +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  if (o == kNan) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// (value, lowest index first) as one unsigned number; 0 is below every element
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  return (static_cast<uint64_t>(ordered(x)) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ int index_of(uint64_t key) { return ~static_cast<int>(static_cast<uint32_t>(key)); }

__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& g, float (&x)[Elem<T>::kVec]) {
  const Pack<T> p = *reinterpret_cast<const Pack<T>*>(&g);
#pragma unroll
  for (int i = 0; i < Elem<T>::kVec; ++i) x[i] = Elem<T>::to_f(p.v[i]);
}

template <typename T>
__device__ __forceinline__ float granule_max(const uint4& g) {
  if constexpr (sizeof(T) == 4) {
    return max_nan(max_nan(__uint_as_float(g.x), __uint_as_float(g.y)), max_nan(__uint_as_float(g.z), __uint_as_float(g.w)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2* h = reinterpret_cast<const __half2*>(&g);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&g);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
}

struct Stats {
  float m, s, w;   // maximum (-inf: nothing there), sum of exp2(d), sum of d exp2(d) with d = (x - m) log2(e)
};

__device__ __forceinline__ Stats merge(Stats a, Stats b) {
  Stats r;
  r.m = max_nan(a.m, b.m);
  if (r.m == -INFINITY) return Stats{-INFINITY, 0.f, 0.f};
  // a part whose weight is zero (empty, or that far below) has no say, whatever its distance
  const float da = (a.m - r.m) * kLog2e, db = (b.m - r.m) * kLog2e;
  const float fa = ex2(da), fb = ex2(db);
  r.s = r.w = 0.f;
  if (fa != 0.f) r.s = a.s * fa, r.w = fa * fmaf(da, a.s, a.w);
  if (fb != 0.f) r.s = fmaf(b.s, fb, r.s), r.w = fmaf(fb, fmaf(db, b.s, b.w), r.w);
  return r;
}

// N statistics, lane l's being number l % N.  A merge rounds by the order of its arguments, so that lanes could end a bit apart: all
// get the first lane's, and with it a token the same log-prob wherever it is asked for.
template <int N>
__device__ __forceinline__ Stats warp_merge(Stats v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    Stats b;
    b.m = __shfl_xor_sync(0xffffffffu, v.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, v.w, o);
    v = merge(v, b);
  }
  return Stats{__shfl_sync(0xffffffffu, v.m, 0), __shfl_sync(0xffffffffu, v.s, 0), __shfl_sync(0xffffffffu, v.w, 0)};
}

template <int W, int kRows>
struct Shared {
  uint64_t list[kRows][kList];          // candidates
  int granule[kRows][kList];            // granules they are in (a warp to a row)
  uint64_t sorted[W * kRows][kMaxTop];  // a warp's alternatives
  uint64_t merged[kMaxTop];
  int count, nan;
  Stats stats[W];
  alignas(16) uint32_t maxima[128];     // of parts of the block's slice
  uint32_t bound;                       // the k-th largest of them
  // written by the other blocks of the cluster, read by the first
  uint64_t part_sorted[8][kMaxTop];
  Stats part_stats[8];
};

// The k largest of `found` (>= k) keys, in order: a key's place is the number of keys above it.
__device__ __forceinline__ void rank_list(const uint64_t* list, int found, int k, uint64_t* out, int lane) {
  for (int base = lane; base < found; base += 64) {
    const uint64_t k0 = list[base], k1 = base + 32 < found ? list[base + 32] : 0;
    int above0 = 0, above1 = 0;
#pragma unroll 4
    for (int i = 0; i < found; ++i) {
      const uint64_t o = list[i];
      above0 += o > k0;
      above1 += o > k1;
    }
    if (above0 < k) out[above0] = k0;
    if (base + 32 < found && above1 < k) out[above1] = k1;
  }
}

// k rounds over `lists` sorted lists of k keys each (lane l walks list l); the result is sorted into `out`.
__device__ __forceinline__ void merge_lists(const uint64_t (*lists)[kMaxTop], int n, int k, uint64_t* out, int lane) {
  int at = 0;
  uint64_t head = lane < n ? lists[lane][0] : 0;
  for (int r = 0; r < k; ++r) {
    const uint64_t best = warp_max_key(head);
    if (lane == 0) out[r] = best;
    if (head == best && best != 0) head = ++at < k ? lists[lane][at] : 0;
  }
}

// W warps of a block share a row's slice; `parts` blocks of a cluster share a row.  Small blocks are held to registers of which
// five (seven) fit a SM: loads of one then run under the arithmetic of the others (602 rows of 78300: 55 us at three, 45 at four).
template <typename T, int W, int NV>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32, W > 4 ? 1 : NV <= 5 ? 7 : NV <= 10 ? 5 : 4) token_log_probs_kernel(const Args a, const int parts) {
  constexpr int VE = Elem<T>::kVec;
  constexpr int kRows = W == 1 ? 4 : 1;                 // rows of a block
  __shared__ Shared<W, kRows> sh;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // waited for before the first remote write
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = W == 1 ? 0 : static_cast<int>(blockIdx.x % parts);
  const int64_t row = W == 1 ? static_cast<int64_t>(blockIdx.x) * kRows + warp : blockIdx.x / parts;
  if (W == 1 && row >= a.rows) return;
  const T* x0 = static_cast<const T*>(a.logits) + row * a.stride;
  // The row is `head` elements up to a 16-byte boundary, whole granules, and a tail; head and tail (fewer than 2 VE elements) lie
  // one to a lane in the first warp, so that every other load is a granule without a branch.
  const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) % 16 / sizeof(T)), a.vocab);
  const int granules = (a.vocab - head) / VE;
  const int first = W == 1 ? lane : part * W * 32 + threadIdx.x;
  const int step = W == 1 ? 32 : parts * W * 32;
  const T* x1 = x0 + head;

  uint4 g[NV];
  const uint32_t low = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;   // -inf
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int gi = first + i * step;
    g[i] = make_uint4(low, low, low, low);
    if (gi < granules) g[i] = *reinterpret_cast<const uint4*>(ld128_stream(x1 + gi * VE).v);
  }
  const bool has_edge = first < a.vocab - granules * VE;
  const int edge_at = first < head ? first : first + granules * VE;
  const float edge = has_edge ? Elem<T>::to_f(x0[edge_at]) : -INFINITY;

  // ---- maximum and sums of the warp's part
  float max0 = max_nan(edge, granule_max<T>(g[0])), max1 = -INFINITY;
#pragma unroll
  for (int i = 1; i < NV; ++i) (i & 1 ? max1 : max0) = max_nan(i & 1 ? max1 : max0, granule_max<T>(g[i]));
  const float lane_max = max_nan(max0, max1);
  float m = lane_max;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  // Exponents d_j = (x_j - m) log2(e).  Rows up to 2^20 form them with one multiply-add, x_j log2(e) - m2, and what the rounding of
  // m2 shifts all of them by (2^-4 at most) is taken out of the sums.  That shift grows with |m| (2^-24 of it) until the sums overflow
  // or vanish, so that larger rows subtract first: exactly where the two are within a factor of two, and to below kFar where they are not.
  const bool large = !(fabsf(m) <= 0x1p20f);
  const float base = m == -INFINITY ? 0.f : m, m2 = base * kLog2e;
  float s = 0.f, w = 0.f;
  auto sums = [&](auto exponent) {
    const float edge_d = max_nan(exponent(edge), kFar);
    // four sums of each: shorter chains, and the likeliest token's 1 costs fewer of the small terms their last bits
    float s4[4] = {ex2(edge_d)}, w4[4] = {edge_d * s4[0]};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[VE];
      unpack<T>(g[i], x);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float d = max_nan(exponent(x[j]), kFar);
        const float e = ex2(d);
        s4[j & 3] += e;
        w4[j & 3] = fmaf(d, e, w4[j & 3]);
      }
    }
    s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    w = (w4[0] + w4[1]) + (w4[2] + w4[3]);
  };
  if (large) sums([&](float x) { return (x - base) * kLog2e; });
  else sums([&](float x) { return fmaf(x, kLog2e, -m2); });
  s = warp_sum(s);
  w = warp_sum(w);
  if (!large) {
    const float shift = fmaf(m, kLog2e, -m2), f = ex2(-shift);   // m2 + shift is m log2(e)
    w = fmaf(-shift, s, w) * f;
    s *= f;
  }
  Stats st{m, s, w};

  // ---- the k largest
  const int k = a.top_k;
  uint64_t* const list = sh.list[W == 1 ? warp : 0];
  const uint32_t below = (1u << lane) - 1;
  // entries `found` to k - 1 of the list: the lowest indices in [lo, hi) whose logit is v
  auto fill = [&](int lo, int hi, float v, int found) {
    for (int base = lo; base < hi && found < k; base += 32) {
      const int j = base + lane;
      const bool hit = j < hi && Elem<T>::to_f(x0[min(j, hi - 1)]) == v;
      const uint32_t all = __ballot_sync(0xffffffffu, hit);
      const int at = found + __popc(all & below);
      if (hit && at < k) list[at] = key_of(v, j);
      found = min(found + __popc(all), k);
    }
    return found;
  };
  // rounds over the warp's part of the row, from memory again (a copy in the caches): rare, and without a limit on equal values
  auto rounds = [&](uint64_t* out) {
    uint64_t last = ~0ull;   // above every key
    for (int r = 0; r < k; ++r) {
      uint64_t best = 0;
      if (has_edge && key_of(edge, edge_at) < last) best = key_of(edge, edge_at);
      for (int gi = first; gi < granules; gi += step) {
        for (int e = 0; e < VE; ++e) {
          const uint64_t c = key_of(Elem<T>::to_f(x1[gi * VE + e]), head + gi * VE + e);
          if (c < last) best = max(best, c);
        }
      }
      last = warp_max_key(best);
      if (lane == 0) out[r] = last;
    }
  };
  const uint64_t* sorted = nullptr;
  if constexpr (W == 1) {
    sorted = sh.sorted[warp];
    if (k > 0) {
      int found = kList + 1;
      if (m == m) {
        // k-th largest of the lanes' two maxima each
        uint32_t cur = ordered(fmaxf(max0, max1)), next = ordered(fminf(max0, max1)), top = 0;
        for (int n = 0; n < k;) {
          top = __reduce_max_sync(0xffffffffu, cur);
          n += __popc(__ballot_sync(0xffffffffu, cur == top));
          if (cur == top) cur = next, next = 0;
        }
        const float bound = from_ordered(top);
        bool over = bound == -INFINITY;                                   // take what is above the bound, not all that reaches it
#pragma unroll 1
        for (int pass = over; pass < 2 && found > kList; ++pass) {
          over = pass == 1;
          const float threshold = over ? from_ordered(top + 1) : bound;   // (NaN behind +inf: nothing)
          // what reaches it: first the granules, then, a granule to a lane, the values.  The granules are read again (from the
          // caches): picking them out of registers would take the whole warp through each.
          int* const hits = sh.granule[warp];
          int n = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            asm("" : "+r"(g[i].x), "+r"(g[i].y), "+r"(g[i].z), "+r"(g[i].w));   // not kept unpacked from the sums until here
            const bool hit = granule_max<T>(g[i]) >= threshold;
            const uint32_t all = __ballot_sync(0xffffffffu, hit);
            const int at = n + __popc(all & below);
            if (hit && at < kList) hits[at] = first + i * step;
            n += __popc(all);
          }
          __syncwarp();
          found = 0;
          auto take = [&](bool hit, float x, int index) {
            const uint32_t all = __ballot_sync(0xffffffffu, hit);
            const int at = found + __popc(all & below);
            if (hit && at < kList) list[at] = key_of(x, index);
            found += __popc(all);
          };
          take(edge >= threshold, edge, edge_at);
          for (int base = 0; base < min(n, kList); base += 32) {
            const bool any = base + lane < min(n, kList);
            const int gi = any ? hits[base + lane] : first;
            Pack<T> again;
            if (any) again = ld128(x1 + gi * VE);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
              const float x = any ? Elem<T>::to_f(again.v[j]) : -INFINITY;
              take(x >= threshold, x, head + gi * VE + j);
            }
          }
          if (n > kList) found = kList + 1;
          __syncwarp();
        }
        if (over && found < k) {
          found = fill(0, a.vocab, bound, found);
          __syncwarp();
        }
      }
      if (found <= kList) rank_list(list, found, k, sh.sorted[warp], lane);
      else rounds(sh.sorted[warp]);
      __syncwarp();
    }
  } else {
    constexpr int kGroup = W == 16 ? 4 : 2, kMaxima = W * 32 / kGroup;   // lanes behind a maximum; 128 or 64 of them
    float gm = lane_max;
#pragma unroll
    for (int o = 1; o < kGroup; o <<= 1) gm = max_nan(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    if (lane % kGroup == 0) sh.maxima[(warp * 32 + lane) / kGroup] = ordered(gm);
    if (lane == 0) sh.stats[warp] = st;
    if (threadIdx.x == 0) sh.count = sh.nan = 0;
    __syncthreads();
    if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp == 0) st = warp_merge<W>(sh.stats[lane % W]);   // the block's
    if (k > 0) {
      if (threadIdx.x < kMaxima) {   // the k-th largest maximum; several threads write the same number if it is there more often
        const uint32_t mine = sh.maxima[threadIdx.x];
        int above = 0, reach = 0;
#pragma unroll 4
        for (int i = 0; i < kMaxima; i += 4) {
          const uint4 o = *reinterpret_cast<const uint4*>(&sh.maxima[i]);
          above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
          reach += (o.x >= mine) + (o.y >= mine) + (o.z >= mine) + (o.w >= mine);
        }
        if (above < k && reach >= k) sh.bound = mine;
        if (mine == kNan) sh.nan = 1;
      }
      __syncthreads();
      const uint32_t top = sh.bound;
      const float bound = from_ordered(top);
      bool over = bound == -INFINITY;                                   // take what is above the bound, not all that reaches it
      int found = kList + 1;
#pragma unroll 1
      for (int pass = over; pass < 2 && !sh.nan; ++pass) {
        over = pass == 1;
        const float threshold = over ? from_ordered(top + 1) : bound;   // (NaN behind +inf: nothing)
        auto take = [&](float x, int index) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kList) list[at] = key_of(x, index);
        };
        if (edge >= threshold) take(edge, edge_at);
        uint32_t reach = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          asm("" : "+r"(g[i].x), "+r"(g[i].y), "+r"(g[i].z), "+r"(g[i].w));   // not kept unpacked from the sums until here
          if (granule_max<T>(g[i]) >= threshold) reach |= 1u << i;
        }
        while (reach) {   // few, at places of their own in every lane: read again (from the caches)
          const int gi = first + (__ffs(reach) - 1) * step;
          reach &= reach - 1;
          const Pack<T> again = ld128(x1 + gi * VE);
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const float x = Elem<T>::to_f(again.v[j]);
            if (x >= threshold) take(x, head + gi * VE + j);
          }
        }
        __syncthreads();
        found = sh.count;
        if (found <= kList || over) break;
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
      }
      if (found <= kList) {
        if (warp == 0) {
          if (over && found < k) {
            if (part == 0) found = fill(0, head, bound, found);
            for (int gi = part * W * 32; gi < granules && found < k; gi += step) {
              found = fill(head + gi * VE, head + min(gi + W * 32, granules) * VE, bound, found);
            }
            if (part == 0) found = fill(head + granules * VE, a.vocab, bound, found);
            if (lane >= found && lane < k) sh.merged[lane] = 0;         // a part of fewer than k
            __syncwarp();
          }
          rank_list(list, found, k, sh.merged, lane);
        }
      } else {
        rounds(sh.sorted[warp]);
        __syncthreads();
        if (warp == 0) merge_lists(sh.sorted, W, k, sh.merged, lane);
      }
    }
    if (warp == 0) __syncwarp();
    if (parts > 1) {
      if (warp == 0) {   // into the first block's shared memory
        if (lane < k) {
          const uint32_t to = ptx::map_to_cta(&sh.part_sorted[part][lane], 0);
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(sh.merged[lane]) : "memory");
        }
        if (lane < 3) {
          const float v = lane == 0 ? st.m : lane == 1 ? st.s : st.w;
          const uint32_t to = ptx::map_to_cta(reinterpret_cast<float*>(&sh.part_stats[part]) + lane, 0);
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
        }
      }
      ptx::cluster_sync();
      if (part != 0) return;
      if (warp == 0) {
        st = warp_merge<8>(lane % 8 < parts ? sh.part_stats[lane % 8] : Stats{-INFINITY, 0.f, 0.f});
        if (k > 0) merge_lists(sh.part_sorted, parts, k, sh.merged, lane);
        __syncwarp();
      }
    }
    if (warp != 0) return;
    sorted = sh.merged;
  }
  const bool none = st.m == -INFINITY;             // a row of -inf: every log-prob is -inf, the entropy 0
  const float log_s = logf(st.s);
  auto log_prob = [&](float x) { return none ? -INFINITY : (x - st.m) - log_s; };
  if (a.entropy && lane == 0) a.entropy[row] = none ? 0.f : fmaf(-kLn2, st.w / st.s, log_s);
  for (int j = lane; j < a.num_tokens; j += 32) {
    const int64_t at = row * a.num_tokens + j;
    const int64_t t = a.tokens_i64 ? static_cast<const int64_t*>(a.tokens)[at] : static_cast<const int32_t*>(a.tokens)[at];
    a.log_probs[at] = t >= 0 && t < a.vocab ? log_prob(Elem<T>::to_f(x0[t])) : 0.f;   // padding scores nothing
  }
  if (lane < k) {
    const uint64_t key = sorted[lane];
    a.top_ids[row * k + lane] = index_of(key);
    a.top_log_probs[row * k + lane] = log_prob(from_ordered(static_cast<uint32_t>(key >> 32)));
  }
}

template <typename T, int W, int NV>
int launch(const Args& a, int parts, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  const int64_t blocks = W == 1 ? (a.rows + 3) / 4 : a.rows * parts;
  OB_REQUIRE(blocks <= 0x7fffffff, OASR_ERR_INVALID, "token_log_probs: too many rows for one call");
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(W == 1 ? 128 : W * 32);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = g_pdl ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, token_log_probs_kernel<T, W, NV>, a, parts);
  return check_launch("token_log_probs launch");
}

template <typename T>
int run(const Args& a, cudaStream_t s) {
  constexpr int VE = Elem<T>::kVec;
  const int64_t granules = a.vocab / VE;   // at most
  const int64_t sms = sm_count();
  // many rows: a warp each, without a block's barriers (8000 of 5002 bf16: 25 us, 35 with four warps a row)
  if (a.rows >= sms * 4 && granules <= 32 * 20) {
    if (granules <= 32 * 5) return launch<T, 1, 5>(a, 1, s);
    if (granules <= 32 * 10) return launch<T, 1, 10>(a, 1, s);
    return launch<T, 1, 20>(a, 1, s);
  }
  if (granules <= 128 * 5) return launch<T, 4, 5>(a, 1, s);
  // still more blocks than stay on the SMs at once: four warps, and for long rows clusters of such (602 rows of 78300 bf16: 37 us; 65 in
  // clusters of 16 warps)
  if (a.rows >= sms * 2 && granules <= 128 * 7) return launch<T, 4, 7>(a, 1, s);
  if (a.rows >= sms * 2 && granules <= 128 * 10 * 8) return launch<T, 4, 10>(a, static_cast<int>((granules + 1279) / 1280), s);
  int parts = 1;   // few rows: a cluster each
  while (parts < 8 && (a.rows * parts < sms || granules > 512 * 16 * parts) && granules > 512 * parts) parts *= 2;
  const int64_t per = (granules + 512 * parts - 1) / (512 * parts);
  if (per <= 2) return launch<T, 16, 2>(a, parts, s);
  if (per <= 4) return launch<T, 16, 4>(a, parts, s);
  if (per <= 8) return launch<T, 16, 8>(a, parts, s);
  return launch<T, 16, 16>(a, parts, s);
}

}  // namespace
}  // namespace ob

extern "C" int oasr_b200_token_log_probs(float* log_probs, float* entropy, float* top_log_probs, int32_t* top_ids, const void* logits,
                                         const void* tokens, int tokens_i64, int64_t rows, int64_t vocab, int64_t stride,
                                         int64_t num_tokens, int64_t top_k, int dtype, void* stream) {
  using namespace ob;
  OB_REQUIRE(rows >= 0 && vocab > 0 && num_tokens >= 0 && top_k >= 0, OASR_ERR_INVALID, "token_log_probs: bad shape");
  OB_REQUIRE(vocab <= 262144, OASR_ERR_UNSUPPORTED, "token_log_probs: at most 262144 tokens in the vocabulary (got %lld)", (long long)vocab);
  OB_REQUIRE(stride >= vocab || rows <= 1, OASR_ERR_INVALID, "token_log_probs: rows of %lld logits %lld apart", (long long)vocab, (long long)stride);
  OB_REQUIRE(top_k <= kMaxTop && top_k <= vocab, OASR_ERR_INVALID, "token_log_probs: top_k must be at most %d and the vocabulary (got %lld)",
             kMaxTop, (long long)top_k);
  if (rows == 0) return OASR_OK;
  OB_REQUIRE(logits && (num_tokens == 0 || (tokens && log_probs)) && (top_k == 0 || (top_log_probs && top_ids)), OASR_ERR_INVALID,
             "token_log_probs: null pointer argument");
  OB_REQUIRE(num_tokens <= 0x7fffffff, OASR_ERR_INVALID, "token_log_probs: too many tokens a row");
  const Args a{log_probs, entropy, top_log_probs, top_ids, logits, tokens, rows, stride, static_cast<int>(vocab), static_cast<int>(num_tokens),
               static_cast<int>(top_k), tokens_i64};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return OB_DISPATCH_FLOAT(dtype, T_, [&]() -> int {
    OB_REQUIRE(is_aligned(logits, sizeof(T_)), OASR_ERR_ALIGN, "token_log_probs: logits must be aligned to their type");
    return run<T_>(a, s);
  });
}
