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
// The answer is whole numbers, so what decides is computed in 64 bits: weights e^(l / temperature) to some 1e-13, their sums in a fixed order.
// They come out of a table of 2^(i / 256) and a polynomial of degree 3 for the rest (the method of Tang, "Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic", 1989).  Weights are taken relative to logits of 0: 64 bits reach 2^250 above and 2^500 below; rows
// that lie elsewhere are taken again relative to their maximum.
// p and q unnormalised: with k children rejected  p_k = max(p - beta_k q, 0) / Pi_k,  Pi_k the sum of the numerators, beta_1 = 1 and
// beta_{k+1} = beta_k + Pi_k.  With q = 1 at x a rejection takes x's weight out of the sum.
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

constexpr int kWarps = 16, kMaxCluster = 8, kTable = 256, kMaxNodes = 1024;

struct Args {
  int32_t *tokens, *path, *counts;
  const void* logits;
  const float* probs;
  const int32_t *drafts, *parents;
  const float *uniforms, *temperatures;
  int64_t ls_b, ls_n, ps_b, ps_n, parents_b;   // strides: logits, draft probabilities, parents of a sequence (0: one tree for all)
  int B, T, V;
  float temperature;
};

struct Kid {
  int node, token;
  float logit, u, q;
};

// What the blocks of a cluster tell one another about a row, a number and a whole number of each warp, and the children of the node.
// Two of each in turn: a barrier lies between a use and the next writing of the same one.
struct Shared {
  double table[kTable];
  double sum[2][kMaxCluster * kWarps];
  int id[2][kMaxCluster * kWarps];
  int kid_count[2];
};

struct Weigher {
  const double* table;
  double rate, ref;   // 256 log2(e) / temperature; weights are relative to e^(ref / temperature)
  float lo, hi;       // logits below are weights of zero, logits above are out of range

  __device__ __forceinline__ void relative_to(float r) {
    ref = r;
    lo = static_cast<float>(fmax(ref - 500. * kTable / rate, static_cast<double>(-FLT_MAX)));   // rounded away from ref by at most as much again
    hi = static_cast<float>(fmin(ref + 250. * kTable / rate, static_cast<double>(FLT_MAX)));
  }
  // e^((l - ref) / temperature)
  __device__ __forceinline__ double operator()(float l) const {
    constexpr double kMagic = 6755399441055744.;   // 1.5 * 2^52: the sum's low word is the rounded number
    constexpr double c1 = 0.6931471805599453 / kTable, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
    if (!(l >= lo)) return 0.;
    const double d = static_cast<double>(fminf(l, hi)) - ref;
    const double t = fma(d, rate, kMagic);
    const int k = __double2loint(t);
    const double f = fma(d, rate, -(t - kMagic));   // in [-1/2, 1/2]
    const double v = table[k & (kTable - 1)], g = fma(fma(f, c3, c2), f, c1);
    const double w = fma(v * f, g, v);
    return __hiloint2double(__double2hiint(w) + ((k >> 8) << 20), __double2loint(w));
  }
};
static_assert(kTable == 256, "the exponent is what is above 8 bits");

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row of logits in vectors of 16 bytes that start at their own boundary: vector j has tokens first(j) .. first(j) + kVec - 1, those
// outside [0, V) at -inf.
template <typename T>
struct Row {
  static constexpr int kVec = Elem<T>::kVec;
  const T* p;
  int V, skew;
  __device__ __forceinline__ Row(const T* p_, int V_) : p(p_), V(V_), skew(static_cast<int>(reinterpret_cast<uintptr_t>(p_) % 16 / sizeof(T))) {}
  __device__ __forceinline__ int vectors() const { return (V + skew + kVec - 1) / kVec; }
  __device__ __forceinline__ int first(int j) const { return j * kVec - skew; }
  __device__ __forceinline__ void load(int j, float (&x)[kVec]) const {
    const int v0 = first(j);
    if (v0 >= 0 && v0 + kVec <= V) {
      const Pack<T> v = ld128(p + v0);
#pragma unroll
      for (int i = 0; i < kVec; ++i) x[i] = Elem<T>::to_f(v.v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) x[i] = v0 + i >= 0 && v0 + i < V ? Elem<T>::to_f(p[v0 + i]) : -INFINITY;
    }
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
};

template <typename T>
__global__ void __launch_bounds__(kWarps * 32, 1) verify_kernel(const Args a, const int C) {
  constexpr int kVec = Elem<T>::kVec;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  int* const parents = reinterpret_cast<int*>(smem + sizeof(Shared));
  Kid* const all_kids = reinterpret_cast<Kid*>(parents + a.T);   // two lists of up to T
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = C > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0, b = static_cast<int>(blockIdx.x) / C;
  for (int i = threadIdx.x; i < kTable; i += kWarps * 32) sh.table[i] = exp2(i * (1. / kTable));
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  for (int i = threadIdx.x; i < a.T; i += kWarps * 32) parents[i] = a.parents[b * a.parents_b + i];
  const float temperature = a.temperatures ? a.temperatures[b] : a.temperature;
  const bool greedy = !(temperature > 0.f);
  const int slots = C * kWarps, mine = rank * kWarps + warp;
  const float* const u = a.uniforms + static_cast<int64_t>(b) * a.T;
  const int32_t* const drafts = a.drafts + static_cast<int64_t>(b) * a.T;
  int32_t* const tokens = a.tokens + static_cast<int64_t>(b) * a.T;
  int32_t* const path = a.path + static_cast<int64_t>(b) * a.T;
  const bool writer = rank == 0 && threadIdx.x == 0;
  __syncthreads();
  if (C > 1) ptx::cluster_sync();   // every block of the cluster runs: its shared memory may be written

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
    double s = 0.;
    for (int i = lane; i < slots; i += 32) s += sh.sum[turn ^ 1][i];
    return warp_sum64(s);
  };
  auto any_flag = [&]() {
    int f = 0;
    for (int i = lane; i < slots; i += 32) f |= sh.id[turn ^ 1][i];
    return __any_sync(0xffffffffu, f != 0);
  };

  int n = 0, count = 0, token = -1, kid_turn = 0;
  if (writer) path[0] = 0;
  Weigher weigh{sh.table, kTable * 1.4426950408889634 / static_cast<double>(temperature), 0., 0.f, 0.f};
  for (;;) {
    const Row<T> row(static_cast<const T*>(a.logits) + b * a.ls_b + n * a.ls_n, a.V);
    const float* const q = a.probs ? a.probs + b * a.ps_b + n * a.ps_n : nullptr;
    const int per = (row.vectors() + slots - 1) / slots, j0 = min(mine * per, row.vectors()), j1 = min(j0 + per, row.vectors());
    Kid* const kids = all_kids + kid_turn * a.T;
    if (warp == 0) {   // the node's children that are tokens
      int found = 0;
      for (int i0 = (n + 1) & ~31; i0 < a.T; i0 += 32) {
        const int i = i0 + lane;
        int x = -1;
        if (i > n && i < a.T && parents[i] == n) x = drafts[i];
        const bool is = x >= 0 && x < a.V;
        const uint32_t m = __ballot_sync(0xffffffffu, is);
        if (is) kids[found + __popc(m & ((1u << lane) - 1))] = Kid{i, x, Elem<T>::to_f(row.p[x]), u[i], q ? q[x] : 1.f};
        found += __popc(m);
      }
      if (lane == 0) sh.kid_count[kid_turn] = found;
    }

    // the row's largest logit, its first token, and whether there is a NaN
    auto largest = [&](float& best, int& at) {
      best = -INFINITY, at = 0x7fffffff;
      bool bad = false;
      for (int j = j0 + lane; j < j1; j += 32) {
        float x[kVec];
        row.load(j, x);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          bad |= x[i] != x[i];
          if (x[i] > best) best = x[i], at = row.first(j) + i;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, best, o);
        const int w = __shfl_xor_sync(0xffffffffu, at, o);
        if (v > best || (v == best && w < at)) best = v, at = w;
      }
      bad = __any_sync(0xffffffffu, bad);
      meet(static_cast<double>(bad ? NAN : best), at);
      best = -INFINITY, at = 0x7fffffff, bad = false;
      for (int i = lane; i < slots; i += 32) {
        const float v = static_cast<float>(sh.sum[turn ^ 1][i]);
        const int w = sh.id[turn ^ 1][i];
        bad |= v != v;
        if (v > best || (v == best && w < at)) best = v, at = w;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, best, o);
        const int w = __shfl_xor_sync(0xffffffffu, at, o);
        if (v > best || (v == best && w < at)) best = v, at = w;
      }
      return !__any_sync(0xffffffffu, bad) && fabsf(best) < INFINITY;   // there is a distribution
    };

    int accepted = -1, accepted_token = 0;
    if (greedy) {
      float best;
      int at;
      const bool fine = largest(best, at);
      const int kid_count = sh.kid_count[kid_turn];
      double beta = 0.;   // q = draft probabilities: p is 1 at `at`, what is left of it after k rejections max(1 - beta q(at), 0)
      double left = 1.;   // (of Pi_k; the other tokens have nothing at any time)
      const float q_at = fine && q ? q[at] : 1.f;
      for (int k = 0; fine && k < kid_count && accepted < 0; ++k) {
        const Kid kid = kids[k];
        if (kid.token == at && static_cast<double>(kid.u) * kid.q * (beta > 0. ? left : 1.) < left) {
          accepted = kid.node, accepted_token = kid.token;
        } else if (q) {
          beta = beta > 0. ? beta + left : 1.;
          left = fmax(1. - beta * q_at, 0.);
        } else if (kid.token == at) {
          left = 0.;
        }
      }
      if (accepted < 0) {
        token = fine && left > 0. ? at : -1;
        if (writer) tokens[count] = token;
        break;
      }
    } else {
      // ---- weights of the row
      auto weigh_all = [&](bool& over) {
        double s0 = 0., s1 = 0.;
        bool out = false;
        for (int j = j0 + lane; j < j1; j += 32) {
          float x[kVec];
          row.load(j, x);
#pragma unroll
          for (int i = 0; i < kVec; i += 2) {
            out |= !(x[i] <= weigh.hi) || !(x[i + 1] <= weigh.hi);
            s0 += weigh(x[i]);
            s1 += weigh(x[i + 1]);
          }
        }
        out = __any_sync(0xffffffffu, out);
        meet(warp_sum64(s0 + s1), out);
        over = any_flag();
        return sum_all();
      };
      bool over, fine = true;
      weigh.relative_to(0.f);
      double total = weigh_all(over);
      if (over || !(total >= 0x1p-200)) {   // the row does not lie around zero
        float best;
        int at;
        fine = largest(best, at);
        if (fine) {
          weigh.relative_to(best);
          total = weigh_all(over);
        }
      }
      const int kid_count = sh.kid_count[kid_turn];
      double rest = total, beta = 0., inv = 1.;
      // (q) sum of max(p - beta q, 0) over the vocabulary
      auto residue = [&]() {
        double s = 0.;
        for (int j = j0 + lane; j < j1; j += 32) {
          float x[kVec], y[kVec];
          row.load(j, x);
          row.load_probs(q, j, y);
#pragma unroll
          for (int i = 0; i < kVec; ++i) s += fmax(fma(weigh(x[i]), inv, -beta * static_cast<double>(y[i])), 0.);
        }
        meet(warp_sum64(s), 0);
        return sum_all();
      };
      auto repeated = [&](int k) {   // an earlier child had the same token
        bool same = false;
        for (int i = lane; i < k; i += 32) same |= kids[i].token == kids[k].token;
        return __any_sync(0xffffffffu, same);
      };
      for (int k = 0; fine && k < kid_count && accepted < 0; ++k) {
        const Kid kid = kids[k];
        double w = weigh(kid.logit);
        if (q) {
          if (beta > 0.) w = fmax(fma(w, inv, -beta * static_cast<double>(kid.q)), 0.);
        } else if (repeated(k)) {
          continue;
        }
        if (static_cast<double>(kid.u) * static_cast<double>(kid.q) * rest < w) {
          accepted = kid.node, accepted_token = kid.token;
        } else if (q) {
          inv = 1. / total;
          beta = beta > 0. ? beta + rest : 1.;
          rest = residue();
        } else {
          rest = fmax(rest - w, 0.);
        }
      }
      if (accepted < 0) {
        // ---- the token behind the path
        const int turn_read = turn ^ 1, span = (slots + 31) / 32;   // a lane's warps: their order is the vocabulary's
        const bool without = !q && fine;
        double part[kMaxCluster * kWarps / 32];
        double lane_sum = 0.;
#pragma unroll
        for (int i = 0; i < kMaxCluster * kWarps / 32; ++i) part[i] = i < span && lane * span + i < slots ? sh.sum[turn_read][lane * span + i] : 0.;
        for (int k = 0; without && k < kid_count; ++k) {
          if (repeated(k)) continue;
          const int owner = (kids[k].token + row.skew) / kVec / per;
          const double w = weigh(kids[k].logit);
#pragma unroll
          for (int i = 0; i < kMaxCluster * kWarps / 32; ++i)
            if (owner == lane * span + i && i < span) part[i] = fmax(part[i] - w, 0.);
        }
#pragma unroll
        for (int i = 0; i < kMaxCluster * kWarps / 32; ++i) lane_sum += part[i];
        double upto = lane_sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const double all = __shfl_sync(0xffffffffu, upto, 31), target = static_cast<double>(u[0]) * all;
        // the first warp whose cumulative sum passes the target, else the last one with something in it
        const uint32_t past = __ballot_sync(0xffffffffu, lane_sum > 0. && upto > target), some = __ballot_sync(0xffffffffu, lane_sum > 0.);
        const int lane_of = past ? __ffs(past) - 1 : 31 - __clz(some | 1u);
        double before = upto - lane_sum, prefix = 0.;
        int owner = -1, last_owner = -1;
        double last_prefix = 0.;
#pragma unroll
        for (int i = 0; i < kMaxCluster * kWarps / 32; ++i) {
          if (part[i] > 0.) {
            last_owner = lane * span + i, last_prefix = before;
            if (owner < 0 && before + part[i] > target) owner = lane * span + i, prefix = before;
          }
          before += part[i];
        }
        if (owner < 0) owner = last_owner, prefix = last_prefix;
        owner = __shfl_sync(0xffffffffu, owner, lane_of);
        prefix = __shfl_sync(0xffffffffu, prefix, lane_of);
        if (!fine || !some) {
          if (writer) tokens[count] = -1;
        } else if (owner == mine) {
          const double goal = target - prefix;
          double passed = 0.;
          int last_positive = -1;
          token = -1;
          for (int j = j0; j < j1 && token < 0; j += 32) {
            float x[kVec], y[kVec];
            double w[kVec], s = 0.;
            int last = -1;
            const bool in = j + lane < j1;
            if (in) row.load(j + lane, x);
            if (in && beta > 0.) row.load_probs(q, j + lane, y);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
              w[i] = in ? weigh(x[i]) : 0.;
              if (in && beta > 0.) w[i] = fmax(fma(w[i], inv, -beta * static_cast<double>(y[i])), 0.);
            }
            if (without) {
              for (int k = 0; k < kid_count; ++k) {
                const int off = kids[k].token - row.first(j + lane);
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                  if (off == i) w[i] = 0.;
              }
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
              s += w[i];
              if (w[i] > 0.) last = row.first(j + lane) + i;
            }
            double upto_here = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double v = __shfl_up_sync(0xffffffffu, upto_here, o);
              if (lane >= o) upto_here += v;
            }
            const uint32_t over_goal = __ballot_sync(0xffffffffu, last >= 0 && passed + upto_here > goal);
            if (over_goal) {
              double run = passed + (upto_here - s);
              int mine_token = last;   // (sums in another order may fall short of the goal by a rounding)
              bool done = false;
#pragma unroll
              for (int i = 0; i < kVec; ++i) {
                run += w[i];
                if (!done && w[i] > 0. && run > goal) mine_token = row.first(j + lane) + i, done = true;
              }
              token = __shfl_sync(0xffffffffu, mine_token, __ffs(over_goal) - 1);
            }
            const uint32_t positive = __ballot_sync(0xffffffffu, last >= 0);
            if (positive) last_positive = __shfl_sync(0xffffffffu, last, 31 - __clz(positive));
            passed += __shfl_sync(0xffffffffu, upto_here, 31);
          }
          if (lane == 0) tokens[count] = token >= 0 ? token : last_positive;
        }
        break;
      }
    }
    if (writer) tokens[count] = accepted_token, path[count + 1] = accepted;
    ++count;
    n = accepted;
    kid_turn ^= 1;
  }
  if (writer) a.counts[b] = count + 1;
  if (rank == 0)
    for (int i = count + 1 + threadIdx.x; i < a.T; i += kWarps * 32) tokens[i] = -1, path[i] = -1;
}

template <typename T>
int launch(const Args& a, cudaStream_t s) {
  // Blocks of a cluster: as many as there are SMs for, as long as each warp has two vectors a lane.
  int C = 1;
  while (C < kMaxCluster && a.B * C * 2 <= sm_count() && a.V > C * kWarps * 64 * Elem<T>::kVec) C *= 2;
  auto bytes = [](int nodes) { return static_cast<int>(sizeof(Shared) + nodes * (4 + 2 * sizeof(Kid))); };
  static SmemLimit limit;
  const cudaError_t e = limit.raise(verify_kernel<T>, bytes(kMaxNodes));
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
  cudaLaunchKernelEx(&cfg, verify_kernel<T>, a, C);
  return check_launch("verify_drafts launch");
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
                       probs_stride_n, parents_stride, static_cast<int>(B), static_cast<int>(T), static_cast<int>(V), static_cast<float>(temperature)};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return OB_DISPATCH_FLOAT(dtype, T_, [&]() -> int { return verify::launch<T_>(a, st); });
}
