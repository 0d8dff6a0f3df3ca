// k_sample_rows.cu -- one token per row of logits, every row with its own
// temperature, top-k, top-p, min-p and random number.
//
// With z = x / T, m the largest z and w = exp(z - m) a token is kept when
//   x >= the k-th largest x                         (top-k; equal ones stay)
//   sum of w over larger x < p * sum of w           (top-p, of what top-k left)
//   w >= min_p                                      (min-p)
// and the draw is the first index whose kept weights, added in index order,
// exceed u times their sum.  All three filters are a least x.
//
// What it has to do is read the logits once.  A cluster of eight blocks holds a
// row in shared memory; what follows is the row's largest value, then
//  * with top-k or top-p: the largest value of each of the cluster's 4096
//    threads bounds the K-th largest from below, so the few values from that
//    bound on are gathered in the first block, sorted, cut and drawn from there;
//  * where that list does not hold what the filters leave (a flat row and a
//    large top-p, very many equal values, a large k): the least x by selection,
//    eight bits at a time, over counts (top-k) or sums of weights (top-p);
//  * then, and without these filters at once, the weights of all that is left
//    are added up, the warp that has the target in its share is found from the
//    blocks' and warps' sums, and it finds the token.
// A draw compares u with sums of up to 2^18 terms, so weights are held to 2^-42
// in f64 and added as integers of 2^-44: no sum depends on its order.
#include "common.h"
#include "kv_dev.cuh"
#include "launch.h"
#include "sample_rows.h"

namespace rpgb {
namespace {

using u64 = unsigned long long;

constexpr int kCluster = 8;  // blocks that share a row
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = 1024;      // values that the first block sorts
constexpr int kMostK = 512;      // the largest k that the list is tried for
constexpr int kFirst = 384;      // the K of rows with top-p alone
constexpr double kFix = 17592186044416.0;  // 2^44

__device__ __forceinline__ void ClusterSync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t ClusterRank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of `p` in the shared memory of block `rank`.
template <typename T>
__device__ __forceinline__ T* In(T* p, uint32_t rank) {
  uint64_t r;
  asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<T*>(r);
}

// Floats in order as integers; NaN and minus infinity (never drawn) as 0.
__device__ __forceinline__ uint32_t Key(float x) {
  const uint32_t u = __float_as_uint(x);
  const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return x > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float FromKey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

struct Shared {
  double power[256];  // 2^(j / 256)
  union {
    struct {
      u64 mass[kBins], all_mass[kBins];
      unsigned count[kBins], all_count[kBins];
      unsigned thread_top[kThreads];
    };
    struct {
      u64 list[kList], weight[kList];  // key and the complement of the index; weights in the list's order
    };
  };
  u64 mine[kList / 4];  // what this block found for the list
  u64 part[kWarps], sum, target;
  unsigned wide[kWarps], top, n_mine, n_all;
  int first;
  uint32_t least;
  int found;
};

// exp((x - top) / T) as 2^y with y = n + j / 256 + r: 2^(j / 256) from a table
// and 2^r (|r| <= 2^-9) by its series to the third power, whose next term is
// under 2^-42.
struct Weights {
  const double* power;
  double top, c;
  __device__ __forceinline__ Weights(const Shared& sh, float top_, float temperature)
      : power(sh.power), top(static_cast<double>(top_)), c(1.4426950408889634 / static_cast<double>(temperature)) {}
  __device__ __forceinline__ double operator()(float x) const {
    const double y = (static_cast<double>(x) - top) * c;
    if (!(y >= -60.0)) return x == INFINITY ? 1.0 : 0.0;  // (under 2^-45; infinities are each other's equals)
    constexpr double kMagic = 6755399441055744.0 / 256.0;  // 1.5 2^52 in units of 1 / 256
    const double t = y + kMagic;
    const double r = y - (t - kMagic);
    const int n = __double2loint(t);
    double q = fma(r, 0.055504108664821580, 0.24022650695910072);
    q = fma(r, q, 0.69314718055994531) * r;
    const double p = power[n & 255];
    const double w = fma(p, q, p);
    return __hiloint2double(__double2hiint(w) + ((n >> 8) << 20), __double2loint(w));
  }
};
__device__ __forceinline__ u64 Fixed(double w) { return static_cast<u64>(__double2ll_rn(w * kFix)); }

__device__ __forceinline__ u64 WarpAdd(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ u64 WarpScan(u64 v, int lane) {  // with the lane's own
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 w = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

// Sorts n (a power of two from 2) keys, the largest first.
__device__ __forceinline__ void Sort(u64* x, int n) {
  for (int k = 2; k <= n; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 u = x[a], v = x[b];
        if ((u < v) == ((a & k) == 0)) {
          x[a] = v;
          x[b] = u;
        }
      }
      __syncthreads();
    }
  }
}

// `u` of a sum of weights: the target is exceeded by exactly one token's running sum.
__device__ __forceinline__ u64 Target(const SampleRowsParams& p, int row, u64 total) {
  const double u = fmin(fmax(p.u != nullptr ? static_cast<double>(p.u[row]) : 0.0, 0.0), 1.0);
  return min(static_cast<u64>(u * static_cast<double>(total)), total - 1);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) SampleRowsKernel(const SampleRowsParams p, int per) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ Shared sh;
  T* vals = reinterpret_cast<T*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = ClusterRank();
  const int row = blockIdx.x / kCluster;
  if (tid < 256) sh.power[tid] = exp2(tid / 256.0);
  if (tid == 0) sh.n_mine = 0;
  dev::GridLaunchDependents();
  dev::GridWait();
  const int begin = min(static_cast<int>(rank) * per, p.vocab), n = min(per, p.vocab - begin);
  const T* src = static_cast<const T*>(p.logits) + row * p.stride + begin;
  const float temperature = p.temperature != nullptr ? p.temperature[row] : 1.f;
  const int top_k = p.top_k != nullptr ? p.top_k[row] : 0;
  const float top_p = p.top_p != nullptr ? p.top_p[row] : 1.f;
  const float min_p = p.min_p != nullptr ? p.min_p[row] : 0.f;
  const bool greedy = !(temperature > 0.f);
  const bool by_k = !greedy && top_k > 1 && top_k < p.vocab, by_p = !greedy && top_p > 0.f && top_p < 1.f;

  // ---- the row into shared memory, and its largest value
  float best = -INFINITY;
  constexpr int kVec = 16 / sizeof(T);
  if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    const int vecs = n / kVec;
    constexpr int kFlight = 4;
    for (int i0 = tid; i0 < vecs; i0 += kThreads * kFlight) {
      uint4 w[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        if (i0 + k * kThreads < vecs) w[k] = reinterpret_cast<const uint4*>(src)[i0 + k * kThreads];
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        if (i0 + k * kThreads < vecs) {
          reinterpret_cast<uint4*>(vals)[i0 + k * kThreads] = w[k];
          const kvd::Pack<T, kVec> x = *reinterpret_cast<const kvd::Pack<T, kVec>*>(&w[k]);
#pragma unroll
          for (int e = 0; e < kVec; ++e) best = fmaxf(best, kvd::ToFloat(x.v[e]));
        }
      }
    }
    for (int i = vecs * kVec + tid; i < n; i += kThreads) {
      vals[i] = src[i];
      best = fmaxf(best, kvd::ToFloat(vals[i]));
    }
  } else {
    constexpr int kFlight = 8;
    for (int i0 = tid; i0 < n; i0 += kThreads * kFlight) {
      T w[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        if (i0 + k * kThreads < n) w[k] = src[i0 + k * kThreads];
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        if (i0 + k * kThreads < n) {
          vals[i0 + k * kThreads] = w[k];
          best = fmaxf(best, kvd::ToFloat(w[k]));
        }
      }
    }
  }
  const unsigned my_key = Key(best);
  sh.thread_top[tid] = my_key;
  {
    const unsigned w = __reduce_max_sync(0xFFFFFFFFu, my_key);
    if (lane == 0) sh.wide[warp] = w;
  }
  __syncthreads();
  if (tid == 0) {
    unsigned w = 0;
    for (int k = 0; k < kWarps; ++k) w = max(w, sh.wide[k]);
    sh.top = w;
  }
  ClusterSync();
  unsigned top = 0;
  for (uint32_t b = 0; b < kCluster; ++b) top = max(top, *In(&sh.top, b));
  const float most = FromKey(top);

  if (top == 0 || greedy) {
    // ---- nothing to draw, or the largest value's lowest index
    int at = INT_MAX;
    if (top != 0 && sh.top == top) {
      for (int i = tid; i < n; i += kThreads) {
        if (Key(kvd::ToFloat(vals[i])) == top) {
          at = begin + i;
          break;
        }
      }
    }
    at = __reduce_min_sync(0xFFFFFFFFu, at);
    __syncthreads();
    if (lane == 0) sh.wide[warp] = static_cast<unsigned>(at);
    __syncthreads();
    if (tid == 0) {
      for (int k = 0; k < kWarps; ++k) at = min(at, static_cast<int>(sh.wide[k]));
      sh.first = at;
    }
    ClusterSync();
    if (rank == 0 && tid == 0) {
      for (uint32_t b = 1; b < kCluster; ++b) at = min(at, *In(&sh.first, b));
      p.tok[row] = top == 0 ? -1 : at;
      if (p.prob != nullptr) p.prob[row] = top == 0 ? kvd::Nan() : 1.f;
    }
    ClusterSync();
    return;
  }

  const Weights weigh(sh, most, temperature);
  uint32_t least_min = 1, cut = 1;
  if (min_p > 0.f && min_p <= 1.f) {
    // under x = top + T log(min_p), less a part in 2^20 of both, no weight reaches min_p; kept() decides the rest
    const float cut = most + temperature * logf(min_p);
    const float low = cut - (fabsf(most) + fabsf(temperature * logf(min_p))) * 9.5367431640625e-7f;
    if (low > -INFINITY && most < INFINITY) least_min = max(1u, Key(low));
  }
  // the weight of a value, 0 where a filter drops it
  auto kept = [&](float v, double& w) -> u64 {
    const uint32_t k = Key(v);
    if (k < least_min || k < cut) return 0;
    w = weigh(v);
    return min_p > 0.f && min_p <= 1.f && w < static_cast<double>(min_p) ? 0 : Fixed(w);
  };

  if (by_k || by_p) {
    // ---- a bound that at least `want` values reach: the want-th largest of the threads' values (its upper 22 bits)
    const int want = by_k ? min(top_k, kMostK + 1) : kFirst;
    bool listed = want <= kMostK;
    uint32_t bound = 0;
    if (listed) {
      unsigned key[kCluster];
#pragma unroll
      for (uint32_t b = 0; b < kCluster; ++b) key[b] = In(sh.thread_top, b)[tid];
      for (int bit = 31; bit >= 10; --bit) {
        const uint32_t try_ = bound | 1u << bit;
        int c = 0;
#pragma unroll
        for (int b = 0; b < kCluster; ++b) c += key[b] >= try_;
        c = __reduce_add_sync(0xFFFFFFFFu, c);
        if (lane == 0) sh.wide[warp] = c;
        __syncthreads();
        int all = lane < kWarps ? static_cast<int>(sh.wide[lane]) : 0;
        all = __reduce_add_sync(0xFFFFFFFFu, all);
        if (all >= want) bound = try_;
        __syncthreads();
      }
      bound = max(bound, 1u);
    }
    // ---- what reaches it, and the sum of all weights where the list may not hold all that counts
    u64 mass = 0;
    for (int i0 = warp * 32; i0 < n; i0 += kThreads) {
      const int i = i0 + lane;
      const uint32_t k = i < n ? Key(kvd::ToFloat(vals[i])) : 0;
      if (!by_k && k != 0) mass += Fixed(weigh(kvd::ToFloat(vals[i])));
      const bool in = listed && k >= bound;
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, in);
      if (mask != 0) {
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(&sh.n_mine, __popc(mask));
        at = __shfl_sync(0xFFFFFFFFu, at, 0) + __popc(mask & ((1u << lane) - 1));
        if (in && at < kList / 4) sh.mine[at] = static_cast<u64>(k) << 32 | ~static_cast<uint32_t>(begin + i);
      }
    }
    mass = WarpAdd(mass);
    if (lane == 0) sh.part[warp] = mass;
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int k = 0; k < kWarps; ++k) s += sh.part[k];
      sh.sum = s;
    }
    ClusterSync();
    if (rank == 0) {
      // ---- the first block sorts the list, cuts it and draws
      unsigned start[kCluster + 1];
      bool fits = listed;
      u64 total = 0;
      start[0] = 0;
      for (uint32_t b = 0; b < kCluster; ++b) {
        const unsigned c = *In(&sh.n_mine, b);
        fits = fits && c <= kList / 4;
        start[b + 1] = start[b] + c;
        total += *In(&sh.sum, b);
      }
      const int m = static_cast<int>(start[kCluster]);
      fits = fits && m <= kList;
      if (tid == 0) sh.found = 0;
      if (fits) {
        int size = 64;
        while (size < m) size <<= 1;
        for (uint32_t b = 0; b < kCluster; ++b) {
          for (int i = tid; i < static_cast<int>(start[b + 1] - start[b]); i += kThreads) sh.list[start[b] + i] = In(sh.mine, b)[i];
        }
        for (int i = m + tid; i < size; i += kThreads) sh.list[i] = 0;
        __syncthreads();
        Sort(sh.list, size);
        const uint32_t least_k = by_k ? static_cast<uint32_t>(sh.list[top_k - 1] >> 32) : 1;
        // weights of the values from least_k on, and their running sums: two values a thread
        u64 w0 = 0, w1 = 0;
        const int i = 2 * tid;
        if (i < m && static_cast<uint32_t>(sh.list[i] >> 32) >= least_k) w0 = Fixed(weigh(FromKey(sh.list[i] >> 32)));
        if (i + 1 < m && static_cast<uint32_t>(sh.list[i + 1] >> 32) >= least_k) {
          w1 = Fixed(weigh(FromKey(sh.list[i + 1] >> 32)));
        }
        u64 incl = WarpScan(w0 + w1, lane);
        if (lane == 31) sh.part[warp] = incl;
        __syncthreads();
        u64 before = 0, sum = 0;
        for (int k = 0; k < kWarps; ++k) {
          if (k < warp) before += sh.part[k];
          sum += sh.part[k];
        }
        incl += before;
        if (by_k) total = sum;
        // the first value with which the sum reaches its share is the last of the kept
        const u64 need = by_p ? static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(total))) : ~0ull;
        if (tid == 0) sh.least = by_p ? 0 : least_k;
        __syncthreads();
        const u64 e0 = incl - w0 - w1, e1 = incl - w1;
        if (w0 > 0 && e0 < need && need <= e0 + w0) sh.least = static_cast<uint32_t>(sh.list[i] >> 32);
        if (w1 > 0 && e1 < need && need <= e1 + w1) sh.least = static_cast<uint32_t>(sh.list[i + 1] >> 32);
        __syncthreads();
        // (0 where the list does not reach the share; with top-k it holds all that counts)
        if (sh.least != 0) {
          cut = sh.least;
          // the kept, in the list's order
          double d0 = 0.0, d1 = 0.0;
          w0 = i < m ? kept(FromKey(sh.list[i] >> 32), d0) : 0;
          w1 = i + 1 < m ? kept(FromKey(sh.list[i + 1] >> 32), d1) : 0;
          sh.weight[i] = w0;
          sh.weight[i + 1] = w1;
          const u64 s = WarpAdd(w0 + w1);
          const int last = __reduce_max_sync(0xFFFFFFFFu, w1 > 0 ? i + 2 : (w0 > 0 ? i + 1 : 0));
          if (lane == 0) {
            sh.part[warp] = s;
            sh.wide[warp] = static_cast<unsigned>(last);
          }
          __syncthreads();
          total = 0;
          int count = 0;
          for (int k = 0; k < kWarps; ++k) {
            total += sh.part[k];
            count = max(count, static_cast<int>(sh.wide[k]));
          }
          const u64 target = Target(p, row, total);
          // what comes before a token by its index
          for (int k = tid; k < count; k += kThreads) {
            const uint32_t index = ~static_cast<uint32_t>(sh.list[k]);
            const u64 own = sh.weight[k];
            u64 sum_before = 0;
            for (int j = 0; j < count; ++j) sum_before += ~static_cast<uint32_t>(sh.list[j]) < index ? sh.weight[j] : 0;
            if (sum_before <= target && target - sum_before < own) {
              p.tok[row] = static_cast<int>(index);
              if (p.prob != nullptr) {
                p.prob[row] = static_cast<float>(weigh(FromKey(sh.list[k] >> 32)) * kFix / static_cast<double>(total));
              }
            }
          }
          if (tid == 0) sh.found = 1;
        }
      }
    }
    ClusterSync();
    const bool found = *In(&sh.found, 0) != 0;
    ClusterSync();  // (it has been read: the first block may end, or go on to use its memory)
    if (found) return;

    // ---- the least key that the filters leave, eight bits at a time
    for (int pass = 0; pass < 2; ++pass) {
      const bool by_mass = pass == 1;
      if (by_mass ? !by_p : !by_k) continue;
      uint32_t prefix = 0;
      unsigned wanted = static_cast<unsigned>(top_k);
      u64 over = 0, need = 0;  // the mass above the prefix's range; the mass that has to be reached
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < kBins; i += kThreads) {
          sh.mass[i] = 0;
          sh.count[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
          const float v = kvd::ToFloat(vals[i]);
          const uint32_t k = Key(v);
          if (k < cut || (shift < 24 && k >> (shift + 8) != prefix)) continue;
          const int bin = k >> shift & 255;
          if (by_mass) {
            atomicAdd(&sh.mass[bin], Fixed(weigh(v)));
          } else {
            atomicAdd(&sh.count[bin], 1u);
          }
        }
        ClusterSync();
        for (int i = tid; i < kBins; i += kThreads) {
          u64 m = 0;
          unsigned c = 0;
          for (uint32_t b = 0; b < kCluster; ++b) {
            m += *In(&sh.mass[i], b);
            c += *In(&sh.count[i], b);
          }
          sh.all_mass[i] = m;
          sh.all_count[i] = c;
        }
        __syncthreads();
        if (tid == 0) {
          int bin = 255;
          if (by_mass) {
            if (shift == 24) {
              u64 total = 0;
              for (int i = 0; i < kBins; ++i) total += sh.all_mass[i];
              need = static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(total)));
            }
            // the lowest bin above which there is less than `need`
            while (bin > 0 && over + sh.all_mass[bin] < need) over += sh.all_mass[bin--];
          } else {
            while (bin > 0 && sh.all_count[bin] < wanted) wanted -= sh.all_count[bin--];
          }
          sh.least = prefix << 8 | static_cast<uint32_t>(bin);
        }
        ClusterSync();  // (before the histograms are cleared too)
        prefix = sh.least;
      }
      cut = max(cut, prefix);  // (min-p does not count for the share)
    }
  }

  // ---- the kept weights: a run of the row for each warp
  const int run = (per + kThreads - 1) / kThreads, lo = min(warp * 32 * run, n), hi = min(lo + 32 * run, n);
  double w = 0.0;
  u64 mine = 0;
  for (int i = lo + lane; i < hi; i += 32) mine += kept(kvd::ToFloat(vals[i]), w);
  mine = WarpAdd(mine);
  if (lane == 0) sh.part[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    u64 s = 0;
    for (int k = 0; k < kWarps; ++k) s += sh.part[k];
    sh.sum = s;
  }
  ClusterSync();
  u64 before = 0, total = 0;
  for (uint32_t b = 0; b < kCluster; ++b) {
    const u64 s = *In(&sh.sum, b);
    if (b < rank) before += s;
    total += s;
  }
  for (int k = 0; k < warp; ++k) before += sh.part[k];
  const u64 target = Target(p, row, total);
  if (before <= target && target - before < mine) {
    // this warp has it: a run for each lane, then the values of that run
    u64 own = 0;
    const int a = min(lo + lane * run, hi), b = min(a + run, hi);
    for (int i = a; i < b; ++i) own += kept(kvd::ToFloat(vals[i]), w);
    const u64 excl = WarpScan(own, lane) - own + before;
    const int who = __ffs(__ballot_sync(0xFFFFFFFFu, excl <= target && target - excl < own)) - 1;
    const int a1 = __shfl_sync(0xFFFFFFFFu, a, who), b1 = __shfl_sync(0xFFFFFFFFu, b, who);
    u64 so_far = __shfl_sync(0xFFFFFFFFu, excl, who);
    for (int i0 = a1; i0 < b1; i0 += 32) {
      const int i = i0 + lane;
      const u64 v = i < b1 ? kept(kvd::ToFloat(vals[i]), w) : 0;
      const u64 incl = so_far + WarpScan(v, lane);
      if (incl - v <= target && target < incl) {
        p.tok[row] = begin + i;
        if (p.prob != nullptr) p.prob[row] = static_cast<float>(w * kFix / static_cast<double>(total));
      }
      so_far = __shfl_sync(0xFFFFFFFFu, incl, 31);
    }
  }
  ClusterSync();  // no block ends while another reads its sums
}

template <typename T>
void Launch(const SampleRowsParams& p, cudaStream_t s) {
  const int per = ((p.vocab + kCluster - 1) / kCluster + 15) / 16 * 16;
  const size_t smem = static_cast<size_t>(per) * sizeof(T);
  const void* fn = reinterpret_cast<const void*>(SampleRowsKernel<T>);
  RPGB_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 << 10));
  LaunchKernelClusterArgs(fn, dim3(static_cast<unsigned>(p.n_rows) * kCluster), dim3(kThreads), smem, s, true, kCluster, p,
                          per);
}

}  // namespace

void LaunchSampleRows(const SampleRowsParams& p, cudaStream_t s) {
  switch (p.type) {
    case ElemType::kF32: Launch<float>(p, s); break;
    case ElemType::kF16: Launch<__half>(p, s); break;
    case ElemType::kBF16: Launch<__nv_bfloat16>(p, s); break;
  }
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

}  // namespace rpgb
