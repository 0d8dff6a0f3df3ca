// k_sample_rows.cu -- one token per row of logits, every row with its own
// temperature, top-k, top-p, min-p and random number.
//
// With z = x / T, m the largest z and w = exp(z - m) a token is kept when
//   x >= the k-th largest x                         (top-k; equal ones stay)
//   sum of w over larger x < p * sum of w           (top-p, of what top-k left)
//   w >= min_p                                      (min-p)
// and the draw is the first index whose kept weights, added in index order,
// exceed u times their sum.  All three filters are a least x, so the row is
// read, the least x found, and the weights from it on added up.
#include "common.h"
#include "kv_dev.cuh"
#include "launch.h"
#include "sample_rows.h"

namespace rpgb {
namespace {

constexpr int kCluster = 8;     // blocks that share a row
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;
// Weights are added as integers of 2^-44 (at most 2^18 of them, each at most
// 1), so that no sum depends on its order.
constexpr double kFix = 17592186044416.0;

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

template <typename T>
struct Row {
  const T* x;   // this block's part, in shared memory
  int n;        // values of it
  __device__ __forceinline__ float operator[](int i) const { return kvd::ToFloat(x[i]); }
};

struct Shared {
  unsigned long long mass[kBins];
  unsigned count[kBins];
  unsigned long long all_mass[kBins];
  unsigned all_count[kBins];
  unsigned long long part[kWarps];
  unsigned long long sum;  // of the block's kept weights
  unsigned key[kWarps];
  int index[kWarps];
  unsigned top;     // key of the block's largest value
  int first;        // its lowest index
  uint32_t prefix;
};

// exp((x - m) / T), accurate to a few units of 2^-53.
__device__ __forceinline__ double Weight(float x, float top, double inv) {
  if (top == INFINITY) return x == INFINITY ? 1.0 : 0.0;
  return exp((static_cast<double>(x) - static_cast<double>(top)) * inv);
}

__device__ __forceinline__ unsigned long long Fixed(double w) {
  return static_cast<unsigned long long>(__double2ll_rn(w * kFix));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) SampleRowsKernel(const SampleRowsParams p, int per) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ Shared sh;
  T* vals = reinterpret_cast<T*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = ClusterRank();
  const int row = blockIdx.x / kCluster;
  dev::GridLaunchDependents();
  dev::GridWait();
  const int begin = min(static_cast<int>(rank) * per, p.vocab), n = min(per, p.vocab - begin);
  const T* src = static_cast<const T*>(p.logits) + row * p.stride + begin;
  const float temperature = p.temperature != nullptr ? p.temperature[row] : 1.f;
  const int top_k = p.top_k != nullptr ? p.top_k[row] : 0;
  const float top_p = p.top_p != nullptr ? p.top_p[row] : 1.f;
  const float min_p = p.min_p != nullptr ? p.min_p[row] : 0.f;

  // ---- the row's largest value and its lowest index
  unsigned best = 0;
  int at = INT_MAX;
  for (int i = tid; i < n; i += kThreads) {
    const T v = src[i];
    vals[i] = v;
    const unsigned k = Key(kvd::ToFloat(v));
    if (k > best) {
      best = k;
      at = i;
    }
  }
  {
    const unsigned w = __reduce_max_sync(0xFFFFFFFFu, best);
    const int i = __reduce_min_sync(0xFFFFFFFFu, best == w && w != 0 ? at : INT_MAX);
    if (lane == 0) {
      sh.key[warp] = w;
      sh.index[warp] = i;
    }
  }
  __syncthreads();
  if (tid == 0) {
    unsigned w = 0;
    int i = INT_MAX;
    for (int k = 0; k < kWarps; ++k) {
      if (sh.key[k] > w || (sh.key[k] == w && sh.index[k] < i)) {
        w = sh.key[k];
        i = sh.index[k];
      }
    }
    sh.top = w;
    sh.first = w != 0 ? begin + i : INT_MAX;
  }
  ClusterSync();
  unsigned top = 0;
  int first = INT_MAX;
  for (uint32_t b = 0; b < kCluster; ++b) {
    const unsigned w = *In(&sh.top, b);
    if (w > top) {
      top = w;
      first = *In(&sh.first, b);
    }
  }
  const bool greedy = !(temperature > 0.f);
  const Row<T> x{vals, n};
  const float most = FromKey(top);
  uint32_t least = 1;
  const double inv = greedy ? 1.0 : 1.0 / static_cast<double>(temperature);
  if (top != 0 && !greedy) {
    // ---- the least key that the filters leave, found eight bits at a time
    for (int pass = 0; pass < 2; ++pass) {
      const bool by_mass = pass == 1;
      if (by_mass ? !(top_p > 0.f && top_p < 1.f) : !(top_k > 1 && top_k < p.vocab)) continue;
      uint32_t prefix = 0;
      unsigned wanted = static_cast<unsigned>(top_k);
      unsigned long long over = 0, need = 0;  // mass above the prefix's range; mass that has to be reached
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < kBins; i += kThreads) {
          sh.mass[i] = 0;
          sh.count[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
          const uint32_t k = Key(x[i]);
          if (k == 0 || k < least || (shift < 24 && k >> (shift + 8) != prefix)) continue;
          const int bin = k >> shift & 255;
          if (by_mass) {
            atomicAdd(&sh.mass[bin], Fixed(Weight(x[i], most, inv)));
          } else {
            atomicAdd(&sh.count[bin], 1u);
          }
        }
        ClusterSync();
        for (int i = tid; i < kBins; i += kThreads) {
          unsigned long long m = 0;
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
          if (by_mass) {
            if (shift == 24) {
              unsigned long long total = 0;
              for (int i = 0; i < kBins; ++i) total += sh.all_mass[i];
              need = static_cast<unsigned long long>(ceil(static_cast<double>(top_p) * static_cast<double>(total)));
            }
            // the lowest bin above which there is less than `need`
            int bin = 255;
            while (bin > 0 && over + sh.all_mass[bin] < need) over += sh.all_mass[bin--];
            sh.prefix = prefix << 8 | static_cast<uint32_t>(bin);
          } else {
            int bin = 255;
            while (bin > 0 && sh.all_count[bin] < wanted) wanted -= sh.all_count[bin--];
            sh.prefix = prefix << 8 | static_cast<uint32_t>(bin);
          }
        }
        ClusterSync();  // (before the histograms are cleared too)
        prefix = sh.prefix;
      }
      least = max(least, prefix);
    }
  }
  // ---- the kept weights as integers, a run of values per thread in index order
  auto kept = [&](int i, double& w) -> unsigned long long {
    const float v = x[i];
    const uint32_t k = Key(v);
    if (k < least || k == 0) return 0;
    w = Weight(v, most, inv);
    return min_p > 0.f && w < static_cast<double>(min_p) ? 0 : Fixed(w);
  };
  const int run = (per + kThreads - 1) / kThreads;
  const int lo = min(tid * run, n), hi = min(lo + run, n);
  unsigned long long mine = 0;
  double w;
  if (top != 0 && !greedy) {
    for (int i = lo; i < hi; ++i) mine += kept(i, w);
  }
  unsigned long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.part[warp] = incl;
  __syncthreads();
  if (tid == 0) {
    unsigned long long s = 0;
    for (int k = 0; k < kWarps; ++k) s += sh.part[k];
    sh.sum = s;
  }
  ClusterSync();
  unsigned long long before = incl - mine, total = 0;
  for (uint32_t b = 0; b < kCluster; ++b) {
    const unsigned long long s = *In(&sh.sum, b);
    if (b < rank) before += s;
    total += s;
  }
  for (int k = 0; k < warp; ++k) before += sh.part[k];
  if (top == 0 || greedy) {
    if (rank == 0 && tid == 0) {
      p.tok[row] = top == 0 ? -1 : first;
      if (p.prob != nullptr) p.prob[row] = top == 0 ? kvd::Nan() : 1.f;
    }
  } else {
    // (the sums are integers: one thread, and one value, has the target)
    const double u = fmin(fmax(p.u != nullptr ? static_cast<double>(p.u[row]) : 0.0, 0.0), 1.0);
    const unsigned long long target = min(static_cast<unsigned long long>(u * static_cast<double>(total)), total - 1);
    if (before <= target && target < before + mine) {
      for (int i = lo; i < hi; ++i) {
        before += kept(i, w);
        if (target < before) {
          p.tok[row] = begin + i;
          if (p.prob != nullptr) p.prob[row] = static_cast<float>(w * kFix / static_cast<double>(total));
          break;
        }
      }
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
