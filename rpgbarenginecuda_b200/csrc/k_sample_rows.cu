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
//    bound on are gathered in the first block, sorted and cut, and drawn from
//    there where few are left;
//  * where that list does not hold what the filters leave (a flat row and a
//    large top-p, very many equal values, a large k): the least x by selection,
//    ten bits of its distance from the largest at a time, over counts (top-k) or
//    sums of weights (top-p);
//  * then, and without these filters at once, the weights of all that is left
//    are added up, the warp that has the target in its share is found from the
//    blocks' and warps' sums, and it finds the token.
// A draw compares u with sums of up to 2^18 terms, so weights are held to 2^-34,
// and sums of them that are compared are integers of 2^-44.
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
constexpr int kBins = 1024, kBinBits = 10;
constexpr int kGroups = 512;     // of eight threads
constexpr int kList = 2048;      // values that the first block sorts
constexpr int kFew = 128;        // kept values that the first block draws from itself
constexpr int kMostK = 1280;     // the largest k that the list is tried for
constexpr int kFirst = 384;      // the K of rows with top-p alone
constexpr double kFix = 17592186044416.0;  // 2^44

__device__ __forceinline__ void ClusterSync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The two halves of it: this block has read what it needs of the others; no
// other block needs this one's memory any more.
__device__ __forceinline__ void ClusterArrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void ClusterWait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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

// Floats in order as integers, the two zeros the same; NaN and minus infinity (never drawn) as 0.
__device__ __forceinline__ uint32_t Key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return x > -INFINITY ? k : 0u;
}
constexpr uint32_t kLowest = 0x00800000u;  // of the lowest finite value
__device__ __forceinline__ float FromKey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

struct Shared {
  float2 power[256];  // 2^(j / 256)
  union {
    unsigned thread_top[kThreads];
    struct {
      // sums of weights in three parts of 15 bits, which 2^15 terms (a block's share) do not overflow
      int part[3][kBins];
      u64 all[kBins / kCluster];  // of all blocks, this block's bins
    } bins;
    u64 list[kList];  // key and the complement of the index
  };
  u64 mine[kList / 4];  // what this block found for the list
  u64 weight[kFew];
  u64 wsum[kWarps], sum, over, listed;
  alignas(16) unsigned group_top[kGroups / kCluster];
  unsigned wide[2 * kWarps], top, n_mine;
  int first;
  uint32_t least, most;
  int found;
};

// Weights exp((x - top) / T) = 2^y as pairs of f32, hi + lo, good to about
// 2^-34 (f64 to the same end took twice the time): x - top and its product with
// c = log2(e) / T carry their rounding errors along, y = n + j / 256 + r, 2^(j /
// 256) comes from a table of pairs and 2^r (|r| <= 2^-9) from its series to the
// third power, whose next term is under 2^-42.  Two values at a time.
struct Weights {
  const float2* power;
  float top, c, c_low;
  bool infinite;  // the largest value is: its equals count alike, nothing else does
  __device__ __forceinline__ Weights(const Shared& sh, float top_, float temperature) : power(sh.power), top(top_) {
    const double cc = fmin(1.4426950408889634 / static_cast<double>(temperature), 3e38);
    c = static_cast<float>(cc);
    c_low = static_cast<float>(cc - static_cast<double>(c));
    infinite = top == INFINITY;
  }
  static __device__ __forceinline__ float2 Two(float x) { return make_float2(x, x); }
  __device__ __forceinline__ void operator()(float2 x, float2& hi, float2& lo) const {
    if (infinite) {
      hi = make_float2(x.x == INFINITY ? 1.f : 0.f, x.y == INFINITY ? 1.f : 0.f);
      lo = Two(0.f);
      return;
    }
    const float2 less = Two(-1.f);
    const float2 d = __fadd2_rn(x, Two(-top));
    const float2 b = __ffma2_rn(x, less, d);                                                   // d - x
    const float2 e = __fadd2_rn(__ffma2_rn(__ffma2_rn(b, less, d), less, x), __ffma2_rn(b, less, Two(-top)));  // what d lost
    const float2 y = __fmul2_rn(d, Two(c));
    float2 z = __ffma2_rn(d, Two(-c), y);  // y less what it should be
    z = __ffma2_rn(d, Two(-c_low), z);
    z = __ffma2_rn(e, Two(-c), z);
    constexpr float kMagic = 12582912.f;  // 1.5 2^23
    const float2 t = __ffma2_rn(y, Two(256.f), Two(kMagic));
    const float2 n = __fadd2_rn(t, Two(-kMagic));
    const float2 r = __ffma2_rn(z, less, __ffma2_rn(n, Two(-0.00390625f), y));
    // (ln 2, its square over 2 and cube over 6; the first is off by 1.9e-9 as f32, which r makes 2^-38)
    float2 q = __ffma2_rn(r, Two(0.055504109f), Two(0.24022651f));
    q = __fmul2_rn(__ffma2_rn(r, q, Two(0.69314718f)), r);
    const uint32_t tx = __float_as_uint(t.x), ty = __float_as_uint(t.y);
    const float2 px = power[tx & 255], py = power[ty & 255];
    const float2 scale = make_float2(__uint_as_float((tx << 15 & 0xFF800000u) + 0x3F800000u),
                                     __uint_as_float((ty << 15 & 0xFF800000u) + 0x3F800000u));
    hi = __fmul2_rn(make_float2(px.x, py.x), scale);
    lo = __fmul2_rn(__ffma2_rn(make_float2(px.x, py.x), q, make_float2(px.y, py.y)), scale);
    if (!(y.x >= -60.f)) hi.x = lo.x = 0.f;  // (NaN too)
    if (!(y.y >= -60.f)) hi.y = lo.y = 0.f;
  }
  __device__ __forceinline__ double operator()(float x) const {
    float2 hi, lo;
    (*this)(Two(x), hi, lo);
    return static_cast<double>(hi.x) + static_cast<double>(lo.x);
  }
  __device__ __forceinline__ u64 Fixed(float x) const { return ToFixed((*this)(x)); }
  // times 2^44, to the nearest integer
  static __device__ __forceinline__ u64 ToFixed(double w) {
    return static_cast<u64>(__double_as_longlong(fma(w, kFix, 4503599627370496.0)) - 0x4330000000000000ll);
  }
  // The same as a 2^30 + b 2^15 + c, b and c within 2^14 of 0, by f32 operations.
  static __device__ __forceinline__ void ToParts(float hi, float lo, int& a, int& b, int& c) {
    constexpr float kMagic = 12582912.f;
    constexpr int kBits = 0x4B400000;
    const float h = hi * 16384.f, t = h + kMagic;
    a = __float_as_int(t) - kBits;
    const float r = fmaf(lo, 536870912.f, (h - (t - kMagic)) * 32768.f), u = r + kMagic;
    b = __float_as_int(u) - kBits;
    c = __float_as_int(fmaf(r - (u - kMagic), 32768.f, kMagic)) - kBits;
  }
  // How far x lies under the largest value, in units of 2^-25 of a factor 2 of
  // weight; what is farther than 2^-31 counts as alike.  Larger values are never farther.
  __device__ __forceinline__ uint32_t Distance(float x) const {
    const float d = (top - x) * c;
    return x == top ? 0u : (d < 31.f ? static_cast<uint32_t>(d * 33554432.f) : 0x3FFFFFFFu);
  }
};
// A running sum of weights: f32 with what its additions lose.
struct Sum {
  float2 hi = make_float2(0.f, 0.f), lo = make_float2(0.f, 0.f);
  __device__ __forceinline__ void Add(float2 h, float2 l) {
    const float2 less = make_float2(-1.f, -1.f), s = __fadd2_rn(hi, h), b = __ffma2_rn(hi, less, s);
    lo = __fadd2_rn(lo, __fadd2_rn(l, __fadd2_rn(__ffma2_rn(__ffma2_rn(b, less, s), less, hi), __ffma2_rn(b, less, h))));
    hi = s;
  }
  __device__ __forceinline__ double Total() const {
    return (static_cast<double>(hi.x) + static_cast<double>(hi.y)) + (static_cast<double>(lo.x) + static_cast<double>(lo.y));
  }
};

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

// Sorts n (a power of two from 64) keys, the largest first.  Up to 128 one warp
// does it without barriers for all.
__device__ __forceinline__ void Sort(u64* x, int n) {
  const bool small = n <= 128;
  const int threads = small ? 32 : kThreads;
  if (threadIdx.x < threads) {
#pragma unroll 1
    for (int k = 2; k <= n; k <<= 1) {
#pragma unroll 1
      for (int j = k >> 1; j > 0; j >>= 1) {
#pragma unroll 1
        for (int i = threadIdx.x; i < n / 2; i += threads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 u = x[a], v = x[b];
          if ((u < v) == ((a & k) == 0)) {
            x[a] = v;
            x[b] = u;
          }
        }
        small ? __syncwarp() : __syncthreads();
      }
    }
  }
  __syncthreads();
}

// What all blocks have found (m in all) into the first block's list, filled up
// to a power of two, which it returns.
__device__ __forceinline__ int Gather(Shared& sh, int m) {
  int size = 64;
  while (size < m) size <<= 1;
  int to = 0;
#pragma unroll 1
  for (uint32_t b = 0; b < kCluster; ++b) {
    const int c = static_cast<int>(*In(&sh.n_mine, b));
    for (int i = threadIdx.x; i < c; i += kThreads) sh.list[to + i] = In(sh.mine, b)[i];
    to += c;
  }
  for (int i = m + threadIdx.x; i < size; i += kThreads) sh.list[i] = 0;
  __syncthreads();
  return size;
}

// `u` of a sum of weights: the target is exceeded by exactly one token's running sum.
__device__ __forceinline__ u64 Target(const SampleRowsParams& p, int row, u64 total) {
  const double u = fmin(fmax(p.u != nullptr ? static_cast<double>(p.u[row]) : 0.0, 0.0), 1.0);
  return min(static_cast<u64>(u * static_cast<double>(total)), total - 1);
}

// Among the row's values with keys from `cut` on: the key of the `need`-th
// largest, or (by_mass) the largest key from which on the weights reach `share`
// of their sum; `cut` where there is none.  First by the distance from the
// largest value, in units of 2^-25 of a factor 2 of weight, ten bits at a time:
// a row's values spread over many bins so, and the few in the bin that counts
// are sorted in the first block, or listed for what follows.  Then, where distances round alike and keys do
// not, by the keys.
template <typename F>
__device__ __forceinline__ uint32_t Select(Shared& sh, const Weights& weigh, bool by_mass, float share, u64 need, uint32_t cut,
                                           int n, F value, uint32_t rank) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  u64 over = 0;  // counts or weights before the prefix's range
  uint32_t prefix = 0, at = 0;
  int listed = -1;  // values of this block that are listed in sh.mine; -1: all are looked through
  constexpr int kAhead = 4;
  // every value that counts, four of a thread at a time
  auto each = [&](auto f) {
    const int count = listed >= 0 ? listed : n;
#pragma unroll 1
    for (int i0 = tid; i0 < count; i0 += kThreads * kAhead) {
      float v[kAhead];
      int i[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        i[e] = i0 + e * kThreads;
        v[e] = -INFINITY;
        if (i[e] < count) {
          if (listed >= 0) i[e] = static_cast<int>(~static_cast<uint32_t>(sh.mine[i[e]]));
          v[e] = value(i[e]);
        }
      }
      f(v, i);
    }
  };
#pragma unroll 1
  for (int digit = 0; digit < 7; ++digit) {
    const bool by_key = digit >= 3;  // three digits of the distance, then four of 8 bits of the key's complement
    const int bits = by_key ? 8 : kBinBits, shift = by_key ? 24 - 8 * (digit - 3) : 20 - 10 * digit;
    if (digit == 1) {
      // what is in the bin
      if (tid == 0) {
    sh.n_mine = 0;
    sh.listed = 0;
  }
      __syncthreads();
      each([&](const float (&v)[kAhead], const int (&i)[kAhead]) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
          if (Key(v[e]) >= cut && weigh.Distance(v[e]) >> 20 == prefix) {
            const unsigned to = atomicAdd(&sh.n_mine, 1u);
            if (to < kList / 4) sh.mine[to] = static_cast<u64>(Key(v[e])) << 32 | ~static_cast<uint32_t>(i[e]);
          }
        }
      });
      ClusterSync();
      int m = 0;
      bool fits = true;
      for (uint32_t c = 0; c < kCluster; ++c) {
        const unsigned x = *In(&sh.n_mine, c);
        fits = fits && x <= kList / 4;
        m += static_cast<int>(x);
      }
      if (fits && m <= kList) {
        // few enough for the first block to sort
        if (rank == 0) {
          const int size = Gather(sh, m);
          Sort(sh.list, size);
          u64 w[4], own = 0;
          const int i = 4 * tid;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t k = i + e < m ? static_cast<uint32_t>(sh.list[i + e] >> 32) : 0;
            w[e] = k == 0 ? 0 : (by_mass ? weigh.Fixed(FromKey(k)) : 1);
            own += w[e];
          }
          u64 before = WarpScan(own, lane);
          if (lane == 31) sh.wsum[warp] = before;
          // (sums of weights that round otherwise than the bins': the last of them then)
          if (tid == 0) sh.least = static_cast<uint32_t>(sh.list[m - 1] >> 32);
          __syncthreads();
          before += over - own;
          for (int k = 0; k < warp; ++k) before += sh.wsum[k];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (before < need && need <= before + w[e]) sh.least = static_cast<uint32_t>(sh.list[i + e] >> 32);
            before += w[e];
          }
        }
        ClusterSync();
        const uint32_t least = *In(&sh.least, 0);
        ClusterSync();  // (it has been read)
        return least;
      }
      if (sh.n_mine <= kList / 4) listed = static_cast<int>(sh.n_mine);
    }
    if (digit == 3) {
      at = prefix;
      prefix = 0;
      if (tid == 0) {
        sh.least = 0xFFFFFFFFu;
        sh.most = 0;
      }
      __syncthreads();
      uint32_t a = 0xFFFFFFFFu, b = 0;
      each([&](const float (&v)[kAhead], const int (&)[kAhead]) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
          const uint32_t k = Key(v[e]);
          if (k >= cut && weigh.Distance(v[e]) == at) {
            a = min(a, k);
            b = max(b, k);
          }
        }
      });
      a = __reduce_min_sync(0xFFFFFFFFu, a);
      b = __reduce_max_sync(0xFFFFFFFFu, b);
      if (lane == 0) {
        atomicMin(&sh.least, a);
        atomicMax(&sh.most, b);
      }
      ClusterSync();
      a = 0xFFFFFFFFu;
      b = 0;
      for (uint32_t c = 0; c < kCluster; ++c) {
        a = min(a, *In(&sh.least, c));
        b = max(b, *In(&sh.most, c));
      }
      ClusterSync();
      if (a == b) return a;
    }
#pragma unroll 1
    for (int i = tid; i < kBins; i += kThreads) sh.bins.part[0][i] = sh.bins.part[1][i] = sh.bins.part[2][i] = 0;
    if (tid == 0) sh.found = -1;
    __syncthreads();
    each([&](const float (&v)[kAhead], const int (&)[kAhead]) {
      float2 hi[kAhead / 2], lo[kAhead / 2];
      if (by_mass) {
#pragma unroll
        for (int e = 0; e < kAhead / 2; ++e) weigh(make_float2(v[2 * e], v[2 * e + 1]), hi[e], lo[e]);
      }
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const uint32_t k = Key(v[e]);
        uint32_t code = weigh.Distance(v[e]);
        const bool in = k >= cut && (!by_key || code == at);
        if (by_key) code = ~k;
        if (!in || (digit != 0 && digit != 3 && code >> (shift + bits) != prefix)) continue;
        const uint32_t bin = code >> shift & ((1u << bits) - 1);
        if (by_mass) {
          int x, y, z;
          Weights::ToParts(e & 1 ? hi[e / 2].y : hi[e / 2].x, e & 1 ? lo[e / 2].y : lo[e / 2].x, x, y, z);
          if (x != 0) atomicAdd(&sh.bins.part[0][bin], x);
          if (y != 0) atomicAdd(&sh.bins.part[1][bin], y);
          if (z != 0) atomicAdd(&sh.bins.part[2][bin], z);
        } else {
          atomicAdd(&sh.bins.part[2][bin], 1);
        }
      }
    });
    ClusterSync();
    {
      // all blocks' sums of this block's bins, four threads to a bin
      const int bin = rank * (kBins / kCluster) + tid / 4;
      u64 sum = 0;
#pragma unroll
      for (int c = 0; c < kCluster / 4; ++c) {
        const uint32_t b = tid % 4 * (kCluster / 4) + c;
        sum += static_cast<u64>(In(sh.bins.part[0], b)[bin] * (1ll << 30) + In(sh.bins.part[1], b)[bin] * (1ll << 15) +
                                In(sh.bins.part[2], b)[bin]);
      }
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      static_assert(4 * kBins / kCluster == kThreads, "threads of a bin");
      if (tid % 4 == 0) sh.bins.all[tid / 4] = sum;
    }
    ClusterSync();
    // the bin in which the sum from the front reaches what is needed: two bins a thread
    static_assert(kBins == 2 * kThreads, "bins of a thread");
    const int bin = 2 * tid;
    const u64* all = In(sh.bins.all, bin / (kBins / kCluster));
    const u64 s0 = all[bin % (kBins / kCluster)], s1 = all[bin % (kBins / kCluster) + 1];
    u64 before = WarpScan(s0 + s1, lane);
    if (lane == 31) sh.wsum[warp] = before;
    before -= s0 + s1;
    __syncthreads();
    u64 total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.wsum[w];
      total += sh.wsum[w];
    }
    if (by_mass && digit == 0) need = static_cast<u64>(ceil(static_cast<double>(share) * static_cast<double>(total)));
    before += over;
    if (before < need && need <= before + s0) {
      sh.found = bin;
      sh.over = before;
    } else if (before + s0 < need && need <= before + s0 + s1) {
      sh.found = bin + 1;
      sh.over = before + s0;
    }
    __syncthreads();
    if (sh.found < 0) return cut;  // fewer values than are wanted: all stay
    prefix = prefix << bits | static_cast<uint32_t>(sh.found);
    over = sh.over;
  }
  return ~prefix;
}

// Three blocks on an SM for 16-bit rows (40 registers a thread): 256 rows 121 us,
// two blocks of 64 registers 132.  Of f32 rows of 151936 two fit: 64 rows 94 us
// with 64 registers, 99 with 40.
template <typename T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2) SampleRowsKernel(const SampleRowsParams p, int per) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ Shared sh;
  T* vals = reinterpret_cast<T*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = ClusterRank();
  const int row = blockIdx.x / kCluster;
  if (tid < 256) {
    const double x = exp2(tid / 256.0);
    const float h = static_cast<float>(x);
    sh.power[tid] = make_float2(h, static_cast<float>(x - static_cast<double>(h)));
  }
  if (tid == 0) {
    sh.n_mine = 0;
    sh.listed = 0;
  }
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
#pragma unroll 1
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
#pragma unroll 1
    for (int i = vecs * kVec + tid; i < n; i += kThreads) {
      vals[i] = src[i];
      best = fmaxf(best, kvd::ToFloat(vals[i]));
    }
  } else {
    constexpr int kFlight = 8;
#pragma unroll 1
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
    unsigned w = my_key;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) w = max(w, __shfl_xor_sync(0xFFFFFFFFu, w, o));
    if (lane % 8 == 0) sh.group_top[tid / 8] = w;
    w = __reduce_max_sync(0xFFFFFFFFu, w);
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
#pragma unroll 1
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
  const bool by_min = min_p > 0.f && min_p <= 1.f;
  // the weights of two values, 0 where a filter drops them
  auto kept = [&](float2 v, float2& hi, float2& lo) {
    weigh(v, hi, lo);
    const uint32_t least = max(least_min, cut);
    if (least == 1) return;  // (what is not finite has no weight)
    if (Key(v.x) < least || (by_min && static_cast<double>(hi.x) + static_cast<double>(lo.x) < static_cast<double>(min_p))) {
      hi.x = lo.x = 0.f;
    }
    if (Key(v.y) < least || (by_min && static_cast<double>(hi.y) + static_cast<double>(lo.y) < static_cast<double>(min_p))) {
      hi.y = lo.y = 0.f;
    }
  };

  if (by_k || by_p) {
    // ---- a bound that at least `want` values reach: the want-th largest of the
    // largest values of groups of the row (its upper 22 bits).  Of 512 groups of
    // eight threads one warp finds it; where more are wanted, of all threads, together.
    const int want = by_k ? min(top_k, kMostK + 1) : kFirst;
    const bool listed = want <= kMostK;
    uint32_t bound = 0;
    if (want <= kGroups / 4 * 3) {
      if (warp == 0) {
        unsigned key[kGroups / 32];
#pragma unroll
        for (int i = 0; i < kGroups / 32; i += 4) {
          const int at = lane * (kGroups / 32) + i;
          const uint4 w = *reinterpret_cast<const uint4*>(In(sh.group_top, at / (kGroups / kCluster)) + at % (kGroups / kCluster));
          key[i] = w.x;
          key[i + 1] = w.y;
          key[i + 2] = w.z;
          key[i + 3] = w.w;
        }
#pragma unroll 1
        for (int bit = 31; bit >= 10; --bit) {
          const uint32_t try_ = bound | 1u << bit;
          int c = 0;
#pragma unroll
          for (int i = 0; i < kGroups / 32; ++i) c += key[i] >= try_;
          if (__reduce_add_sync(0xFFFFFFFFu, c) >= want) bound = try_;
        }
        if (lane == 0) sh.least = bound;
      }
      __syncthreads();
      bound = sh.least;
    } else if (listed) {
      unsigned key[kCluster];
#pragma unroll
      for (uint32_t b = 0; b < kCluster; ++b) key[b] = In(sh.thread_top, b)[tid];
#pragma unroll 1
      for (int bit = 31; bit >= 10; --bit) {
        const uint32_t try_ = bound | 1u << bit;
        int c = 0;
#pragma unroll
        for (int b = 0; b < kCluster; ++b) c += key[b] >= try_;
        c = __reduce_add_sync(0xFFFFFFFFu, c);
        unsigned* wide = sh.wide + (bit & 1) * kWarps;
        if (lane == 0) wide[warp] = c;
        __syncthreads();
        int all = lane < kWarps ? static_cast<int>(wide[lane]) : 0;
        if (__reduce_add_sync(0xFFFFFFFFu, all) >= want) bound = try_;
      }
    }
    bound = max(bound, kLowest);
    // ---- what reaches it, and the sum of all weights where the list may not hold all that counts
    const float bound_value = listed ? FromKey(bound) : INFINITY;
    Sum sum;
    u64 in_list = 0;  // weights of what is listed
    constexpr int kAhead = 4;
#pragma unroll 1
    for (int i0 = warp * 32 * kAhead; i0 < n; i0 += kThreads * kAhead) {
      float v[kAhead];
      bool any = false;
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int i = i0 + e * 32 + lane;
        v[e] = i < n ? kvd::ToFloat(vals[i]) : -INFINITY;
        any |= v[e] >= bound_value;
      }
      float2 h[kAhead / 2], l[kAhead / 2];
      if (!by_k) {
#pragma unroll
        for (int e = 0; e < kAhead / 2; ++e) {
          weigh(make_float2(v[2 * e], v[2 * e + 1]), h[e], l[e]);
          sum.Add(h[e], l[e]);
        }
      }
      if (listed && __any_sync(0xFFFFFFFFu, any)) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
          const bool in = v[e] >= bound_value;
          const uint32_t mask = __ballot_sync(0xFFFFFFFFu, in);
          if (mask != 0) {
            unsigned at = 0;
            if (!by_k && in) {
              in_list += Weights::ToFixed(static_cast<double>(e & 1 ? h[e / 2].y : h[e / 2].x) +
                                          static_cast<double>(e & 1 ? l[e / 2].y : l[e / 2].x));
            }
            if (lane == 0) at = atomicAdd(&sh.n_mine, __popc(mask));
            at = __shfl_sync(0xFFFFFFFFu, at, 0) + __popc(mask & ((1u << lane) - 1));
            if (in && at < kList / 4) {
              sh.mine[at] = static_cast<u64>(Key(v[e])) << 32 | ~static_cast<uint32_t>(begin + i0 + e * 32 + lane);
            }
          }
        }
      }
    }
    const u64 mass = WarpAdd(Weights::ToFixed(sum.Total()));
    in_list = WarpAdd(in_list);
    if (lane == 0) {
      sh.wsum[warp] = mass;
      if (in_list != 0) atomicAdd(&sh.listed, in_list);
    }
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int k = 0; k < kWarps; ++k) s += sh.wsum[k];
      sh.sum = s;
    }
    ClusterSync();
    bool fits = listed;
    u64 total = 0, there = 0;
    int m = 0;
    for (uint32_t b = 0; b < kCluster; ++b) {
      const unsigned c = *In(&sh.n_mine, b);
      fits = fits && c <= kList / 4;
      m += static_cast<int>(c);
      total += *In(&sh.sum, b);
      there += *In(&sh.listed, b);
    }
    u64 need = by_p ? static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(total))) : 0;
    fits = fits && m <= kList && (by_k || there >= need);
    if (fits) {
      if (rank == 0) {
        // ---- the first block sorts the list and cuts it
        Sort(sh.list, Gather(sh, m));
        uint32_t least = by_k && top_k <= m ? static_cast<uint32_t>(sh.list[top_k - 1] >> 32) : 1;
        // weights of the values from there on, and their running sums: four values a thread
        u64 w[4], own = 0;
        int kept_here = 0;
        const int i = 4 * tid;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = i + e < m ? static_cast<uint32_t>(sh.list[i + e] >> 32) : 0;
          w[e] = 0;
          if (k >= least && k != 0) {
            w[e] = weigh.Fixed(FromKey(k));
            ++kept_here;
          }
          own += w[e];
        }
        if (by_p) {
          u64 before = WarpScan(own, lane);
          if (lane == 31) sh.wsum[warp] = before;
          if (tid == 0) sh.least = 1;
          __syncthreads();
          u64 sum = 0;
          for (int k = 0; k < kWarps; ++k) {
            if (k < warp) before += sh.wsum[k];
            sum += sh.wsum[k];
          }
          before -= own;
          if (by_k) need = static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(sum)));
          // the first value with which the sum reaches the share is the last of the kept
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (before < need && need <= before + w[e]) sh.least = static_cast<uint32_t>(sh.list[i + e] >> 32);
            before += w[e];
          }
          __syncthreads();
          least = max(least, sh.least);
          kept_here = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) kept_here += i + e < m && static_cast<uint32_t>(sh.list[i + e] >> 32) >= least;
        }
        kept_here = __reduce_add_sync(0xFFFFFFFFu, kept_here);
        if (lane == 0) sh.wide[warp] = static_cast<unsigned>(kept_here);
        __syncthreads();
        int count = 0;
        for (int k = 0; k < kWarps; ++k) count += static_cast<int>(sh.wide[k]);
        if (count <= kFew && warp < kFew / 32) {
          // ---- few: drawn here.  What comes before a token by its index is added up for each.
          const uint32_t key = tid < count ? static_cast<uint32_t>(sh.list[tid] >> 32) : 0;
          const double d = key != 0 ? weigh(FromKey(key)) : 0.0;
          const u64 mine_w = key < least_min || (by_min && d < static_cast<double>(min_p)) ? 0 : Weights::ToFixed(d);
          sh.weight[tid] = mine_w;
          asm volatile("bar.sync 1, %0;" ::"n"(kFew) : "memory");
          const uint32_t index = ~static_cast<uint32_t>(sh.list[tid]);
          u64 all = 0, before = 0;
#pragma unroll 1
          for (int j = 0; j < count; ++j) {
            const u64 x = sh.weight[j];
            all += x;
            before += ~static_cast<uint32_t>(sh.list[j]) < index ? x : 0;
          }
          const u64 target = Target(p, row, all);
          if (tid < count && before <= target && target - before < mine_w) {
            p.tok[row] = static_cast<int>(index);
            if (p.prob != nullptr) p.prob[row] = static_cast<float>(d * kFix / static_cast<double>(all));
          }
        }
        if (tid == 0) {
          sh.found = count <= kFew;
          sh.least = least;
        }
      }
      ClusterSync();
      const bool found = *In(&sh.found, 0) != 0;
      cut = *In(&sh.least, 0);
      if (found) {
        ClusterSync();  // (it has been read: the first block may end)
        return;
      }
    } else {
      // ---- the least key that the filters leave
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {
        if (pass == 0 ? by_k : by_p) {
          cut = Select(sh, weigh, pass == 1, top_p, static_cast<u64>(top_k), cut, n, [&](int i) { return kvd::ToFloat(vals[i]); },
                       rank);
        }
      }
    }
  }

  // ---- the kept weights: a run of the row for each warp
  const int run = (per + kThreads - 1) / kThreads, lo = min(warp * 32 * run, n), hi = min(lo + 32 * run, n);
  const float floor_ = fmaxf(cut > 1 ? FromKey(cut) : -INFINITY, least_min > 1 ? FromKey(least_min) : -INFINITY);
  Sum sum;
  constexpr int kAhead = 4;
#pragma unroll 1
  for (int i0 = lo; i0 < hi; i0 += 32 * kAhead) {
    float v[kAhead];
    bool any = false;
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int i = i0 + e * 32 + lane;
      v[e] = i < hi ? kvd::ToFloat(vals[i]) : -INFINITY;
      any |= v[e] >= floor_;
    }
    if (__any_sync(0xFFFFFFFFu, any)) {
#pragma unroll
      for (int e = 0; e < kAhead; e += 2) {
        float2 h, l;
        kept(make_float2(v[e], v[e + 1]), h, l);
        sum.Add(h, l);
      }
    }
  }
  const u64 mine = WarpAdd(Weights::ToFixed(sum.Total()));
  if (lane == 0) sh.wsum[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    u64 s = 0;
    for (int k = 0; k < kWarps; ++k) s += sh.wsum[k];
    sh.sum = s;
  }
  ClusterSync();
  u64 before = 0, total = 0;
  for (uint32_t b = 0; b < kCluster; ++b) {
    const u64 s = *In(&sh.sum, b);
    if (b < rank) before += s;
    total += s;
  }
  ClusterArrive();
  for (int k = 0; k < warp; ++k) before += sh.wsum[k];
  const u64 target = Target(p, row, total);
  if (before <= target && target - before < mine) {
    // This warp has it: a run for each lane, then the values of that run.  (These
    // sums round elsewhere than the warp's, by 2^-44: what is past the end goes to
    // the last that is kept.)
    Sum run_sum;
    const int a = min(lo + lane * run, hi), b = min(a + run, hi);
#pragma unroll 1
    for (int i0 = 0; i0 < run; i0 += kAhead) {
      float v[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) v[e] = a + i0 + e < b ? kvd::ToFloat(vals[a + i0 + e]) : -INFINITY;
#pragma unroll
      for (int e = 0; e < kAhead; e += 2) {
        float2 h, l;
        kept(make_float2(v[e], v[e + 1]), h, l);
        run_sum.Add(h, l);
      }
    }
    const u64 own = Weights::ToFixed(run_sum.Total());
    const u64 incl = before + WarpScan(own, lane);
    const uint32_t over = __ballot_sync(0xFFFFFFFFu, own > 0 && target < incl), some = __ballot_sync(0xFFFFFFFFu, own > 0);
    const int who = over != 0 ? __ffs(over) - 1 : 31 - __clz(some);
    const int a1 = __shfl_sync(0xFFFFFFFFu, a, who), b1 = __shfl_sync(0xFFFFFFFFu, b, who);
    u64 so_far = __shfl_sync(0xFFFFFFFFu, incl - own, who);
    int last = -1;  // the lane's last kept value
    bool found = false;
#pragma unroll 1
    for (int i0 = a1; i0 < b1 && !found; i0 += 32) {
      const int i = i0 + lane;
      float2 h, l;
      kept(make_float2(i < b1 ? kvd::ToFloat(vals[i]) : -INFINITY, -INFINITY), h, l);
      const u64 w = Weights::ToFixed(static_cast<double>(h.x) + static_cast<double>(l.x));
      const u64 to = so_far + WarpScan(w, lane);
      if (w > 0) last = i;
      const uint32_t here = __ballot_sync(0xFFFFFFFFu, w > 0 && target < to);
      if (here != 0) {
        last = __shfl_sync(0xFFFFFFFFu, i, __ffs(here) - 1);
        found = true;
      }
      so_far = __shfl_sync(0xFFFFFFFFu, to, 31);
    }
    if (!found) last = __reduce_max_sync(0xFFFFFFFFu, last);
    if (lane == 0) {
      p.tok[row] = begin + last;
      if (p.prob != nullptr) p.prob[row] = static_cast<float>(weigh(kvd::ToFloat(vals[last])) * kFix / static_cast<double>(total));
    }
  }
  __syncwarp();
  ClusterWait();  // no block ends while another reads its sums
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
