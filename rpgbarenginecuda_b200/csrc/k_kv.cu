// k_kv.cu -- writing a paged key-value cache and reading it back.
#include "common.h"
#include "kv_dev.cuh"
#include "launch.h"

namespace rpgb {
namespace {

constexpr int kThreads = 128;

template <KvType KIND>
__host__ __device__ constexpr float MostCode() {
  return KIND == KvType::kQ8 ? 127.f : 7.f;
}

// Largest of the lanes' values as the bits of a non-negative float; a NaN has
// the largest bits of all, so it wins.
template <int LANES>
__device__ __forceinline__ uint32_t LanesMax(uint32_t v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
__device__ __forceinline__ uint32_t MaxAbs4(const float (&x)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
  return m;
}
// The scale of a group from the bits of its largest magnitude: rounded to f16
// (the cache's format), kept finite for magnitudes past its range (which then
// saturate), NaN for a group that holds one.
template <KvType KIND>
__device__ __forceinline__ __half GroupScale(uint32_t max_bits) {
  const float m = __uint_as_float(max_bits);
  return __float2half_rn(max_bits > 0x7F800000u ? m : fminf(m * (1.f / MostCode<KIND>()), 65504.f));
}

// Codes of four consecutive values x, nearest with ties to even.  A scale that
// was rounded down (far down where it is subnormal) needs the clamp.
template <KvType KIND>
__device__ __forceinline__ void StoreCodes(char* row, int i, const float (&x)[4], float d) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float c = d > 0.f ? fminf(fmaxf(rintf(x[e] / d), -MostCode<KIND>()), MostCode<KIND>()) : 0.f;
    const int q = static_cast<int>(c);
    w |= KIND == KvType::kQ8 ? static_cast<uint32_t>(q & 255) << (8 * e) : static_cast<uint32_t>(q + 8) << (4 * e);
  }
  if (KIND == KvType::kQ8) {
    *reinterpret_cast<uint32_t*>(row + i) = w;
  } else {
    *reinterpret_cast<uint16_t*>(row + i / 2) = static_cast<uint16_t>(w);
  }
}

// 1 / sqrt(mean x^2 + eps) of a head, in f32.  The squares and sums round one
// by one (no fused multiply-add) in a fixed tree: the halves' lanes, then
// lanes 8, 4, 2 and 1 apart.
template <int D>
__device__ __forceinline__ float InvRms(const float (&a)[4], const float (&b)[4], float eps) {
  float t[4], s;
  if (D == 128) {  // runs of four values first
    float u = __fmul_rn(a[0], a[0]), v = __fmul_rn(b[0], b[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) {
      u = __fadd_rn(u, __fmul_rn(a[e], a[e]));
      v = __fadd_rn(v, __fmul_rn(b[e], b[e]));
    }
    s = __fadd_rn(u, v);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xFFFFFFFFu, s, o));
  } else {  // the lanes first, then the values of a lane
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = __fadd_rn(__fmul_rn(a[e], a[e]), __fmul_rn(b[e], b[e]));
#pragma unroll
      for (int o = D / 16; o > 0; o >>= 1) t[e] = __fadd_rn(t[e], __shfl_xor_sync(0xFFFFFFFFu, t[e], o));
    }
    s = __fadd_rn(__fadd_rn(t[0], t[2]), __fadd_rn(t[1], t[3]));
  }
  return rsqrtf(__fadd_rn(__fmul_rn(s, 1.0f / D), eps));
}

// One row t, one head per D / 8 lanes.  Lane i holds values 4 i .. 4 i + 3 of
// the first half (a) and of the second (b), so a rotation pair (j, j + D / 2)
// sits in one lane and a scale group of 64 values in the same lanes.  Norm and
// rotation round every product and sum on its own, so a value that falls near
// a rounding boundary of the cache gets the code of the formulas evaluated
// step by step in f32.
template <int D, KvType KIND, typename T>
__global__ void __launch_bounds__(kThreads) KvAppendKernel(const KvAppendParams p) {
  constexpr int L = D / 8;
  dev::GridLaunchDependents();
  dev::GridWait();  // (launched before the stream's previous kernel has finished)
  const int64_t t = blockIdx.x;
  const int hq = p.q_out != nullptr ? p.n_heads : 0;
  const int head = blockIdx.y * (kThreads / L) + threadIdx.x / L;  // the q heads that are wanted, k heads, v heads
  const int i = threadIdx.x % L;
  const bool live = head < hq + 2 * p.kv.n_kv;
  const int pos = p.pos[t];
  const int seq = p.seq != nullptr ? p.seq[t] : static_cast<int>(t);
  const int page = pos < 0 ? -1 : kvd::PageOf(p.table, p.kv.n_pages, seq, pos >> p.kv.page_log2);
  const bool ok = page >= 0 && (p.rope == nullptr || pos < p.rope_positions);
  enum { kQ, kK, kV };
  const int kind = head < hq ? kQ : (head < hq + p.kv.n_kv ? kK : kV);
  const int h = kind == kQ ? head : (kind == kK ? head - hq : head - hq - p.kv.n_kv);
  const int col = (kind == kQ ? h : p.n_heads + (kind == kV ? p.kv.n_kv : 0) + h) * D;

  float a[4] = {}, b[4] = {};
  if (live && ok) {
    const T* x = static_cast<const T*>(p.qkv) + t * p.qkv_stride + col;
    kvd::Load4(x + 4 * i, a);
    kvd::Load4(x + D / 2 + 4 * i, b);
  }
  const float* w = kind == kQ ? p.q_norm : (kind == kK ? p.k_norm : nullptr);
  const float r = InvRms<D>(a, b, p.eps);  // every lane takes part, whatever its head
  if (w != nullptr) {
    float wa[4], wb[4];
    kvd::Load4(w + 4 * i, wa);
    kvd::Load4(w + D / 2 + 4 * i, wb);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = __fmul_rn(__fmul_rn(a[e], r), wa[e]);
      b[e] = __fmul_rn(__fmul_rn(b[e], r), wb[e]);
    }
  }
  if (kind != kV && p.rope != nullptr && ok) {
    const float* rr = p.rope + static_cast<int64_t>(pos) * D;
    float c[4], s[4];
    kvd::Load4(rr + 4 * i, c);
    kvd::Load4(rr + D / 2 + 4 * i, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = a[e], y = b[e];
      a[e] = __fsub_rn(__fmul_rn(x, c[e]), __fmul_rn(y, s[e]));
      b[e] = __fadd_rn(__fmul_rn(y, c[e]), __fmul_rn(x, s[e]));
    }
  }
  uint32_t ma = 0, mb = 0;
  if (KIND != KvType::kF16) {
    ma = MaxAbs4(a);
    mb = MaxAbs4(b);
    if (D == kKvGroup) ma = mb = max(ma, mb);
    ma = LanesMax<L>(ma);
    mb = D == kKvGroup ? ma : LanesMax<L>(mb);
  }
  if (!live) return;
  if (kind == kQ) {
    if (!ok) {  // padding rows are zero, rows without a place NaN
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = b[e] = pos < 0 ? 0.f : kvd::Nan();
    }
    T* q = static_cast<T*>(p.q_out) + t * p.q_stride + static_cast<int64_t>(h) * D;
    kvd::Store4(q + 4 * i, a);
    kvd::Store4(q + D / 2 + 4 * i, b);
    return;
  }
  if (!ok) return;
  const int at = pos & ((1 << p.kv.page_log2) - 1);
  char* row = (kind == kK ? p.kv.k : p.kv.v) + kvd::CodeOffset(p.kv, page, h, at);
  if (KIND == KvType::kF16) {
    kvd::Store4(reinterpret_cast<__half*>(row) + 4 * i, a);
    kvd::Store4(reinterpret_cast<__half*>(row) + D / 2 + 4 * i, b);
    return;
  }
  __half* sc = reinterpret_cast<__half*>((kind == kK ? p.kv.k_scale : p.kv.v_scale) +
                                         kvd::ScaleOffset(p.kv, page, h, at));
  const __half da = GroupScale<KIND>(ma), db = GroupScale<KIND>(mb);
  if (i == 0) {
    if (D == kKvGroup) {
      *sc = da;
    } else {
      *reinterpret_cast<__half2*>(sc) = __halves2half2(da, db);
    }
  }
  StoreCodes<KIND>(row, 4 * i, a, __half2float(da));
  StoreCodes<KIND>(row, D / 2 + 4 * i, b, __half2float(db));
}

// One row t; eight consecutive values of one head's k or v row per thread.
template <int D, KvType KIND, typename T>
__global__ void __launch_bounds__(kThreads) KvGatherKernel(const KvGatherParams p) {
  constexpr int L = D / 8;
  dev::GridLaunchDependents();
  dev::GridWait();
  const int64_t t = blockIdx.x;
  const int head = blockIdx.y * (kThreads / L) + threadIdx.x / L;  // k heads, then v heads
  const int i = (threadIdx.x % L) * 8;
  if (head >= 2 * p.kv.n_kv) return;
  const bool is_k = head < p.kv.n_kv;
  const int h = is_k ? head : head - p.kv.n_kv;
  T* out = static_cast<T*>(is_k ? p.k_out : p.v_out);
  if (out == nullptr) return;
  out += t * p.out_stride + static_cast<int64_t>(h) * D + i;
  const int pos = p.pos[t];
  const int seq = p.seq != nullptr ? p.seq[t] : static_cast<int>(t);
  const int page = pos < 0 ? -1 : kvd::PageOf(p.table, p.kv.n_pages, seq, pos >> p.kv.page_log2);
  const int at = pos & ((1 << p.kv.page_log2) - 1);
  float x[2][4];
  if (page < 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = pos < 0 ? 0.f : kvd::Nan();
  } else {
    const char* row = (is_k ? p.kv.k : p.kv.v) + kvd::CodeOffset(p.kv, page, h, at);
    const __half* sc = nullptr;
    if (KIND != KvType::kF16) {
      sc = reinterpret_cast<const __half*>((is_k ? p.kv.k_scale : p.kv.v_scale) + kvd::ScaleOffset(p.kv, page, h, at));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = kvd::Value<KIND>(row, sc, i + e);
  }
  kvd::Store4(out, x[0]);
  kvd::Store4(out + 4, x[1]);
}

template <template <int, KvType, typename> class F, typename P>
void Dispatch(const P& p, cudaStream_t s) {
  auto by_type = [&](auto dim, auto kind) {
    constexpr int D = decltype(dim)::value;
    constexpr KvType K = decltype(kind)::value;
    switch (p.type) {
      case ElemType::kF32: return F<D, K, float>::Run(p, s);
      case ElemType::kF16: return F<D, K, __half>::Run(p, s);
      case ElemType::kBF16: return F<D, K, __nv_bfloat16>::Run(p, s);
    }
  };
  auto by_kind = [&](auto dim) {
    switch (p.kv.type) {
      case KvType::kF16: return by_type(dim, std::integral_constant<KvType, KvType::kF16>());
      case KvType::kQ8: return by_type(dim, std::integral_constant<KvType, KvType::kQ8>());
      case KvType::kQ4: return by_type(dim, std::integral_constant<KvType, KvType::kQ4>());
    }
  };
  if (p.kv.head_dim == 64) {
    by_kind(std::integral_constant<int, 64>());
  } else {
    by_kind(std::integral_constant<int, 128>());
  }
}

template <int D, KvType KIND, typename T>
struct Append {
  static void Run(const KvAppendParams& p, cudaStream_t s) {
    constexpr int kHeads = kThreads / (D / 8);
    const int heads = (p.q_out != nullptr ? p.n_heads : 0) + 2 * p.kv.n_kv;
    const dim3 grid(static_cast<unsigned>(p.n_tok), (heads + kHeads - 1) / kHeads);
    LaunchKernelArgs(reinterpret_cast<const void*>(KvAppendKernel<D, KIND, T>), grid, dim3(kThreads), 0, s, true, p);
  }
};
template <int D, KvType KIND, typename T>
struct Gather {
  static void Run(const KvGatherParams& p, cudaStream_t s) {
    constexpr int kHeads = kThreads / (D / 8);
    const dim3 grid(static_cast<unsigned>(p.n_tok), (2 * p.kv.n_kv + kHeads - 1) / kHeads);
    LaunchKernelArgs(reinterpret_cast<const void*>(KvGatherKernel<D, KIND, T>), grid, dim3(kThreads), 0, s, true, p);
  }
};

}  // namespace

void LaunchKvAppend(const KvAppendParams& p, cudaStream_t s) {
  Dispatch<Append>(p, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

void LaunchKvGather(const KvGatherParams& p, cudaStream_t s) {
  Dispatch<Gather>(p, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

}  // namespace rpgb
