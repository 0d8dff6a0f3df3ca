// k_kv.cu -- writing a paged key-value cache and reading it back.
//
// Both are bound by memory and by the issue of what goes with it.  append
// reads a q|k|v row and writes q and the cache: the 2811 rows of 16 / 8 heads
// in f32 take 16.5 us (floor 12.5 us at the measured copy rate of 6.55 TB/s);
// 10624 rows of 32 / 8 heads in f16 into 4 bits 51 us (35), where the norm,
// the rotation and the codes keep the SMs issuing three quarters of the time.
// gather reads 41000 rows of 8 heads in 4 bits and writes them in f16 in 42 us
// (33).  A single row takes 1.7 to 2.4 us on the GPU (calls in a graph).
#include <atomic>

#include "common.h"
#include "kv_dev.cuh"
#include "launch.h"

namespace rpgb {
namespace {

// Threads of an append block: 10624 rows of 32 / 8 heads in f16 into 4 bits
// take 51.1 us with 64, 53.4 with 128, 78.8 with 256.
constexpr int kThreads = 64;

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
__device__ __forceinline__ uint32_t MaxAbs8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
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

// Codes of eight consecutive values: the IEEE quotient x / d rounded to the
// nearest integer, ties to even.  The product with 1 / d is off the quotient
// by less than 1e-4 (quotients are at most 127.1), so its rounding is the same
// unless it is that close to a tie; the low bits of 1.5 2^23 + y are y rounded.
// A scale that was rounded far down (it is subnormal) or is the largest can
// leave quotients past the largest code; those take the slow way too.
template <KvType KIND>
__device__ __forceinline__ void StoreCodes(char* row, int i, const float (&x)[8], float d) {
  constexpr float kMost = MostCode<KIND>();
  constexpr float kRound = 12582912.f;
  constexpr float kZero = KIND == KvType::kQ8 ? 0.f : 8.f;  // the code that stands for zero
  uint32_t c[8];
  const float inv = 1.f / d;
  float off = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = x[e] * inv;
    const float z = y + (kRound + kZero);
    off = fmaxf(off, fabsf(y - (z - (kRound + kZero))));
    c[e] = __float_as_uint(z);
  }
  if (!(off < 0.4999f && d >= 6.2e-5f && d < 65504.f)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = d > 0.f ? fminf(fmaxf(rintf(x[e] / d), -kMost), kMost) : 0.f;
      c[e] = static_cast<uint32_t>(static_cast<int>(q + kZero));
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    w[k] = __byte_perm(__byte_perm(c[4 * k], c[4 * k + 1], 0x0040), __byte_perm(c[4 * k + 2], c[4 * k + 3], 0x0040),
                       0x5410);
  }
  if (KIND == KvType::kQ8) {
    *reinterpret_cast<uint2*>(row + i) = make_uint2(w[0], w[1]);
  } else {
    w[0] &= 0x0F0F0F0Fu;
    w[1] &= 0x0F0F0F0Fu;
    *reinterpret_cast<uint32_t*>(row + i / 2) = __byte_perm(w[0] | w[0] >> 4, w[1] | w[1] >> 4, 0x6420);
  }
}

// 1 / sqrt(mean x^2 + eps) of a head, in f32.  The squares and sums round one
// by one (no fused multiply-add), in an order that is part of the operator's
// definition: it decides the code of a value that falls beside a rounding
// boundary (a sum from the left gives another 8-bit code for 5 values in a
// million).  The orders are those of torch.mean over rows of 64 and of 128 on
// this GPU, so that codes can be held against an evaluation there.
template <int D>
__device__ __forceinline__ float InvRms(const float (&a)[8], const float (&b)[8], float eps) {
  float s;
  if (D == 128) {  // runs of four values, then runs 64, 32, 16, 8 and 4 values apart
    float u[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float p = __fmul_rn(a[4 * h], a[4 * h]), q = __fmul_rn(b[4 * h], b[4 * h]);
#pragma unroll
      for (int e = 4 * h + 1; e < 4 * h + 4; ++e) {
        p = __fadd_rn(p, __fmul_rn(a[e], a[e]));
        q = __fadd_rn(q, __fmul_rn(b[e], b[e]));
      }
      u[h] = __fadd_rn(p, q);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) u[h] = __fadd_rn(u[h], __shfl_xor_sync(0xFFFFFFFFu, u[h], o));
    }
    s = __fadd_rn(u[0], u[1]);
  } else {  // values 32, 16, 8, 4, 2 and 1 apart
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = __fadd_rn(__fmul_rn(a[e], a[e]), __fmul_rn(b[e], b[e]));
#pragma unroll
      for (int o = 2; o > 0; o >>= 1) t[e] = __fadd_rn(t[e], __shfl_xor_sync(0xFFFFFFFFu, t[e], o));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
      for (int e = 0; e < o; ++e) t[e] = __fadd_rn(t[e], t[e + o]);
    }
    s = t[0];
  }
  return rsqrtf(__fadd_rn(__fmul_rn(s, 1.0f / D), eps));
}

// One row t per block (and a part of its heads when the rows are few), one
// head per D / 16 lanes at a time.  Lane i holds values 8 i .. 8 i + 7 of the
// first half (a) and of the second (b), so a rotation pair (j, j + D / 2) sits
// in one lane and a scale group of 64 values in the same lanes; the rotation
// stays in registers for all heads.  Norm and rotation round every product and
// sum on its own, in the order of InvRms and of the formulas as written, so
// equal rows get equal codes whatever the launch.
template <int D, KvType KIND, typename T>
__global__ void __launch_bounds__(kThreads) KvAppendKernel(const KvAppendParams p) {
  constexpr int L = D / 16, kHeads = kThreads / L;
  dev::GridLaunchDependents();
  dev::GridWait();  // (launched before the stream's previous kernel has finished)
  const int64_t t = blockIdx.x;
  const int hq = p.q_out != nullptr ? p.n_heads : 0;
  const int heads = hq + 2 * p.kv.n_kv;  // the q heads that are wanted, k heads, v heads
  const int i = threadIdx.x % L;
  const int skip = p.n_heads - hq;
  // the heads of a row follow one another: head x (of those wanted) is its head x, past the q heads that are not
  const T* x0 = static_cast<const T*>(p.qkv) + t * p.qkv_stride + static_cast<int64_t>(skip) * D + 8 * i;
  int head = blockIdx.y * kHeads + threadIdx.x / L;
  kvd::Raw8<T> xa, xb;  // of the next head, requested one round ahead
  if (head < heads) {
    xa.Load(x0 + head * D);
    xb.Load(x0 + head * D + D / 2);
  }
  const int pos = p.pos[t];
  const int seq = p.seq != nullptr ? p.seq[t] : static_cast<int>(t);
  const bool turn = p.rope != nullptr && pos >= 0 && pos < p.rope_positions;
  float cs[8], sn[8];
  if (turn) {
    const float* rr = p.rope + static_cast<int64_t>(pos) * D;
    kvd::Load8(rr + 8 * i, cs);
    kvd::Load8(rr + D / 2 + 8 * i, sn);
  }
  const int page = pos < 0 ? -1 : kvd::PageOf(p.table, p.kv.n_pages, seq, pos >> p.kv.page_log2);
  const bool ok = page >= 0 && (p.rope == nullptr || turn);
  const int at = pos & ((1 << p.kv.page_log2) - 1);
  enum { kQ, kK, kV };
  // (every lane of a warp goes round as often: the shuffles need them all)
  for (int head0 = blockIdx.y * kHeads; head0 < heads; head0 += gridDim.y * kHeads, head += gridDim.y * kHeads) {
    const bool live = head < heads;
    const int kind = head < hq ? kQ : (head < hq + p.kv.n_kv ? kK : kV);
    const int h = kind == kQ ? head : (kind == kK ? head - hq : head - hq - p.kv.n_kv);
    float a[8] = {}, b[8] = {};
    if (live) {
      xa.Floats(a);
      xb.Floats(b);
      const int next = head + gridDim.y * kHeads;
      if (next < heads) {
        xa.Load(x0 + next * D);
        xb.Load(x0 + next * D + D / 2);
      }
    }
    const float* w = kind == kQ ? p.q_norm : (kind == kK ? p.k_norm : nullptr);
    // (a warp has heads of one kind, or of several: the shuffles need all its lanes)
    const float r = __any_sync(0xFFFFFFFFu, w != nullptr) ? InvRms<D>(a, b, p.eps) : 1.f;
    if (w != nullptr) {
      float wa[8], wb[8];
      kvd::Load8(w + 8 * i, wa);
      kvd::Load8(w + D / 2 + 8 * i, wb);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] = __fmul_rn(__fmul_rn(a[e], r), wa[e]);
        b[e] = __fmul_rn(__fmul_rn(b[e], r), wb[e]);
      }
    }
    if (kind != kV && turn) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = a[e], y = b[e];
        a[e] = __fsub_rn(__fmul_rn(x, cs[e]), __fmul_rn(y, sn[e]));
        b[e] = __fadd_rn(__fmul_rn(y, cs[e]), __fmul_rn(x, sn[e]));
      }
    }
    uint32_t ma = 0, mb = 0;
    if (KIND != KvType::kF16 && __any_sync(0xFFFFFFFFu, kind != kQ)) {
      ma = MaxAbs8(a);
      mb = MaxAbs8(b);
      if (D == kKvGroup) ma = mb = max(ma, mb);
      ma = LanesMax<L>(ma);
      mb = D == kKvGroup ? ma : LanesMax<L>(mb);
    }
    if (!live) continue;
    if (kind == kQ) {
      if (!ok) {  // padding rows are zero, rows without a place NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = b[e] = pos < 0 ? 0.f : kvd::Nan();
      }
      T* q = static_cast<T*>(p.q_out) + t * p.q_stride + static_cast<int64_t>(h) * D;
      kvd::Store8(q + 8 * i, a);
      kvd::Store8(q + D / 2 + 8 * i, b);
      continue;
    }
    if (!ok) continue;
    char* row = (kind == kK ? p.kv.k : p.kv.v) + kvd::CodeOffset(p.kv, page, h, at);
    if (KIND == KvType::kF16) {
      kvd::Store8(reinterpret_cast<__half*>(row) + 8 * i, a);
      kvd::Store8(reinterpret_cast<__half*>(row) + D / 2 + 8 * i, b);
      continue;
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
    StoreCodes<KIND>(row, 8 * i, a, __half2float(da));
    StoreCodes<KIND>(row, D / 2 + 8 * i, b, __half2float(db));
  }
}

// Sixteen consecutive values of one head's k or v row per thread and row; the
// block's threads cover (values of a head) x (k heads, then v heads) x (rows),
// and each takes kRows rows of every blockDim.z at once, so that their chains
// of loads (position, page, codes) run side by side.  41000 rows of 8 heads to
// f16 with one row a thread, two and four: f16 63.9, 56.2 and 54.5 us, 8 bits
// 58.8, 56.2 and 62.7, 4 bits 55.8, 41.7 and 41.7; 40 rows 1.8, 2.1 and 2.5.
constexpr int kRows = 2;
template <int D, KvType KIND, typename T>
__global__ void __launch_bounds__(256) KvGatherKernel(const KvGatherParams p) {
  dev::GridLaunchDependents();
  dev::GridWait();
  const int i = threadIdx.x * 16;
  const int head = blockIdx.y * blockDim.y + threadIdx.y;
  if (head >= 2 * p.kv.n_kv) return;
  const bool is_k = head < p.kv.n_kv;
  const int h = is_k ? head : head - p.kv.n_kv;
  T* out = static_cast<T*>(is_k ? p.k_out : p.v_out);
  if (out == nullptr) return;
  const char* plane = is_k ? p.kv.k : p.kv.v;
  const char* scales = is_k ? p.kv.k_scale : p.kv.v_scale;
  const bool wide = (reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(p.out_stride * sizeof(T))) % 32 == 0;
  int64_t t[kRows];
  int pos[kRows], page[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    t[r] = (static_cast<int64_t>(blockIdx.x) * kRows + r) * blockDim.z + threadIdx.z;
    pos[r] = -1;
    page[r] = -1;
    if (t[r] < p.n_tok) pos[r] = p.pos[t[r]];
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (pos[r] >= 0) {
      const int seq = p.seq != nullptr ? p.seq[t[r]] : static_cast<int>(t[r]);
      page[r] = kvd::PageOf(p.table, p.kv.n_pages, seq, pos[r] >> p.kv.page_log2);
    }
  }
  kvd::Codes16<KIND> codes[kRows];
  __half d[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (page[r] >= 0) {
      const int at = pos[r] & ((1 << p.kv.page_log2) - 1);
      codes[r].Load(plane + kvd::CodeOffset(p.kv, page[r], h, at), i);
      if (KIND != KvType::kF16) {
        d[r] = *reinterpret_cast<const __half*>(scales + kvd::ScaleOffset(p.kv, page[r], h, at) + i / kKvGroup * 2);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (t[r] >= p.n_tok) continue;
    T* row = out + t[r] * p.out_stride + static_cast<int64_t>(h) * D + i;
    if (page[r] >= 0) {
      codes[r].Store(row, d[r], wide, p.magic);
    } else {  // padding rows are zero, rows without a place NaN
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = pos[r] < 0 ? 0.f : kvd::Nan();
      kvd::Store8(row, x);
      kvd::Store8(row + 8, x);
    }
  }
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

int NumSms() {
  static std::atomic<int> sms[64];
  int dev = 0, n = 0;
  RPGB_CUDA(cudaGetDevice(&dev));
  RPGB_CHECK(dev < 64, "kv: device %d", dev);
  n = sms[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    RPGB_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    sms[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Up to 32 blocks for every SM (14 run at once) a row's heads go to blocks of
// their own (latency); past that a block keeps its row's rotation for all its
// heads.  Rows of 32 / 8 heads in f16 to f16, a row in blocks of 8 heads and in
// one: 1 row 1.7 and 3.8 us, 300 3.2 and 5.3, 600 4.6 and 7.6, 1200 10.1 and
// 9.3, 9600 62 and 44; of 16 / 2 heads in f32 to 4 bits 1200 rows 7.1 and 7.6,
// 2400 13.5 and 13.3; the border is at 789 and at 1578 rows.
template <int D, KvType KIND, typename T>
struct Append {
  static void Run(const KvAppendParams& p, cudaStream_t s) {
    constexpr int kHeads = kThreads / (D / 16);
    const int heads = (p.q_out != nullptr ? p.n_heads : 0) + 2 * p.kv.n_kv;
    const int parts = (heads + kHeads - 1) / kHeads;
    const dim3 grid(static_cast<unsigned>(p.n_tok), p.n_tok * parts <= 32 * NumSms() ? parts : 1);
    LaunchKernelArgs(reinterpret_cast<const void*>(KvAppendKernel<D, KIND, T>), grid, dim3(kThreads), 0, s, true, p);
  }
};

// Up to 24 blocks for every SM a block takes kRows rows; past that as many more
// as fit its threads.  Rows of 2 heads from 8 to 16
// bits: 600 rows 2.3 and 2.6 us, 6000 3.4 and 3.7, 7000 4.0 and 3.7, 12000 6.7
// and 4.9, 41000 24.9 and 16.7; to f32 7000 5.3 and 7.3, 12000 9.7 and 8.8; the
// border is at 7104 rows.  (8 heads fill a block's threads either way.)
template <int D, KvType KIND, typename T>
struct Gather {
  static void Run(const KvGatherParams& p, cudaStream_t s) {
    constexpr int L = D / 16;
    const int heads = 2 * p.kv.n_kv, y = heads < 256 / L ? heads : 256 / L;
    const int64_t blocks = (p.n_tok + kRows - 1) / kRows * ((heads + y - 1) / y);
    const int64_t z = blocks <= 24 * NumSms() ? 1 : 256 / (L * y);
    const dim3 block(L, y, static_cast<unsigned>(z));
    const dim3 grid(static_cast<unsigned>((p.n_tok + kRows * z - 1) / (kRows * z)), (heads + y - 1) / y);
    LaunchKernelArgs(reinterpret_cast<const void*>(KvGatherKernel<D, KIND, T>), grid, block, 0, s, true, p);
  }
};

}  // namespace

void LaunchKvAppend(const KvAppendParams& p, cudaStream_t s) {
  Dispatch<Append>(p, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

void LaunchKvGather(const KvGatherParams& p, cudaStream_t s) {
  KvGatherParams a = p;
  a.magic = kvd::kMagic;
  Dispatch<Gather>(a, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

}  // namespace rpgb
