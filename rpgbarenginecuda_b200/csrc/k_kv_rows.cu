// k_kv_rows.cu -- attention of several rows that read one page list: new tokens
// of a conversation, or the conversations of a group over what they share.
#include "common.h"
#include "kv_dev.cuh"
#include "launch.h"

namespace rpgb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows of a list: [begin, end) within [0, n_rows].
__device__ __forceinline__ int RowBegin(const KvRowsParams& p, int list) { return min(max(p.rows[list], 0), p.n_rows); }
__device__ __forceinline__ int RowEnd(const KvRowsParams& p, int list) {
  return min(max(p.rows[list + 1], RowBegin(p, list)), p.n_rows);
}
// The table's row that holds a list's pages.
__device__ __forceinline__ int TableRow(const KvRowsParams& p, int list) {
  return p.prefix != nullptr ? RowBegin(p, list) : list;
}

// Positions [start, end) that a row sees of its list; `past`: it would see some behind the table.
struct Seen {
  int start, end;
  bool past;
};
__device__ __forceinline__ Seen SeenBy(const KvRowsParams& p, int row) {
  const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
  Seen s;
  s.start = p.starts != nullptr ? max(p.starts[row], 0) : 0;
  int64_t end = max(p.ends[row], 0);
  if (p.prefix != nullptr) end = min(end, static_cast<int64_t>(max(p.prefix[row], 0)));
  s.past = end > cap && s.start < end;
  s.end = static_cast<int>(min(end, cap));
  if (s.start >= s.end) s.start = s.end = 0;
  return s;
}

template <typename T>
__device__ __forceinline__ float Element(const void* q, int64_t i) {
  return kvd::ToFloat(static_cast<const T*>(q)[i]);
}
__device__ __forceinline__ float Element(const void* q, ElemType t, int64_t i) {
  return t == ElemType::kF32 ? Element<float>(q, i)
                             : (t == ElemType::kF16 ? Element<__half>(q, i) : Element<__nv_bfloat16>(q, i));
}
__device__ __forceinline__ void Put(void* out, ElemType t, int64_t i, float x) {
  switch (t) {
    case ElemType::kF32: static_cast<float*>(out)[i] = x; break;
    case ElemType::kF16: static_cast<__half*>(out)[i] = kvd::FromFloat<__half>(x); break;
    case ElemType::kBF16: static_cast<__nv_bfloat16*>(out)[i] = kvd::FromFloat<__nv_bfloat16>(x); break;
  }
}

// A score in units of log2 from a product of q and k.
__device__ __forceinline__ float Score(const KvRowsParams& p, float x, float slope, int distance) {
  x *= p.scale;
  if (p.cap > 0.f) {
    // tanh |t| = (1 - e) / (1 + e) with e = exp(-2 |t|)
    const float e = Exp2(fabsf(x) * (-2.f * kLog2e) / p.cap);
    x = copysignf(p.cap * __fdividef(1.f - e, 1.f + e), x) + x * 0.f;  // (NaN stays NaN)
  }
  return (x - slope * static_cast<float>(abs(distance))) * kLog2e;
}

// One row by the formula, a position at a time, by a warp.
template <int D, KvType KIND>
__device__ __forceinline__ void PlainRow(const KvRowsParams& p, int table_row, int head, int64_t q_at, float slope, int pos,
                                         int from, int to, float (&acc)[D / 32], float& m, float& l) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  float x[N];
  l = 0.f;
  m = -INFINITY;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    acc[e] = 0.f;
    x[e] = Element(p.q, p.type, q_at + lane * N + e);
    l += x[e] * 0.f;  // NaN with a NaN or an infinity in q
  }
  l = dev::WarpSum(l);
#pragma unroll 1
  for (int at = from; at < to && l == l; ++at) {
    const int page = kvd::PageOf(p.table, p.kv.n_pages, table_row, at >> p.kv.page_log2);
    if (page < 0) {
      l = kvd::Nan();
      break;
    }
    const int in = at & ((1 << p.kv.page_log2) - 1);
    const int64_t code = kvd::CodeOffset(p.kv, page, head, in);
    float k[N], v[N];
    if (KIND == KvType::kF16) {
      using Row = kvd::Pack<__half, N>;
      const Row kr = *reinterpret_cast<const Row*>(p.kv.k + code + lane * 2 * N);
      const Row vr = *reinterpret_cast<const Row*>(p.kv.v + code + lane * 2 * N);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        k[e] = __half2float(kr.v[e]);
        v[e] = __half2float(vr.v[e]);
      }
    } else {
      const int64_t scale = kvd::ScaleOffset(p.kv, page, head, in) + 2 * (lane * N / kKvGroup);
      const float dk = __half2float(*reinterpret_cast<const __half*>(p.kv.k_scale + scale));
      const float dv = __half2float(*reinterpret_cast<const __half*>(p.kv.v_scale + scale));
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = lane * N + e;
        if (KIND == KvType::kQ8) {
          k[e] = static_cast<float>(reinterpret_cast<const int8_t*>(p.kv.k + code)[i]) * dk;
          v[e] = static_cast<float>(reinterpret_cast<const int8_t*>(p.kv.v + code)[i]) * dv;
        } else {
          const int kc = reinterpret_cast<const uint8_t*>(p.kv.k + code)[i / 2] >> (4 * (i & 1)) & 15;
          const int vc = reinterpret_cast<const uint8_t*>(p.kv.v + code)[i / 2] >> (4 * (i & 1)) & 15;
          k[e] = static_cast<float>(kc - 8) * dk;
          v[e] = static_cast<float>(vc - 8) * dv;
        }
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) dot += x[e] * k[e];
    const float s = Score(p, dev::WarpSum(dot), slope, pos - at);
    const float now = fmaxf(m, s), ref = now == -INFINITY ? 0.f : now;
    const float alpha = Exp2(m - ref), w = Exp2(s - ref);
    m = now;
    l = l * alpha + w;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = acc[e] * alpha + w * v[e];
  }
}

template <int D, KvType KIND>
__global__ void __launch_bounds__(256) PlainKernel(const KvRowsParams p) {
  constexpr int N = D / 32;
  dev::GridLaunchDependents();
  dev::GridWait();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int row = static_cast<int>(item / p.n_heads), h = static_cast<int>(item % p.n_heads);
  if (row >= p.n_rows) return;
  int lo = 0, hi = p.n_lists;  // the first list that ends behind the row
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    RowEnd(p, mid) > row ? hi = mid : lo = mid + 1;
  }
  if (lo == p.n_lists || RowBegin(p, lo) > row) return;
  const int head = h / (p.n_heads / p.kv.n_kv);
  const Seen s = SeenBy(p, row);
  float acc[N], m, l;
  const float slope = p.slopes != nullptr ? p.slopes[h] : 0.f;
  const int pos = p.slopes != nullptr ? p.pos[row] : 0;
  const int64_t in_head = static_cast<int64_t>(h) * D + lane * N;
  PlainRow<D, KIND>(p, TableRow(p, lo), head, row * p.q_stride + static_cast<int64_t>(h) * D, slope, pos, s.start, s.end,
                    acc, m, l);
  if (p.prefix != nullptr && p.prefix[row] > p.prefix[RowBegin(p, lo)]) l = kvd::Nan();
  if (s.past) l = kvd::Nan();
  float f = l != 0.f ? 1.f / l : 0.f, g = 0.f;
  if (p.own != nullptr) {
    const float a = m + log2f(l), b = p.own_lse[static_cast<int64_t>(row) * p.n_heads + h];
    const float top = fmaxf(a, b), ref = top == -INFINITY ? 0.f : top;
    const float wa = Exp2(a - ref), wb = Exp2(b - ref), sum = wa + wb;
    f = sum != 0.f ? f * wa / sum : 0.f;
    g = sum != 0.f ? wb / sum : 0.f;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float y = acc[e] * f;
    if (p.own != nullptr) y += g * p.own[static_cast<int64_t>(row) * p.n_heads * D + in_head + e];
    Put(p.out, p.type, row * p.out_stride + in_head + e, y);
  }
}

template <int D, KvType KIND>
void Launch(const KvRowsParams& p, cudaStream_t s) {
  const int64_t warps = static_cast<int64_t>(p.n_rows) * p.n_heads;
  LaunchKernelArgs(reinterpret_cast<const void*>(PlainKernel<D, KIND>), dim3(static_cast<unsigned>((warps + 7) / 8)),
                   dim3(256), 0, s, true, p);
}

template <int D>
void ByKind(const KvRowsParams& p, cudaStream_t s) {
  switch (p.kv.type) {
    case KvType::kF16: return Launch<D, KvType::kF16>(p, s);
    case KvType::kQ8: return Launch<D, KvType::kQ8>(p, s);
    case KvType::kQ4: return Launch<D, KvType::kQ4>(p, s);
  }
}

}  // namespace

int64_t KvRowsWorkspace(int, int, int head_dim) { return 2ll * 160 * 256 * (head_dim + 2) * 4 + 65536; }

void LaunchKvRows(const KvRowsParams& p, cudaStream_t s) {
  p.kv.head_dim == 64 ? ByKind<64>(p, s) : ByKind<128>(p, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

}  // namespace rpgb
