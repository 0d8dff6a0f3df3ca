// k_kv_attend.cu -- attention of one new token per conversation over a paged
// key-value cache.
#include "common.h"
#include "kv_dev.cuh"

namespace rpgb {
namespace {

constexpr int kWarps = 4;

// One block per (q head, conversation): warps take positions in turn, each
// with its own running maximum and sum, joined at the end.
template <int D, KvType KIND, typename T>
__global__ void __launch_bounds__(32 * kWarps) KvAttendKernel(const KvAttendParams p) {
  constexpr int N = D / 32;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  const int seq = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = hq / (p.n_heads / p.kv.n_kv);
  const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
  const int64_t want = max(p.lens[seq], 0);
  const int len = static_cast<int>(min(want, cap));
  const int start = p.starts != nullptr ? max(p.starts[seq], 0) : 0;
  const T* qr = static_cast<const T*>(p.q) + seq * p.q_stride + static_cast<int64_t>(hq) * D;
  float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) q[e] = kvd::ToFloat(qr[lane + 32 * e]) * p.scale;
  for (int pos = start + warp; pos < len; pos += kWarps) {
    const int page = kvd::PageOf(p.table, p.kv.n_pages, seq, pos >> p.kv.page_log2);
    const int at = pos & ((1 << p.kv.page_log2) - 1);
    float k[N], v[N];
    if (page < 0) {
#pragma unroll
      for (int e = 0; e < N; ++e) k[e] = v[e] = kvd::Nan();
    } else {
      const int64_t co = kvd::CodeOffset(p.kv, page, h, at), so_ = kvd::ScaleOffset(p.kv, page, h, at);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        k[e] = kvd::Value<KIND>(p.kv.k + co, reinterpret_cast<const __half*>(p.kv.k_scale + so_), lane + 32 * e);
        v[e] = kvd::Value<KIND>(p.kv.v + co, reinterpret_cast<const __half*>(p.kv.v_scale + so_), lane + 32 * e);
      }
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) s += q[e] * k[e];
    s = dev::WarpSum(s);
    const float mn = fmaxf(m, s), ms = mn == -INFINITY ? 0.f : mn;
    const float al = expf(m - ms), w = expf(s - ms);
    l = l * al + w;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = o[e] * al + w * v[e];
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) so[warp][lane + 32 * e] = o[e];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
  if (top == -INFINITY) top = 0.f;
  float sum = 0.f, wt[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    wt[w] = expf(sm[w] - top);
    sum += wt[w] * sl[w];
  }
  T* out = static_cast<T*>(p.out) + seq * p.out_stride + static_cast<int64_t>(hq) * D;
  for (int d = threadIdx.x; d < D; d += 32 * kWarps) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w) x += wt[w] * so[w][d];
    x = sum != 0.f ? x / sum : 0.f;      // nothing seen: zero
    if (want > cap) x = kvd::Nan();      // positions past the table
    out[d] = kvd::FromFloat<T>(x);
  }
}

template <int D, KvType KIND>
void ByType(const KvAttendParams& p, cudaStream_t s) {
  const dim3 grid(p.table.n_seq, p.n_heads);
  switch (p.type) {
    case ElemType::kF32: KvAttendKernel<D, KIND, float><<<grid, 32 * kWarps, 0, s>>>(p); return;
    case ElemType::kF16: KvAttendKernel<D, KIND, __half><<<grid, 32 * kWarps, 0, s>>>(p); return;
    case ElemType::kBF16: KvAttendKernel<D, KIND, __nv_bfloat16><<<grid, 32 * kWarps, 0, s>>>(p); return;
  }
}
template <int D>
void ByKind(const KvAttendParams& p, cudaStream_t s) {
  switch (p.kv.type) {
    case KvType::kF16: return ByType<D, KvType::kF16>(p, s);
    case KvType::kQ8: return ByType<D, KvType::kQ8>(p, s);
    case KvType::kQ4: return ByType<D, KvType::kQ4>(p, s);
  }
}

}  // namespace

int64_t KvAttendWorkspace(int64_t n_seq, int n_heads, int n_kv, int head_dim) {
  const int group = n_heads / n_kv, chunks = (group + kKvMaxQueries - 1) / kKvMaxQueries;
  const int64_t counters = (n_seq * n_kv * chunks * 4 + 255) / 256 * 256;
  return counters + static_cast<int64_t>(2 * kKvMaxBlocks) * kKvMaxQueries * (head_dim + 2) * 4;
}

void LaunchKvAttend(const KvAttendParams& p, cudaStream_t s) {
  p.kv.head_dim == 64 ? ByKind<64>(p, s) : ByKind<128>(p, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

}  // namespace rpgb
