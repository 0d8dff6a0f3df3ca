// kv_dev.cuh -- device helpers of the paged key-value cache kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "kernels.cuh"
#include "kv.h"

namespace rpgb {
namespace kvd {

__device__ __forceinline__ float Nan() { return __uint_as_float(0x7FC00000u); }

// Pool page of position `pos` of conversation `seq`, or -1 where the table has none.
__device__ __forceinline__ int PageOf(const KvTable& t, int n_pages, int seq, int64_t page) {
  if (seq < 0 || seq >= t.n_seq || page >= t.max_pages) return -1;
  const int id = __ldg(t.pages + seq * t.stride + page);
  return static_cast<unsigned>(id) < static_cast<unsigned>(n_pages) ? id : -1;
}

// Byte offset of a position's codes / scales inside the planes.
__device__ __forceinline__ int64_t CodeOffset(const KvPages& kv, int page, int head, int at) {
  return page * kv.page_stride + head * kv.head_stride + at * kv.pos_stride;
}
__device__ __forceinline__ int64_t ScaleOffset(const KvPages& kv, int page, int head, int at) {
  return page * kv.scale_page_stride + head * kv.scale_head_stride +
         static_cast<int64_t>(at) * (2 * (kv.head_dim / kKvGroup));
}

// N consecutive elements (16-byte loads and stores where they fill one).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};
__device__ __forceinline__ float ToFloat(float x) { return x; }
__device__ __forceinline__ float ToFloat(__half x) { return __half2float(x); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T FromFloat(float x);
template <>
__device__ __forceinline__ float FromFloat<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half FromFloat<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ void Load4(const T* p, float (&x)[4]) {
  const Pack<T, 4> r = *reinterpret_cast<const Pack<T, 4>*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = ToFloat(r.v[i]);
}
template <typename T>
__device__ __forceinline__ void Store4(T* p, const float (&x)[4]) {
  Pack<T, 4> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = FromFloat<T>(x[i]);
  *reinterpret_cast<Pack<T, 4>*>(p) = r;
}

// Value `i` of a cache row (codes at `row`, its scales at `sc`).
template <KvType KIND>
__device__ __forceinline__ float Value(const char* row, const __half* sc, int i) {
  if (KIND == KvType::kF16) return __half2float(reinterpret_cast<const __half*>(row)[i]);
  const float d = __half2float(sc[i / kKvGroup]);
  if (KIND == KvType::kQ8) return static_cast<float>(reinterpret_cast<const int8_t*>(row)[i]) * d;
  const int b = reinterpret_cast<const uint8_t*>(row)[i >> 1];
  return static_cast<float>(((i & 1) ? (b >> 4) : (b & 15)) - 8) * d;
}

}  // namespace kvd
}  // namespace rpgb
