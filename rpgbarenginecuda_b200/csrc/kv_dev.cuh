// kv_dev.cuh -- device helpers of the paged key-value cache kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "kernels.cuh"
#include "kv.h"

// The kernels of the paged cache start before the stream's previous kernel has
// ended and wait for it; what it may have written is read by plain loads after
// the wait, not by the read-only path, which promises nothing about such data.

namespace rpgb {
namespace kvd {

__device__ __forceinline__ float Nan() { return __uint_as_float(0x7FC00000u); }

// Pool page of position `pos` of conversation `seq`, or -1 where the table has none.
__device__ __forceinline__ int PageOf(const KvTable& t, int n_pages, int seq, int64_t page) {
  if (seq < 0 || seq >= t.n_seq || page >= t.max_pages) return -1;
  const int id = t.pages[seq * t.stride + page];
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
// Eight values, 16 bytes at a time.
template <typename T>
__device__ __forceinline__ void Load8(const T* p, float (&x)[8]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < 8; j += N) {
    const Pack<T, N> r = *reinterpret_cast<const Pack<T, N>*>(p + j);
#pragma unroll
    for (int i = 0; i < N; ++i) x[j + i] = ToFloat(r.v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void Store8(T* p, const float (&x)[8]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < 8; j += N) {
    Pack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = FromFloat<T>(x[j + i]);
    *reinterpret_cast<Pack<T, N>*>(p + j) = r;
  }
}

// Eight values as they are in memory, to be converted later.
template <typename T>
struct Raw8 {
  static constexpr int N = sizeof(T) / 2;
  uint4 w[N];
  __device__ __forceinline__ void Load(const T* p) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = reinterpret_cast<const uint4*>(p)[j];
  }
  __device__ __forceinline__ void Floats(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const Pack<T, 8 / N> r = *reinterpret_cast<const Pack<T, 8 / N>*>(&w[j]);
#pragma unroll
      for (int i = 0; i < 8 / N; ++i) x[j * (8 / N) + i] = ToFloat(r.v[i]);
    }
  }
};

// 32 bytes, a whole sector, in one store.
__device__ __forceinline__ void Store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ uint32_t HalfBits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 BitsHalf(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// 1024 + u as f16 is 0x6400 | u for u < 1024, so a code in the low bits of
// 0x6400 becomes the integer it stands for by one exact subtraction (or, four
// bits up, one exact multiply-add).
__device__ __forceinline__ uint32_t SubHalf(uint32_t x, uint32_t bias) {
  return HalfBits(__hsub2(BitsHalf(x), BitsHalf(bias)));
}
// The 0x6400 pair comes to the kernels as an argument: as a constant beside
// the mask it would take a second instruction, since one may hold a single
// literal.
constexpr uint32_t kMagic = 0x64006400u;
constexpr uint32_t kBias8 = 0x64806480u;  // 1024 + 128
constexpr uint32_t kBias4 = 0x64086408u;  // 1024 + 8
template <uint32_t MASK>
__device__ __forceinline__ uint32_t MaskOr(uint32_t w, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(magic));  // (w & MASK) | magic
  return r;
}
// The 4-bit codes 0 and 4 (1 and 5) of a word as integers.
__device__ __forceinline__ uint32_t Low4(uint32_t w, uint32_t magic) {
  return SubHalf(MaskOr<0x000F000Fu>(w, magic), kBias4);
}
__device__ __forceinline__ uint32_t High4(uint32_t w, uint32_t magic) {  // (1024 + 16 u) / 16 - 72 = u - 8
  return HalfBits(
      __hfma2(BitsHalf(MaskOr<0x00F000F0u>(w, magic)), BitsHalf(0x2C002C00u), BitsHalf(0xD480D480u)));
}

// Sixteen consecutive values of a cache row.  An integer of 8 bits times an
// f16 scale is exact in f32, so one f16 product rounds as the f32 product
// rounded to f16 does.
template <KvType KIND>
struct Codes16 {
  static constexpr int kWords = KIND == KvType::kF16 ? 8 : (KIND == KvType::kQ8 ? 4 : 2);
  uint32_t w[kWords];
  __device__ __forceinline__ void Load(const char* row, int i) {
    if (KIND == KvType::kQ4) {
      const uint2 x = *reinterpret_cast<const uint2*>(row + i / 2);
      w[0] = x.x;
      w[1] = x.y;
    } else {
#pragma unroll
      for (int j = 0; j < kWords / 4; ++j) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + i * (KIND == KvType::kF16 ? 2 : 1) + 16 * j);
        w[4 * j] = x.x;
        w[4 * j + 1] = x.y;
        w[4 * j + 2] = x.z;
        w[4 * j + 3] = x.w;
      }
    }
  }
  // The values before the scale, in pairs.
  __device__ __forceinline__ void Pairs(uint32_t (&y)[8], uint32_t magic) const {
    if (KIND == KvType::kF16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = w[j % kWords];
    } else if (KIND == KvType::kQ8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = w[j % kWords] ^ 0x80808080u;
        y[2 * j] = SubHalf(__byte_perm(u, magic, 0x5150), kBias8);
        y[2 * j + 1] = SubHalf(__byte_perm(u, magic, 0x5352), kBias8);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t a = Low4(w[j], magic), b = High4(w[j], magic);            // codes 0, 4; 1, 5
        const uint32_t c = Low4(w[j] >> 8, magic), d = High4(w[j] >> 8, magic);  // codes 2, 6; 3, 7
        y[4 * j] = __byte_perm(a, b, 0x5410);
        y[4 * j + 1] = __byte_perm(c, d, 0x5410);
        y[4 * j + 2] = __byte_perm(a, b, 0x7632);
        y[4 * j + 3] = __byte_perm(c, d, 0x7632);
      }
    }
  }
  // `wide`: out is a multiple of 32 bytes.
  template <typename T>
  __device__ __forceinline__ void Store(T* out, __half d, bool wide, uint32_t magic) const {
    constexpr int N = 8 * sizeof(T);  // bytes of half the values
    uint32_t y[4 * sizeof(T)], h[8];
    Pairs(h, magic);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (sizeof(T) == 2 && !IsBf16(out)) {
        y[j] = KIND == KvType::kF16 ? h[j] : HalfBits(__hmul2(BitsHalf(h[j]), __half2half2(d)));
      } else {
        float2 x = __half22float2(BitsHalf(h[j]));
        if (KIND != KvType::kF16) {
          x.x *= __half2float(d);
          x.y *= __half2float(d);
        }
        if (sizeof(T) == 2) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(x.x, x.y);
          y[j] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          y[2 * j % (4 * sizeof(T))] = __float_as_uint(x.x);
          y[(2 * j + 1) % (4 * sizeof(T))] = __float_as_uint(x.y);
        }
      }
    }
    if (wide) {
#pragma unroll
      for (int k = 0; k < 2 * N / 32; ++k) {
        uint32_t z[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = y[8 * k + j];
        Store32(reinterpret_cast<char*>(out) + 32 * k, z);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2 * N / 16; ++k) {
        reinterpret_cast<uint4*>(out)[k] = make_uint4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
      }
    }
  }
  static __device__ __forceinline__ bool IsBf16(const __nv_bfloat16*) { return true; }
  static __device__ __forceinline__ bool IsBf16(const void*) { return false; }
};

}  // namespace kvd
}  // namespace rpgb
