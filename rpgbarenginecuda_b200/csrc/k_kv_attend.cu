// k_kv_attend.cu -- attention of one new token per conversation over a paged
// key-value cache: o = softmax(scale q K^T) V per q head, over positions
// [start, len) of each conversation.
//
// What it has to do is read the cache once: 4 G flops per cached byte pair at
// most (G query heads share a KV head), far under what the tensor cores do in
// the time HBM takes, so the kernel is a stream of cache pages with the math
// kept off its way.
//
//  * Work.  An item is a (conversation, KV head, chunk of at most 8 query
//    heads); its positions are cut into tiles and the tiles of all items, in
//    order, are dealt evenly over a persistent grid, wherever the item borders
//    fall.  Every block finds its share from the lengths on the device, so the
//    host needs to know none, ragged batches stay balanced and one long
//    conversation fills the GPU.  An item inside one block is written at once;
//    otherwise the blocks leave (max, sum, vector) records in the workspace
//    and the last of them to finish joins them in block order.
//  * Data.  Each warp takes R consecutive positions of a tile and owns a ring
//    of shared-memory slots filled with 16-byte asynchronous copies, DEPTH
//    steps ahead of the math, across item borders.  Rows outside the range
//    are not read but filled with zeros.  16-byte chunks are permuted so that
//    every read of a tile is free of bank conflicts.
//  * Math.  S^T = K q^T and O^T += V^T P^T as m16n8k16 tensor-core products
//    with the positions (S) or value dimensions (O) as the 16 rows and 8
//    query columns, so a group of 2 to 8 query heads wastes little; tcgen05
//    has 128 rows but would need V and the converted codes staged through
//    shared or tensor memory again for a product that is not the bound.
//    Codes become exact f16 integers with two instructions per pair; a scale
//    multiplies the group's partial score (K) or the weight of its position (V).
//  * Precision.  f16 operands, f32 accumulation.  q is scaled by a power of
//    two to a largest value in [1, 2) and split into two f16 terms (one when
//    it is 16-bit, which is then exact), the softmax weights are split into
//    two f16 terms, and scaled up by 2^14 (and by the power of two above the
//    largest V scale seen) so that small ones stay normal numbers: 22 bits
//    throughout.  With at most 4 query heads the second terms ride in the
//    other 4 columns at no cost.  Each step's product starts from zero and is
//    added to the running output in f32 registers: the tensor cores truncate
//    when they add, which over a long conversation would add up.
#include <atomic>

#include "common.h"
#include "kv_dev.cuh"

namespace rpgb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWeightBits = 14;  // weights are scaled by 2^14

template <int D_, KvType KIND_, bool PACK_>
struct Cfg {
  static constexpr int D = D_;
  static constexpr KvType KIND = KIND_;
  static constexpr bool PACK = PACK_;  // at most 4 query heads: first and second terms share 8 columns
  static constexpr bool QUANT = KIND != KvType::kF16;
  static constexpr int QUERIES = PACK ? 4 : 8;
  static constexpr int R = QUANT || D == 64 ? 32 : 16;  // positions of a warp's step
  static constexpr int TILE = kWarps * R;
  static constexpr int DEPTH = KIND == KvType::kQ4 ? 3 : 2;
  static constexpr int MT = R / 16;     // 16-position tiles of a step
  static constexpr int KS = D / 16;     // 16-value slices of a head
  static constexpr int NG = QUANT ? D / kKvGroup : 1;
  static constexpr int ROW = KIND == KvType::kF16 ? 2 * D : (KIND == KvType::kQ8 ? D : D / 2);
  static constexpr int CPR = ROW / 16;  // 16-byte chunks of a row
  static constexpr int SC = QUANT ? R * NG * 2 : 0;
  static constexpr int SLOT = R * ROW + SC;
  static constexpr int RING = DEPTH * 2 * SLOT;  // per warp: K and V
  static constexpr int COMB = QUERIES * D * 4;   // per warp
  static constexpr int SMEM = kWarps * (RING + COMB);
  static constexpr int BLOCKS = PACK || D == 64 ? 3 : 2;  // resident per SM: what registers and shared memory allow
};

// Byte offset of 16-byte chunk c of row r in a tile of 128-byte lines.  The
// chunk's place in its line is permuted by the row so that the lanes of one
// load (8 rows of one chunk for ldmatrix; see LoadK / LoadV for the codes)
// touch different banks.
template <typename C, bool V>
__device__ __forceinline__ int ChunkAt(int r, int c) {
  int key;
  if (C::KIND == KvType::kF16) {
    key = r & 7;
  } else if (C::KIND == KvType::kQ8) {
    key = V ? ((r >> 1) & 3) << 1 : (C::D == 128 ? (r & 1) << 2 : 0);
  } else {
    key = V ? (C::D == 128 ? ((r >> 1) & 3) << 1 : ((r >> 2) & 1) << 1) : (C::D == 128 ? ((r >> 1) & 1) << 1 : 0);
  }
  const int q = r * C::CPR + c;
  return (q >> 3) * 128 + (((q & 7) ^ key) << 4);
}

// ------------------------------------------------------------------ instructions

__device__ __forceinline__ void CopyAsync16(uint32_t dst, const void* src, bool read) {
  const int n = read ? 16 : 0;  // the rest is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void CopyCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void CopyWait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void LdMatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void LdMatrixT(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t Transposed(uint32_t x) {  // of an 8 x 8 matrix of 16-bit values
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void Mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t Lds32(uint32_t a) {
  uint32_t x;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
  return x;
}
__device__ __forceinline__ uint32_t Lds16(uint32_t a) {
  uint16_t x;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(a) : "memory");
  return x;
}
__device__ __forceinline__ uint2 Lds64(uint32_t a) {
  uint2 x;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(a) : "memory");
  return x;
}
__device__ __forceinline__ uint4 Lds128(uint32_t a) {
  uint4 x;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(a) : "memory");
  return x;
}
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t HalfBits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 BitsHalf(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t PackHalf(float lo, float hi) { return HalfBits(__floats2half2_rn(lo, hi)); }

// 1024 + u as f16 is 0x6400 | u for u < 1024, so a code in the low bits of
// 0x6400 becomes the integer it stands for by one exact subtraction (or, four
// bits up, one exact multiply-add).
__device__ __forceinline__ uint32_t SubHalf(uint32_t x, uint32_t bias) {
  return HalfBits(__hsub2(BitsHalf(x), BitsHalf(bias)));
}
constexpr uint32_t kMagic = 0x64006400u;
constexpr uint32_t kMagicByte = 0x64u;
constexpr uint32_t kBias8 = 0x64806480u;  // 1024 + 128
constexpr uint32_t kBias4 = 0x64086408u;  // 1024 + 8
__device__ __forceinline__ uint32_t Low4(uint32_t w) { return SubHalf((w & 0x000F000Fu) | kMagic, kBias4); }
__device__ __forceinline__ uint32_t High4(uint32_t w) {  // (1024 + 16 u) / 16 - 72 = u - 8
  return HalfBits(__hfma2(BitsHalf((w & 0x00F000F0u) | kMagic), BitsHalf(0x2C002C00u), BitsHalf(0xD480D480u)));
}

// ------------------------------------------------------------------ work

// The positions of a conversation: [start, len), tiles counted from `base`.
struct Span {
  int start, len, base, tiles;
};
template <typename C>
__device__ __forceinline__ Span SpanOf(const KvAttendParams& p, int seq) {
  const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
  Span s;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(__ldg(p.lens + seq), 0)), cap));
  s.start = p.starts != nullptr ? max(__ldg(p.starts + seq), 0) : 0;
  if (s.start >= s.len) s.start = s.len = 0;
  s.base = s.start & ~15;  // a 16-position unit lies in one page
  s.tiles = max(1, (s.len - s.base + C::TILE - 1) / C::TILE);  // an empty item still writes its zeros
  return s;
}

// A place in the sequence of tiles: conversation, item of it (KV head and
// query chunk), tile of the item.
template <typename C>
struct Cursor {
  int seq, item, tile;
  Span span;
  __device__ __forceinline__ void Next(const KvAttendParams& p, int items) {
    if (++tile < span.tiles) return;
    tile = 0;
    if (++item < items) return;
    item = 0;
    if (++seq < p.table.n_seq) span = SpanOf<C>(p, seq);
  }
};

// One step of a warp: R positions, their memory, what of them is in range.
struct Step {
  int lo, hi;                // rows [lo, hi) are in range
  int64_t off[2], soff[2];   // code and scale offsets of the 16-row halves
  bool have[2];              // the half has rows in range, and a page
  uint32_t bad;              // bit h: half h has rows in range but no page
};
template <typename C>
__device__ __forceinline__ Step StepAt(const KvAttendParams& p, const Cursor<C>& c, int warp, int chunks, bool more) {
  Step s;
  const int pos = c.span.base + c.tile * C::TILE + warp * C::R;
  s.lo = c.span.start - pos;
  s.hi = more ? c.span.len - pos : 0;
  s.bad = 0;
  const int head = c.item / chunks;
  const int mask = (1 << p.kv.page_log2) - 1;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s.off[h] = s.soff[h] = 0;
    s.have[h] = false;
    if (h < C::MT && s.hi > 16 * h && s.lo < 16 * h + 16) {
      const int at = pos + 16 * h;
      const int page = kvd::PageOf(p.table, p.kv.n_pages, c.seq, at >> p.kv.page_log2);
      if (page >= 0) {
        s.have[h] = true;
        s.off[h] = kvd::CodeOffset(p.kv, page, head, at & mask);
        if (C::QUANT) s.soff[h] = kvd::ScaleOffset(p.kv, page, head, at & mask);
      } else {
        s.bad |= 1u << h;
      }
    }
  }
  return s;
}
template <typename C, bool V>
__device__ __forceinline__ void Issue(const KvAttendParams& p, const Step& s, uint32_t slot, int lane) {
  const char* plane = V ? p.kv.v : p.kv.k;
  if (s.have[0] || s.have[1]) {
#pragma unroll
    for (int j = 0; j < C::R * C::CPR / 32; ++j) {
      constexpr int kRows = 32 / C::CPR;  // rows of one copy instruction: all in one half
      const int r = lane / C::CPR + kRows * j, c = lane % C::CPR;
      const int h = kRows * j / 16;
      const bool read = s.have[h] && r >= s.lo && r < s.hi;
      const char* src = plane + s.off[h] + (r & 15) * p.kv.pos_stride + c * 16;
      CopyAsync16(slot + ChunkAt<C, V>(r, c), read ? src : plane, read);
    }
    if (C::QUANT) {  // a half's scales are dense: 16 rows of 2 NG bytes
      constexpr int kPer = 16 * C::NG * 2 / 16;
      if (lane < C::MT * kPer) {
        const char* sp = V ? p.kv.v_scale : p.kv.k_scale;
        const bool second = lane >= kPer, read = second ? s.have[1] : s.have[0];
        CopyAsync16(slot + C::R * C::ROW + lane * 16,
                    read ? sp + (second ? s.soff[1] : s.soff[0]) + (lane % kPer) * 16 : sp, read);
      }
    }
  }
  CopyCommit();
}

// ------------------------------------------------------------------ operands

// K of 16 positions, 16-value slice ks, as the A fragment (rows = positions).
// Code tiles: lane t of a row takes 16 consecutive values of a 64-value group
// (they are a slice's columns in that order; LoadQ takes q the same way).
template <typename C>
struct KRows {
  uint4 w[2];  // q8: 16 codes of rows g and g + 8; q4: .x, .y
  __device__ __forceinline__ void Load(uint32_t tile, int mt, int gp, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 16 * mt + 8 * i + g;
      if (C::KIND == KvType::kQ8) {
        w[i] = Lds128(tile + ChunkAt<C, false>(r, 4 * gp + t));
      } else {
        const uint2 x = Lds64(tile + ChunkAt<C, false>(r, 2 * gp + (t >> 1)) + (t & 1) * 8);
        w[i].x = x.x;
        w[i].y = x.y;
      }
    }
  }
  __device__ __forceinline__ void Fragment(uint32_t (&a)[4], int j) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (C::KIND == KvType::kQ8) {
        const uint32_t u = (j == 0 ? w[i].x : j == 1 ? w[i].y : j == 2 ? w[i].z : w[i].w) ^ 0x80808080u;
        a[i] = SubHalf(__byte_perm(u, kMagicByte, 0x4140), kBias8);
        a[2 + i] = SubHalf(__byte_perm(u, kMagicByte, 0x4342), kBias8);
      } else {
        const uint32_t u = (j < 2 ? w[i].x : w[i].y) >> ((j & 1) * 8);
        a[i] = Low4(u);
        a[2 + i] = High4(u);
      }
    }
  }
};

// V^T of a 64-value group and 16 positions as A fragments of four 16-row
// tiles (rows = values).  Lane g takes values 8 g .. 8 g + 7 of the group:
// row g of tile i is value 8 g + i, row g + 8 value 8 g + 4 + i.
template <typename C>
__device__ __forceinline__ void VFragments(uint32_t (&a)[4][4], uint32_t tile, int kt, int gp, int lane) {
  const int g = lane >> 2, t = lane & 3;
  uint32_t lo[4], hi[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 16 * kt + 2 * t + (j & 1) + 8 * (j >> 1);
    if (C::KIND == KvType::kQ8) {
      const uint2 x = Lds64(tile + ChunkAt<C, true>(r, 4 * gp + (g >> 1)) + (g & 1) * 8);
      lo[j] = x.x;
      hi[j] = x.y;
    } else {
      lo[j] = Lds32(tile + ChunkAt<C, true>(r, 2 * gp + (g >> 2)) + (g & 3) * 4);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // position pairs 2 t, 2 t + 1 and 8 further
    if (C::KIND == KvType::kQ8) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t w0 = m ? hi[2 * k] : lo[2 * k], w1 = m ? hi[2 * k + 1] : lo[2 * k + 1];
        const uint32_t x = __byte_perm(w0, w1, 0x5140) ^ 0x80808080u, y = __byte_perm(w0, w1, 0x7362) ^ 0x80808080u;
        a[0][2 * k + m] = SubHalf(__byte_perm(x, kMagicByte, 0x4140), kBias8);
        a[1][2 * k + m] = SubHalf(__byte_perm(x, kMagicByte, 0x4342), kBias8);
        a[2][2 * k + m] = SubHalf(__byte_perm(y, kMagicByte, 0x4140), kBias8);
        a[3][2 * k + m] = SubHalf(__byte_perm(y, kMagicByte, 0x4342), kBias8);
      }
    } else {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t x = __byte_perm(lo[2 * k], lo[2 * k + 1], m ? 0x7632 : 0x5410), y = x >> 8;
        a[0][2 * k + m] = Low4(x);
        a[1][2 * k + m] = High4(x);
        a[2][2 * k + m] = Low4(y);
        a[3][2 * k + m] = High4(y);
      }
    }
  }
}

// Value of a head that column pair b (0, 1), element e of lane t's B fragment
// of slice ks stands for: the order LdMatrix or KRows gives K in.
template <typename C>
__device__ __forceinline__ constexpr int ValueOf(int ks, int b, int e, int t) {
  return C::KIND == KvType::kF16 ? 16 * ks + 8 * b + 2 * t + e
         : C::KIND == KvType::kQ8
             ? 64 * (ks >> 2) + 16 * t + 4 * (ks & 3) + 2 * b + e
             : 64 * (ks >> 2) + 16 * t + 8 * ((ks & 3) >> 1) + 2 * (ks & 1) + b + 4 * e;
}

template <typename C, typename T>
__device__ __forceinline__ void ReadQ(float (&x)[C::KS][2][2], const T* row, int t) {
#pragma unroll
  for (int ks = 0; ks < C::KS; ++ks) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int e = 0; e < 2; ++e) x[ks][b][e] = kvd::ToFloat(row[ValueOf<C>(ks, b, e, t)]);
    }
  }
}

__device__ __forceinline__ float LaneQuadMax(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
}

// ------------------------------------------------------------------ kernel

template <typename C>
__global__ void __launch_bounds__(kThreads, C::BLOCKS) KvAttendKernel(const KvAttendParams p) {
  constexpr int D = C::D;
  extern __shared__ __align__(128) char smem[];
  __shared__ float s_m[kWarps][8], s_l[kWarps][8];
  __shared__ long long s_sum[kWarps + 1], s_begin;
  __shared__ int s_seq, s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / p.kv.n_kv;
  const int chunks = (group + kKvMaxQueries - 1) / kKvMaxQueries;
  const int per_chunk = (group + chunks - 1) / chunks;
  const int items = p.kv.n_kv * chunks;

  // This block's share of the tiles: prefix sums of the conversations' tiles,
  // a run of conversations per thread.
  const int run = (p.table.n_seq + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int i = 0; i < run; ++i) {
    const int s = tid * run + i;
    if (s < p.table.n_seq) mine += static_cast<long long>(SpanOf<C>(p, s).tiles) * items;
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) s_sum[warp] = upto;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) upto += total;
    total += s_sum[w];
  }
  const long long blocks = min(static_cast<long long>(gridDim.x), total);
  if (blockIdx.x >= blocks) return;
  const long long first = total * blockIdx.x / blocks, last = total * (blockIdx.x + 1) / blocks;
  if (first >= upto - mine && first < upto) {
    long long at = upto - mine;
    int s = tid * run;
    for (;; ++s) {
      const long long n = static_cast<long long>(SpanOf<C>(p, s).tiles) * items;
      if (first < at + n) break;
      at += n;
    }
    s_seq = s;
    s_begin = at;
  }
  __syncthreads();
  Cursor<C> use;
  use.seq = s_seq;
  use.span = SpanOf<C>(p, use.seq);
  use.item = static_cast<int>((first - s_begin) / use.span.tiles);
  use.tile = static_cast<int>((first - s_begin) % use.span.tiles);
  Cursor<C> fill = use;

  const uint32_t ring = dev::SmemAddr(smem) + warp * C::RING;
  float* comb = reinterpret_cast<float*>(smem + kWarps * C::RING);
  uint32_t bad = 0;  // two bits per step in flight
  long long to_fill = last - first;
#pragma unroll
  for (int d = 0; d < C::DEPTH; ++d) {
    const Step s = StepAt<C>(p, fill, warp, chunks, to_fill > 0);
    Issue<C, false>(p, s, ring + (2 * d) * C::SLOT, lane);
    Issue<C, true>(p, s, ring + (2 * d + 1) * C::SLOT, lane);
    bad = bad << 2 | s.bad;
    if (--to_fill > 0) fill.Next(p, items);
  }

  uint32_t qh[C::KS][2], ql[C::PACK ? 1 : C::KS][2];
  const bool two_terms = p.type == ElemType::kF32;
  float cs[2];                 // from products of the f16 terms to scores in log2 units
  float m[2], l[2];            // of columns 2 t and 2 t + 1
  float acc[D / 16][4];
  int nu = 0;                  // biased exponent of the power of two over the V scales seen
  int seg = 0;                 // first tile of the item in this block
  bool fresh = true;
  int slot = 0;

  for (long long at = first; at < last; ++at) {
    Step next = StepAt<C>(p, fill, warp, chunks, to_fill > 0);
    const int chunk = use.item % chunks;
    const int queries = min(per_chunk, group - chunk * per_chunk);
    const int64_t col = (static_cast<int64_t>(use.item / chunks) * group + chunk * per_chunk) * D;
    if (fresh) {
      fresh = false;
      seg = use.tile;
      const int qi = C::PACK ? g & 3 : g;
      float x[C::KS][2][2] = {};
      if (qi < queries) {
        const int64_t o = use.seq * p.q_stride + col + qi * D;
        switch (p.type) {
          case ElemType::kF32: ReadQ<C>(x, static_cast<const float*>(p.q) + o, t); break;
          case ElemType::kF16: ReadQ<C>(x, static_cast<const __half*>(p.q) + o, t); break;
          case ElemType::kBF16: ReadQ<C>(x, static_cast<const __nv_bfloat16*>(p.q) + o, t); break;
        }
      }
      float top = 0.f;
#pragma unroll
      for (int ks = 0; ks < C::KS; ++ks) {
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[ks][e >> 1][e & 1]));
      }
      top = LaneQuadMax(top);
      // 2^-e of the largest value's exponent (kept in f32's normal range)
      const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 1), 253);
      const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
      const float up = __uint_as_float(static_cast<uint32_t>(e) << 23) * (p.scale * kLog2e);
#pragma unroll
      for (int ks = 0; ks < C::KS; ++ks) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float u = x[ks][b][0] * down, v = x[ks][b][1] * down;
          const uint32_t h = PackHalf(u, v);
          const float2 f = __half22float2(BitsHalf(h));
          const uint32_t lo = PackHalf(u - f.x, v - f.y);
          if (C::PACK) {
            qh[ks][b] = two_terms && g >= 4 ? lo : h;
          } else {
            qh[ks][b] = h;
            ql[ks][b] = lo;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        cs[c] = __shfl_sync(0xFFFFFFFFu, up, 4 * (C::PACK ? (2 * t + c) & 3 : 2 * t + c));
        m[c] = -INFINITY;
        l[c] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
      }
      nu = 127 - 25;
    }

    const int pos = use.span.base + use.tile * C::TILE + warp * C::R;
    const int lo = use.span.start - pos, hi = use.span.len - pos;
    const bool work = lo < C::R && hi > 0;
    const uint32_t bad_now = (bad >> (2 * (C::DEPTH - 1))) & 3u;
    const uint32_t kslot = ring + (2 * slot) * C::SLOT, vslot = kslot + C::SLOT;

    // ---- scores
    CopyWait<2 * C::DEPTH - 1>();
    __syncwarp();
    float s[C::MT][4];
    if (work) {
#pragma unroll
      for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
        for (int c = 0; c < 4; ++c) s[mt][c] = 0.f;
        if (!C::QUANT) {
#pragma unroll
          for (int ks = 0; ks < C::KS; ++ks) {
            uint32_t a[4];
            LdMatrix(a, kslot + ChunkAt<C, false>(16 * mt + (lane & 15), 2 * ks + (lane >> 4)));
            Mma(s[mt], a, qh[ks][0], qh[ks][1]);
            if (!C::PACK && two_terms) Mma(s[mt], a, ql[C::PACK ? 0 : ks][0], ql[C::PACK ? 0 : ks][1]);
          }
        } else {
#pragma unroll
          for (int gp = 0; gp < C::NG; ++gp) {
            KRows<C> rows;
            rows.Load(kslot, mt, gp, lane);
            float part[4] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int ks = 4 * gp + j;
              uint32_t a[4];
              rows.Fragment(a, j);
              Mma(part, a, qh[ks][0], qh[ks][1]);
              if (!C::PACK && two_terms) Mma(part, a, ql[C::PACK ? 0 : ks][0], ql[C::PACK ? 0 : ks][1]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float d = __half2float(__ushort_as_half(static_cast<unsigned short>(
                  Lds16(kslot + C::R * C::ROW + ((16 * mt + 8 * i + g) * C::NG + gp) * 2))));
              s[mt][2 * i] += part[2 * i] * d;
              s[mt][2 * i + 1] += part[2 * i + 1] * d;
            }
          }
        }
        if (C::PACK && two_terms) {
#pragma unroll
          for (int c = 0; c < 4; ++c) s[mt][c] += __shfl_xor_sync(0xFFFFFFFFu, s[mt][c], 2);
        }
      }
    }
    __syncwarp();
    Issue<C, false>(p, next, kslot, lane);

    // ---- weights
    float alpha[2] = {1.f, 1.f};
    if (work) {
      float mx[2] = {-INFINITY, -INFINITY};
      const bool edge = lo > 0 || hi < C::R || bad_now != 0;
#pragma unroll
      for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = s[mt][c] * cs[c & 1];
          if (edge) {
            const int r = 16 * mt + 8 * (c >> 1) + g;
            if ((bad_now >> mt) & 1) v = kvd::Nan();
            if (r < lo || r >= hi) v = -INFINITY;
          }
          s[mt][c] = v;
          mx[c & 1] = fmaxf(mx[c & 1], v);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xFFFFFFFFu, mx[c], o));
        const float mn = fmaxf(m[c], mx[c]);
        const float ref = mn == -INFINITY ? 0.f : mn;
        alpha[c] = Exp2(m[c] - ref);
        m[c] = mn;
        float sum = 0.f;
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float w = Exp2(s[mt][2 * i + c] - ref);
            s[mt][2 * i + c] = w;
            sum += w;
          }
        }
        l[c] = l[c] * alpha[c] + sum;
      }
    }

    // ---- values
    CopyWait<2 * C::DEPTH - 1>();
    __syncwarp();
    if (work) {
      float ws[C::MT][2][C::NG];  // weight factors of the lane's rows
      if (!C::QUANT) {
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) ws[mt][0][0] = ws[mt][1][0] = static_cast<float>(1 << kWeightBits);
      } else {
        uint32_t top = 0;
        const bool edge = lo > 0 || hi < C::R;
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 16 * mt + 8 * i + g;
#pragma unroll
            for (int gp = 0; gp < C::NG; ++gp) {
              uint32_t d = Lds16(vslot + C::R * C::ROW + (r * C::NG + gp) * 2);
              if (edge && (r < lo || r >= hi)) d = 0;  // a scale out of range may be anything
              top = max(top, d & 0x7FFFu);
              ws[mt][i][gp] = __half2float(__ushort_as_half(static_cast<unsigned short>(d)));
            }
          }
        }
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        const int e = min(static_cast<int>(__float_as_uint(__half2float(
                              __ushort_as_half(static_cast<unsigned short>(top)))) >> 23), 127 + 16) + 1;
        if (e > nu) {
          const float f = __uint_as_float(static_cast<uint32_t>(127 + nu - e) << 23);
          alpha[0] *= f;
          alpha[1] *= f;
          nu = e;
        }
        const float up = __uint_as_float(static_cast<uint32_t>(127 + kWeightBits + 127 - nu) << 23);
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int gp = 0; gp < C::NG; ++gp) ws[mt][i][gp] *= up;
          }
        }
      }
#pragma unroll
      for (int gp = 0; gp < C::NG; ++gp) {
        uint32_t b[C::MT][2][C::PACK ? 1 : 2];
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float u = s[mt][2 * i] * ws[mt][i][gp], v = s[mt][2 * i + 1] * ws[mt][i][gp];
            const uint32_t h = PackHalf(u, v);
            const float2 f = __half22float2(BitsHalf(h));
            const uint32_t r = PackHalf(u - f.x, v - f.y);
            if (C::PACK) {
              b[mt][i][0] = Transposed(t >= 2 ? r : h);
            } else {
              b[mt][i][0] = Transposed(h);
              b[mt][i][C::PACK ? 0 : 1] = Transposed(r);
            }
          }
        }
        constexpr int kTiles = C::QUANT ? 4 : D / 16;
        if (C::QUANT) {
          float part[4][4] = {};
#pragma unroll
          for (int kt = 0; kt < C::MT; ++kt) {
            uint32_t a[4][4];
            VFragments<C>(a, vslot, kt, gp, lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
              for (int n = 0; n < (C::PACK ? 1 : 2); ++n) Mma(part[i], a[i], b[kt][0][n], b[kt][1][n]);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              acc[4 * gp + i][c] = acc[4 * gp + i][c] * alpha[c & 1] + part[i][c];
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            float part[4] = {};
#pragma unroll
            for (int kt = 0; kt < C::MT; ++kt) {
              uint32_t a[4];
              LdMatrixT(a, vslot + ChunkAt<C, true>(16 * kt + (lane & 7) + ((lane >> 4) << 3),
                                                    2 * i + ((lane >> 3) & 1)));
#pragma unroll
              for (int n = 0; n < (C::PACK ? 1 : 2); ++n) Mma(part, a, b[kt][0][n], b[kt][1][n]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][c] = acc[i][c] * alpha[c & 1] + part[c];
          }
        }
      }
    }
    __syncwarp();
    Issue<C, true>(p, next, vslot, lane);
    bad = bad << 2 | next.bad;
    if (--to_fill > 0) fill.Next(p, items);
    slot = slot + 1 == C::DEPTH ? 0 : slot + 1;

    // ---- the end of the item, or of this block's share of it
    if (use.tile + 1 == use.span.tiles || at + 1 == last) {
      fresh = true;
      const float down = C::QUANT ? __uint_as_float(static_cast<uint32_t>(nu - kWeightBits) << 23) : 1.f / (1 << kWeightBits);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[c] += __shfl_xor_sync(0xFFFFFFFFu, l[c], o);
      }
      float* mineq = comb + warp * (C::COMB / 4);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = acc[i][c];
          if (C::PACK) v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
          const int value = C::QUANT ? 64 * (i >> 2) + 8 * g + 4 * (c >> 1) + (i & 3) : 16 * i + 8 * (c >> 1) + g;
          if (!C::PACK || t < 2) mineq[(2 * t + (c & 1)) * D + value] = v * down;
        }
      }
      if (g == 0 && (!C::PACK || t < 2)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          s_m[warp][2 * t + c] = m[c];
          s_l[warp][2 * t + c] = l[c];
        }
      }
      __syncthreads();
      const bool whole = seg == 0 && use.tile + 1 == use.span.tiles;
      const int64_t out = use.seq * p.out_stride + col;
      const bool past = static_cast<int64_t>(max(__ldg(p.lens + use.seq), 0)) >
                        (static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2);
      // The warps' shares joined: value i of the item's queries, its sum, its maximum.
      auto join = [&](int i, float& sum, float& top) {
        const int q = i / D;
        top = s_m[0][q];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][q]);
        const float ref = top == -INFINITY ? 0.f : top;
        float v = 0.f;
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = Exp2(s_m[w][q] - ref);
          v += f * comb[w * (C::COMB / 4) + i];
          sum += f * s_l[w][q];
        }
        return v;
      };
      bool finish = whole;
      if (!whole) {
        // This block's record: one for an item that began in an earlier block,
        // one for an item that begins here.  Blocks b0 .. b1 hold the parts.
        const long long item0 = at - use.tile, item1 = item0 + use.span.tiles - 1;
        const int b0 = static_cast<int>(((item0 + 1) * blocks - 1) / total);
        const int b1 = static_cast<int>(((item1 + 1) * blocks - 1) / total);
        constexpr int kRecord = kKvMaxQueries * (D + 2);
        float* records = reinterpret_cast<float*>(static_cast<char*>(p.workspace) +
                                                  (static_cast<int64_t>(p.table.n_seq) * items * 4 + 255) / 256 * 256);
        auto record = [&](int b) { return records + (2 * b + (b == b0 ? 1 : 0)) * kRecord; };
        unsigned* count = static_cast<unsigned*>(p.workspace) + static_cast<int64_t>(use.seq) * items + use.item;
        float* rec = record(blockIdx.x);
        for (int i = tid; i < queries * D; i += kThreads) {
          float sum, top;
          rec[i] = join(i, sum, top);
          if (i % D == 0) {
            rec[kKvMaxQueries * D + i / D] = top;
            rec[kKvMaxQueries * (D + 1) + i / D] = sum;
          }
        }
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(count, 1u) == static_cast<unsigned>(b1 - b0);
        __syncthreads();
        finish = s_last != 0;
        if (finish) {
          // The last block joins all records: warp w adds up records b0 + w,
          // b0 + w + 4, ... under the maximum of all, in that order.
          __threadfence();
          if (tid == 0) *count = 0;
          constexpr int kVec = C::QUERIES * D / 128;  // float4 of a lane
          float top[C::QUERIES], sum[C::QUERIES];
          float4 v[kVec];
#pragma unroll
          for (int q = 0; q < C::QUERIES; ++q) {
            top[q] = -INFINITY;
            sum[q] = 0.f;
          }
#pragma unroll
          for (int k = 0; k < kVec; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int b = b0 + lane; b <= b1; b += 32) {
            const float* r = record(b) + kKvMaxQueries * D;
#pragma unroll
            for (int q = 0; q < C::QUERIES; ++q) {
              if (q < queries) top[q] = fmaxf(top[q], __ldcg(r + q));
            }
          }
#pragma unroll
          for (int q = 0; q < C::QUERIES; ++q) top[q] = dev::WarpMax(top[q]);
#pragma unroll 2
          for (int b = b0 + warp; b <= b1; b += kWarps) {
            const float* r = record(b);
            float f[C::QUERIES];
#pragma unroll
            for (int q = 0; q < C::QUERIES; ++q) {
              f[q] = 0.f;
              if (q < queries) {
                f[q] = Exp2(__ldcg(r + kKvMaxQueries * D + q) - (top[q] == -INFINITY ? 0.f : top[q]));
                sum[q] += f[q] * __ldcg(r + kKvMaxQueries * (D + 1) + q);
              }
            }
#pragma unroll
            for (int k = 0; k < kVec; ++k) {
              const int q = k * 128 / D + (D == 128 ? 0 : lane >> 4);
              if (q < queries) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(r) + 32 * k + lane);
                const float fq = D == 128 ? f[k % C::QUERIES] : (lane >= 16 ? f[(2 * k + 1) % C::QUERIES] : f[(2 * k) % C::QUERIES]);
                v[k].x += fq * x.x;
                v[k].y += fq * x.y;
                v[k].z += fq * x.z;
                v[k].w += fq * x.w;
              }
            }
          }
#pragma unroll
          for (int k = 0; k < kVec; ++k) reinterpret_cast<float4*>(mineq)[32 * k + lane] = v[k];
          if (lane == 0) {
#pragma unroll
            for (int q = 0; q < C::QUERIES; ++q) {
              s_m[warp][q] = top[q];
              s_l[warp][q] = sum[q];
            }
          }
          __syncthreads();
        }
      }
      if (finish) {
        for (int i = tid; i < queries * D; i += kThreads) {
          float sum, top;
          float v = join(i, sum, top);
          v = sum != 0.f ? v / sum : 0.f;  // nothing in range: zero
          if (past) v = kvd::Nan();
          switch (p.type) {
            case ElemType::kF32: static_cast<float*>(p.out)[out + i] = v; break;
            case ElemType::kF16: static_cast<__half*>(p.out)[out + i] = __float2half_rn(v); break;
            case ElemType::kBF16: static_cast<__nv_bfloat16*>(p.out)[out + i] = __float2bfloat16_rn(v); break;
          }
        }
      }
      __syncthreads();  // the next item writes the join area again
    }
    use.Next(p, items);
  }
  CopyWait<0>();
}

template <int D, KvType KIND, bool PACK>
void Launch(const KvAttendParams& p, int chunks, cudaStream_t s) {
  using C = Cfg<D, KIND, PACK>;
  static std::atomic<int> resident[64];  // blocks the device holds at once
  int dev = 0;
  RPGB_CUDA(cudaGetDevice(&dev));
  RPGB_CHECK(dev < 64, "kv: device %d", dev);
  int grid = resident[dev].load(std::memory_order_acquire);
  if (grid == 0) {
    int sms = 0, per = 0;
    RPGB_CUDA(cudaFuncSetAttribute(KvAttendKernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    RPGB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    RPGB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, KvAttendKernel<C>, kThreads, C::SMEM));
    RPGB_CHECK(per > 0, "kv: the attend kernel does not fit device %d", dev);
    grid = sms * per < kKvMaxBlocks ? sms * per : kKvMaxBlocks;
    resident[dev].store(grid, std::memory_order_release);
  }
  // no more blocks than tiles there can be
  const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
  const int64_t tiles = ((cap + 15) / C::TILE + 1) * p.kv.n_kv * chunks;
  if (tiles < grid && tiles * p.table.n_seq < grid) grid = static_cast<int>(tiles * p.table.n_seq);
  KvAttendKernel<C><<<grid, kThreads, C::SMEM, s>>>(p);
}

template <int D, KvType KIND>
void ByQueries(const KvAttendParams& p, cudaStream_t s) {
  const int group = p.n_heads / p.kv.n_kv, chunks = (group + kKvMaxQueries - 1) / kKvMaxQueries;
  if (group <= 4) {
    Launch<D, KIND, true>(p, chunks, s);
  } else {
    Launch<D, KIND, false>(p, chunks, s);
  }
}
template <int D>
void ByKind(const KvAttendParams& p, cudaStream_t s) {
  switch (p.kv.type) {
    case KvType::kF16: return ByQueries<D, KvType::kF16>(p, s);
    case KvType::kQ8: return ByQueries<D, KvType::kQ8>(p, s);
    case KvType::kQ4: return ByQueries<D, KvType::kQ4>(p, s);
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
