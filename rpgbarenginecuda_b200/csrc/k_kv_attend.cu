// k_kv_attend.cu -- attention of one new token per conversation over a paged
// key-value cache: o = softmax(scale q K^T) V per q head, over positions
// [start, len) of each conversation.
//
// What it has to do is read the cache once: 4 G flops per cached pair of
// values (G query heads share a KV head), far under what the tensor cores do
// in the time HBM takes.  So the kernel is a stream of cache pages with the
// math kept out of its way, and what bounds it is HBM (f16, 8 bits) or the
// rate at which the SMs issue the conversions (4 bits).
//
//  * Work.  An item is a (conversation, KV head, chunk of at most 8 query
//    heads); its positions are cut into tiles, and the tiles of all items, in
//    order, are dealt evenly over a persistent grid, wherever the item borders
//    fall.  A border is weighed as a tile or two, which is what ending an item
//    costs.  Every block finds its share from the lengths on the device, so
//    the host needs to know none, ragged batches stay balanced and one long
//    conversation fills the GPU.  An item inside one block is written at once;
//    otherwise the blocks leave (vector, max, sum) records in the workspace
//    and the last of them to finish joins them in block order, so the result
//    does not depend on which is last.
//  * Data.  A warp takes R consecutive positions of a tile and has a slot of
//    shared memory for their K and one for their V, filled by 16-byte
//    asynchronous copies: the next step's K while this step's V is at work and
//    the other way round, across item borders.  (One step ahead is enough: 12
//    warps keep about 100 KB in flight per SM; two steps ahead took 119 us
//    where one takes 113.)  Page lookups and offsets of up to 32 steps of 16
//    positions, 16 of 32, are worked out at once, one 16-position half per
//    lane.  Positions out of range are not used whatever they hold: their
//    scores become -infinity, their V scales or rows zero.  16-byte chunks are
//    permuted so that every read of a tile is free of bank conflicts.
//  * Math.  S^T = K q^T and O^T += V^T P^T on mma.sync with the positions (S)
//    or value dimensions (O) as the 16 rows and 8 query columns, so 2 to 8
//    query heads waste little.  tcgen05 has 128 rows for a query side of 8 and
//    would need codes staged once more through shared or tensor memory, for
//    products that take a fifth of the time as they are.  Codes of K go to
//    the integer tensor cores as they are (4-bit ones spread to bytes), with q
//    as three signed base-256 digits; codes of V become exact f16 integers,
//    two instructions per pair.  A scale multiplies the group's partial score
//    (K) or the weight of its position (V).
//  * Precision.  f32 sums throughout.  With an f16 cache q is scaled by a power
//    of two to a largest value in [1, 2) and split into two f16 terms (a 16-bit
//    q needs one); with a quantised one it is a 24-bit integer relative to its
//    largest value.  The softmax weights are split into two f16 terms and
//    carry a power of two that keeps small ones (times the largest V scale
//    seen) normal numbers: 22 bits.  With at most 4 query heads the second
//    terms and digits ride in the other 4 columns at no cost.  Each step's
//    product starts from zero and is added to the running output in f32
//    registers: the tensor cores truncate when they add, which would grow over
//    a long conversation.
//  * Infinities in an f16 cache give what the formula gives in f32: a warp
//    whose share came out NaN does it again without splits (PlainShare).
//
// Measured on one B200 (floor: bytes at the measured copy rate of 6.55 TB/s):
// 32 conversations of 32 / 8 heads to 8192 positions in f16 107 us (104.5),
// 16 to 3840 in 8 bits 25 us (12.9), one of 65521 in 8 bits 36 us (21.2), 64
// to 4096 in 4 bits 56 us (27.7), one of 21 positions of 16 / 8 heads 5.4 us.
// Between 4096 and 16384 positions the time grows as the floor does in f16 and
// 8 bits and 1.5 times as fast in 4 bits; the line through these times leaves
// 8 us for no data in f16, 13 in 8 and 4 bits and 15 for one conversation: the
// start (lengths, pages, data: three round trips) and the joins.
#include <atomic>

#include "common.h"
#include "kv_dev.cuh"
#include "launch.h"

namespace rpgb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWeightBits = 14;  // weights are scaled by 2^14

template <int D_, KvType KIND_, bool PACK_, int WARPS_>
struct Cfg {
  static constexpr int WARPS = WARPS_;  // of a block: they share an item
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int D = D_;
  static constexpr KvType KIND = KIND_;
  static constexpr bool PACK = PACK_;  // at most 4 query heads: first and second terms share 8 columns
  static constexpr bool QUANT = KIND != KvType::kF16;
  static constexpr int QUERIES = PACK ? 4 : 8;
  static constexpr int R = QUANT || D == 64 ? 32 : 16;  // positions of a warp's step
  static constexpr int TILE = WARPS * R;
  static constexpr int MT = R / 16;     // 16-position tiles of a step
  static constexpr int KS = D / 16;     // 16-value slices of a head
  static constexpr int NG = QUANT ? D / kKvGroup : 1;
  static constexpr int ROW = KIND == KvType::kF16 ? 2 * D : (KIND == KvType::kQ8 ? D : D / 2);
  static constexpr int CPR = ROW / 16;  // 16-byte chunks of a row
  // Tiles (borders included) a block is started for.  One conversation of 16 /
  // 8 heads in f16 with 1, 2, 3 and 4: 100 positions 7.0, 6.1, 7.0 and 6.0 us,
  // 300 8.2, 7.5, 8.0 and 10.4, 2851 11.8, 10.8, 11.3 and 13.4; of 32 / 8 heads
  // in 8 bits to 500 8.3, 9.1, 12.0 and 13.6.
  static constexpr int LEAST = 2;
  // the end of an item costs a block about as much as so many tiles
  static constexpr int BORDER = (QUANT ? 1 : 2) * (WARPS == 1 ? 2 : 1);
  static constexpr int SC = QUANT ? R * NG * 2 : 0;  // scales of a step
  static constexpr int KSLOT = R * ROW + 2 * SC;     // K codes, K scales, V scales
  static constexpr int VSLOT = R * ROW;
  static constexpr int RING = KSLOT + VSLOT;  // per warp
  static_assert(KSLOT % 128 == 0 && VSLOT % 128 == 0, "tiles are 128-byte lines");
  static constexpr int COMB = QUERIES * D * 4;   // per warp
  static constexpr int MAXBLOCKS = WARPS == 1 ? kKvMaxBlocks : 512;
  // the join area: the warps' vectors, then the factors of up to BATCH records
  static constexpr int FACTORS = WARPS == 1 ? 0 : QUERIES * MAXBLOCKS * 4;
  static constexpr int JOIN = WARPS * COMB > FACTORS ? WARPS * COMB : FACTORS;
  static constexpr int BATCH = JOIN / (QUERIES * 4);
  // q as B fragments: f16 terms, or up to three digit tiles of 8-bit integers
  static constexpr int QTILES = QUANT ? (PACK ? 2 : 3) : (PACK ? 1 : 2);
  static constexpr int QWORDS = QUANT ? 4 * NG : 2 * KS;  // of a lane and tile
  static constexpr int QBYTES = QTILES * QWORDS * 128;
  static constexpr int SMEM = WARPS * RING + JOIN + QBYTES;
  // Resident per SM: 12 warps where registers allow (168 a thread; of these
  // the 8-bit form for up to 4 queries of 128 values spills 4 or 5), 8 for more
  // queries of 128 values (200 to 223).  With 64 conversations to 16384 in 4
  // bits, 8 warps take 187 us, 12 take 175 and 16 (128 registers, which spill)
  // 185.
  static constexpr int BLOCKS = (PACK || D == 64 ? 12 : 8) / WARPS;
};

// Byte offset of 16-byte chunk c of row r in a tile of 128-byte lines.  The
// chunk's place in its line is permuted (an exclusive or with bits of the row)
// so that the lanes of one load (8 rows of one chunk for ldmatrix; see
// KFragments and VFragments for the codes) touch different banks.
template <typename C, bool V>
__host__ __device__ constexpr int ChunkAt(int r, int c) {
  const int key = C::KIND == KvType::kF16  ? r & 7
                  : C::KIND == KvType::kQ8 ? (V ? ((r >> 1) & 3) << 1 : (C::D == 128 ? (r & 1) << 2 : 0))
                  : V                      ? (C::D == 128 ? ((r >> 1) & 3) << 1 : ((r >> 2) & 1) << 1)
                                           : (C::D == 128 ? ((r >> 1) & 1) << 1 : 0);
  const int q = r * C::CPR + c;
  return (q >> 3) * 128 + (((q & 7) ^ key) << 4);
}
// The address dr rows and dc chunks from `base`, the address of (r, c): where
// r and dr, c and dc share no bits the permutation is linear, so this is one
// exclusive or with a constant at most.
template <typename C, bool V>
__device__ __forceinline__ uint32_t Moved(uint32_t base, int dr, int dc) {
  const int x = ChunkAt<C, V>(dr, dc);
  return (base ^ (x & 127)) + (x & ~127);
}

// ------------------------------------------------------------------ instructions

__device__ __forceinline__ void CopyAsync16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// The same with nothing to add to.
__device__ __forceinline__ void MmaFirst(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Products of integer codes (signed bytes, or 4-bit ones as unsigned bytes)
// and signed digits; 32 values of a row at a time.
template <bool UNSIGNED>
__device__ __forceinline__ void MmaInt(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (UNSIGNED) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
template <bool UNSIGNED>
__device__ __forceinline__ void MmaIntFirst(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int c) {
  if (UNSIGNED) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c));
  } else {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c));
  }
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
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
               : "r"(a)
               : "memory");
  return x;
}
__device__ __forceinline__ void Sts32(uint32_t a, uint32_t x) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(x) : "memory");
}
__device__ __forceinline__ uint64_t Lds64u(uint32_t a) {
  uint64_t x;
  asm volatile("ld.shared.u64 %0, [%1];" : "=l"(x) : "r"(a) : "memory");
  return x;
}
__device__ __forceinline__ ulonglong2 Lds64x2(uint32_t a) {
  ulonglong2 x;
  asm volatile("ld.shared.v2.u64 {%0,%1}, [%2];" : "=l"(x.x), "=l"(x.y) : "r"(a) : "memory");
  return x;
}
__device__ __forceinline__ void Sts64(uint32_t a, uint64_t x) {
  asm volatile("st.shared.u64 [%0], %1;" ::"r"(a), "l"(x) : "memory");
}
__device__ __forceinline__ void Sts128Zero(uint32_t a) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0) : "memory");
}
// An atomic that releases what the block wrote (after a barrier) and acquires
// what the blocks before it released.
__device__ __forceinline__ unsigned AddAcqRel(unsigned* p, unsigned v) {
  unsigned old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
using kvd::BitsHalf;
using kvd::HalfBits;
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 Both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 Fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 Mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 Add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ uint32_t PackHalf(float lo, float hi) { return HalfBits(__floats2half2_rn(lo, hi)); }

using kvd::High4;
using kvd::kBias8;
using kvd::Low4;
using kvd::SubHalf;
// An integer sum that starts at the bits of 1.5 2^23 is that float plus the sum.
constexpr int kIntStart = 0x4B400000;
constexpr float kIntBias = 12582912.f;

// ------------------------------------------------------------------ work

// The positions of a conversation: [start, len), tiles counted from `base`.
struct Span {
  int start, len, base, tiles;
};
template <typename C>
__device__ __forceinline__ Span SpanOf(const KvAttendParams& p, int seq) {
  const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
  Span s;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(p.lens[seq], 0)), cap));
  s.start = p.starts != nullptr ? max(p.starts[seq], 0) : 0;
  if (s.start >= s.len) s.start = s.len = 0;
  s.base = s.start & ~(C::R - 1);  // a step lies in one page, or its halves in two of 16
  s.tiles = max(1, (s.len - s.base + C::TILE - 1) / C::TILE);  // an empty item still writes its zeros
  return s;
}

// A place in the sequence of tiles: conversation, KV head, query chunk, tile.
template <typename C>
struct Cursor {
  int seq, head, chunk, tile;
  Span span;
  __device__ __forceinline__ void Next(const KvAttendParams& p, int chunks, int n = 1) {
    tile += n;
    if (tile < span.tiles) return;
    tile = 0;
    if (++chunk < chunks) return;
    chunk = 0;
    if (++head < p.kv.n_kv) return;
    head = 0;
    if (++seq < p.table.n_seq) span = SpanOf<C>(p, seq);
  }
};

// The copying side of a warp.  The places of the next steps are worked out
// together, one 16-row half per lane, and left in shared memory; the page ids
// they need are requested one such batch earlier.
struct Places {
  uint64_t code[32], scale[32];  // byte offsets of the halves in the planes
};
template <typename C>
struct Filler {
  static constexpr int kSteps = 32 / C::MT;
  static constexpr uint32_t kStep = (1u << C::MT) - 1;  // the halves of a step
  Cursor<C>* at;       // the first step after the batch; in shared memory, to leave the registers to the math
  int left;            // steps not yet put in a batch
  int count = 0;       // steps of the batch not yet issued
  uint32_t have = 0;   // bit per half of the batch, the next step's lowest: it has rows in range and a page
  uint32_t bad = 0;    // as `have`: it has rows in range but no page
  int page = 0;        // this lane's half of the next batch
  uint32_t place;      // shared-memory address of the next step's first code offset
  uint32_t places;

  static __device__ __forceinline__ int Pos(const Cursor<C>& c, int warp, int lane) {
    return c.span.base + (c.tile + lane / C::MT) * C::TILE + warp * C::R + (lane % C::MT) * 16;
  }
  __device__ __forceinline__ bool InRange(const Cursor<C>& c, int pos, int lane) const {
    return lane / C::MT < min(left, c.span.tiles - c.tile) && pos + 16 > c.span.start && pos < c.span.len;
  }
  __device__ __forceinline__ void Request(const KvAttendParams& p, const Cursor<C>& c, int warp, int lane) {
    const int pos = Pos(c, warp, lane);
    // (positions in range lie inside the table: SpanOf)
    if (left > 0 && InRange(c, pos, lane)) {
      page = p.table.pages[c.seq * p.table.stride + (pos >> p.kv.page_log2)];
    }
  }
  __device__ __forceinline__ void Batch(const KvAttendParams& p, int warp, int lane, int chunks) {
    __syncwarp();  // the last batch has been read
    Cursor<C> c = *at;
    const int pos = Pos(c, warp, lane);
    const bool in = InRange(c, pos, lane);
    const bool ok = in && static_cast<unsigned>(page) < static_cast<unsigned>(p.kv.n_pages);
    const uint32_t row = pos & ((1 << p.kv.page_log2) - 1);
    const uint64_t id = static_cast<uint32_t>(page), head = static_cast<uint32_t>(c.head);
    Sts64(places + lane * 8, (id * p.page16 + head * p.head16 + static_cast<uint64_t>(row) * p.pos16) << 4);
    if (C::QUANT) Sts64(places + 256 + lane * 8, ((id * p.spage16 + head * p.shead16) << 4) + row * (2 * C::NG));
    have = __ballot_sync(0xFFFFFFFFu, ok);
    bad = __ballot_sync(0xFFFFFFFFu, in && !ok);
    count = min(kSteps, min(left, c.span.tiles - c.tile));
    left -= count + (c.tile + count == c.span.tiles ? C::BORDER : 0);
    place = places;
    if (left > 0) {
      c.Next(p, chunks, count);
      Request(p, c, warp, lane);
      if (lane == 0) *at = c;
    }
    __syncwarp();
  }

  // Copies the next step's K codes (and all its scales) or V codes into a
  // slot.  Halves that are out of range or have no page are left as they are.
  // `lane_off` is the lane's part of a source offset.
  template <bool V>
  __device__ __forceinline__ void Issue(const KvAttendParams& p, uint32_t slot, int lane, int64_t lane_off) {
    constexpr int kRows = 32 / C::CPR, kPerHalf = 16 / kRows;  // rows of a copy instruction: all in one half
    const uint32_t dst = slot + ChunkAt<C, V>(lane / C::CPR, lane % C::CPR);
    const char* plane = (V ? p.kv.v : p.kv.k) + lane_off;
    if ((have & kStep) == kStep && p.pos16 == C::ROW / 16) {  // the usual case: all of it, dense rows
      ulonglong2 off;
      if (C::MT == 2) {
        off = Lds64x2(place);
      } else {
        off.x = off.y = Lds64u(place);
      }
#pragma unroll
      for (int h = 0; h < C::MT; ++h) {
        const char* src = plane + (h == 0 ? off.x : off.y);
#pragma unroll
        for (int j = 0; j < kPerHalf; ++j) CopyAsync16(Moved<C, V>(dst, kRows * (h * kPerHalf + j), 0), src + 512 * j);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < C::MT * kPerHalf; ++i) {
        const int h = i / kPerHalf;
        if (!((have >> h) & 1)) continue;
        CopyAsync16(slot + ChunkAt<C, V>(lane / C::CPR + kRows * i, lane % C::CPR),
                    plane + Lds64u(place + 8 * h) + (i % kPerHalf) * kRows * p.kv.pos_stride);
      }
    }
    if (C::QUANT && !V) {
      constexpr int kPer = 2 * C::NG;  // a half's scales are dense: 16 rows of 2 NG bytes, in 16-byte pieces
      const int h = lane / kPer % C::MT;
      if (lane < 2 * C::MT * kPer && ((have >> h) & 1)) {
        const char* sp = (lane < C::MT * kPer ? p.kv.k_scale : p.kv.v_scale) + lane % kPer * 16;
        CopyAsync16(slot + C::R * C::ROW + lane * 16, sp + Lds64u(place + 256 + 8 * h));
      }
    }
    CopyCommit();
  }
  // After both: on to the next step.  Returns the step's `bad`.
  __device__ __forceinline__ uint32_t Pop() {
    const uint32_t b = bad & kStep;
    --count;
    place += 8 * C::MT;
    have >>= C::MT;
    bad >>= C::MT;
    return b;
  }
};

// Block b of n takes tiles [total b / n, total (b + 1) / n); ShareOf is the
// block that has tile x.  Few tiles (blocks are fewer than 2^11) need no 64-bit division.
__device__ __forceinline__ long long ShareBegin(long long total, int b, int n) {
  if (total < (1 << 21)) return static_cast<uint32_t>(total) * static_cast<uint32_t>(b) / static_cast<uint32_t>(n);
  return total * b / n;
}
__device__ __forceinline__ int ShareOf(long long x, long long total, int n) {
  if (total < (1 << 21)) {
    return (static_cast<uint32_t>(x + 1) * static_cast<uint32_t>(n) - 1) / static_cast<uint32_t>(total);
  }
  return static_cast<int>(((x + 1) * n - 1) / total);
}

// ------------------------------------------------------------------ operands

// Where a lane's part of a K tile lies: for ldmatrix, or 16 consecutive values
// (lane t's run) of row g.
template <typename C>
__device__ __forceinline__ int KLaneOffset(int lane) {
  const int g = lane >> 2, t = lane & 3;
  if (C::KIND == KvType::kF16) return ChunkAt<C, false>(lane & 15, lane >> 4);
  return C::KIND == KvType::kQ8 ? ChunkAt<C, false>(g, t) : ChunkAt<C, false>(g, t >> 1) + (t & 1) * 8;
}
// K codes of 16 positions (rows g, g + 8 of tile mt) and a 64-value group as A
// fragments of two 32-value slices.  The columns of a slice are the lanes'
// runs, 8 values of each: q8 codes as they are, 4-bit codes spread to bytes,
// the even values of the 8, then the odd ones (WriteQ takes q the same way).
template <typename C>
__device__ __forceinline__ void KFragments(uint32_t (&a)[2][4], uint32_t base, int mt, int gp) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (C::KIND == KvType::kQ8) {
      const uint4 x = Lds128(Moved<C, false>(base, 16 * mt + 8 * i, 4 * gp));
      a[0][i] = x.x;
      a[0][2 + i] = x.y;
      a[1][i] = x.z;
      a[1][2 + i] = x.w;
    } else {
      const uint2 x = Lds64(Moved<C, false>(base, 16 * mt + 8 * i, 2 * gp));
      a[0][i] = x.x & 0x0F0F0F0Fu;
      a[0][2 + i] = (x.x >> 4) & 0x0F0F0F0Fu;
      a[1][i] = x.y & 0x0F0F0F0Fu;
      a[1][2 + i] = (x.y >> 4) & 0x0F0F0F0Fu;
    }
  }
}

// V^T of a 64-value group and 16 positions as A fragments of four 16-row
// tiles (rows = values).  Lane g takes values 8 g .. 8 g + 7 of the group:
// row g of tile i is value 8 g + i, row g + 8 value 8 g + 4 + i.
template <typename C>
__device__ __forceinline__ int VLaneOffset(int lane) {
  const int g = lane >> 2, t = lane & 3;
  if (C::KIND == KvType::kF16) {  // for ldmatrix
    return ChunkAt<C, true>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
  }
  return C::KIND == KvType::kQ8 ? ChunkAt<C, true>(2 * t, g >> 1) + (g & 1) * 8
                                : ChunkAt<C, true>(2 * t, g >> 2) + (g & 3) * 4;
}
template <typename C>
__device__ __forceinline__ void VFragments(uint32_t (&a)[4][4], uint32_t base, int kt, int gp, uint32_t magic) {
  uint32_t lo[4], hi[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 16 * kt + (j & 1) + 8 * (j >> 1);  // from row 2 t
    if (C::KIND == KvType::kQ8) {
      const uint2 x = Lds64(Moved<C, true>(base, r, 4 * gp));
      lo[j] = x.x;
      hi[j] = x.y;
    } else {
      lo[j] = Lds32(Moved<C, true>(base, r, 2 * gp));
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // position pairs 2 t, 2 t + 1 and 8 further
    if (C::KIND == KvType::kQ8) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t w0 = m ? hi[2 * k] : lo[2 * k], w1 = m ? hi[2 * k + 1] : lo[2 * k + 1];
        const uint32_t x = __byte_perm(w0, w1, 0x5140) ^ 0x80808080u, y = __byte_perm(w0, w1, 0x7362) ^ 0x80808080u;
        a[0][2 * k + m] = SubHalf(__byte_perm(x, magic, 0x5150), kBias8);
        a[1][2 * k + m] = SubHalf(__byte_perm(x, magic, 0x5352), kBias8);
        a[2][2 * k + m] = SubHalf(__byte_perm(y, magic, 0x5150), kBias8);
        a[3][2 * k + m] = SubHalf(__byte_perm(y, magic, 0x5352), kBias8);
      }
    } else {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t x = __byte_perm(lo[2 * k], lo[2 * k + 1], m ? 0x7632 : 0x5410), y = x >> 8;
        a[0][2 * k + m] = Low4(x, magic);
        a[1][2 * k + m] = High4(x, magic);
        a[2][2 * k + m] = Low4(y, magic);
        a[3][2 * k + m] = High4(y, magic);
      }
    }
  }
}

// A lane's values of a q row: f16 caches take pairs 16 ks + 8 b + 2 t (value
// 4 ks + 2 b + e of x), quantised ones the run 16 t of every 64 values.
template <typename C, typename T>
__device__ __forceinline__ void ReadQ(float (&x)[C::D / 4], const T* row, int t) {
  if (!C::QUANT) {
#pragma unroll
    for (int i = 0; i < C::D / 8; ++i) {
      const kvd::Pack<T, 2> r = *reinterpret_cast<const kvd::Pack<T, 2>*>(row + 8 * i + 2 * t);
      x[2 * i] = kvd::ToFloat(r.v[0]);
      x[2 * i + 1] = kvd::ToFloat(r.v[1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < C::D / 16; ++i) {
      float y[4];
      kvd::Load4(row + 64 * (i >> 2) + 16 * t + 4 * (i & 3), y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e];
    }
  }
}

// The lanes' q rows (lane g: column g's query) as B fragments in shared
// memory: word i of tile n, lane at base + ((n * QWORDS + i) / 4 * 32 + lane) *
// 16 + i % 4 * 4, written by warp i % C::WARPS.  Returns what turns a product
// back into a score in log2 units (the scale's magnitude included; its sign
// goes into the fragments, so that the largest product is the largest score).
//
// f16 cache: q times a power of two that brings its largest value into
// [1, 2), as two f16 terms (the second is zero for a 16-bit q).  Quantised
// cache: q / largest as a 24-bit integer in three signed base-256 digits.
template <typename C>
__device__ __forceinline__ float WriteQ(uint32_t base, const float (&x)[C::D / 4], float scale, bool f32, int warp,
                                        int lane, float (&bias)[C::NG][C::QTILES]) {
  const int g = lane >> 2;
  uint32_t top_bits = 0;
#pragma unroll
  for (int i = 0; i < C::D / 4; ++i) top_bits = max(top_bits, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top_bits = max(top_bits, __shfl_xor_sync(0xFFFFFFFFu, top_bits, 1));
  top_bits = max(top_bits, __shfl_xor_sync(0xFFFFFFFFu, top_bits, 2));
  const float sign = scale < 0.f ? -1.f : (scale > 0.f ? 1.f : 0.f), mag = fabsf(scale) * kLog2e;
  // positive, so that scores of -infinity stay; with a NaN or an infinity in q no score means anything
  auto back = [&](float f) { return top_bits >= 0x7F800000u ? kvd::Nan() : fmaxf(f, 1e-30f); };
  auto put = [&](int n, int i, uint32_t w) {
    const int k = n * C::QWORDS + i;
    if (i % C::WARPS == warp) Sts32(base + ((k >> 2) * 32 + lane) * 16 + (k & 3) * 4, w);
  };
  if (!C::QUANT) {
    const int e = min(max(static_cast<int>(top_bits >> 23), 1), 253);  // kept in f32's normal range
    const float down = sign * __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
    for (int i = 0; i < C::QWORDS; ++i) {
      const float u = x[2 * i] * down, v = x[2 * i + 1] * down;
      const uint32_t h = PackHalf(u, v);
      const float2 f = __half22float2(BitsHalf(h));
      const uint32_t r = PackHalf(u - f.x, v - f.y);
      if (C::PACK) {
        put(0, i, f32 && g >= 4 ? r : h);
      } else {
        put(0, i, h);
        put(C::QTILES - 1, i, r);
      }
    }
    return back(__uint_as_float(static_cast<uint32_t>(e) << 23) * mag);
  }
  constexpr float most = 8355700.f;  // 127 in every digit, less room for the product's rounding
  const float top = fmaxf(__uint_as_float(top_bits), 1e-30f);
  const float to_int = sign * (most / top);
  int sum[C::NG][C::QTILES] = {};
#pragma unroll
  for (int i = 0; i < C::QWORDS; ++i) {  // word i: values 4 (i & 1) .. of the run's 8-value half, i / 4 the group
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int first = 16 * (i >> 2) + 8 * ((i >> 1) & 1);
      const int v = first + (C::KIND == KvType::kQ8 ? 4 * (i & 1) + e : 2 * e + (i & 1));
      // with 128 added to every digit the digits are the bytes, each plus 128
      u[e] = static_cast<uint32_t>(__float2int_rn(x[v] * to_int) + 0x808080);
    }
    const uint32_t p01 = __byte_perm(u[0], u[1], 0x5140), p23 = __byte_perm(u[2], u[3], 0x5140);
    uint32_t digit[3] = {__byte_perm(p01, p23, 0x5410), __byte_perm(p01, p23, 0x7632),
                         __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410)};
#pragma unroll
    for (int d = 0; d < 3; ++d) digit[d] ^= 0x80808080u;
    uint32_t w[3];
    if (C::PACK) {
      w[0] = g < 4 ? digit[2] : digit[1];
      w[1] = g < 4 ? digit[0] : 0;
    } else {
      w[0] = digit[2];
      w[1] = digit[1];
      w[2] = digit[0];
    }
#pragma unroll
    for (int n = 0; n < C::QTILES; ++n) {
      put(n, i, w[n]);
      sum[i >> 2][n] = __dp4a(static_cast<int>(w[n]), 0x01010101, sum[i >> 2][n]);
    }
  }
#pragma unroll
  for (int gp = 0; gp < C::NG; ++gp) {
#pragma unroll
    for (int n = 0; n < C::QTILES; ++n) {
      int v = sum[gp][n];
      v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
      v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
      bias[gp][n] = kIntBias + (C::KIND == KvType::kQ4 ? 8.f * static_cast<float>(v) : 0.f);
    }
  }
  return back(top / most * 65536.f * mag);  // the highest digit counts 65536
}

// ------------------------------------------------------------------ kernel

__device__ __forceinline__ void AddScaled(float4& v, float f, const float4& x) {
  v.x += f * x.x;
  v.y += f * x.y;
  v.z += f * x.z;
  v.w += f * x.w;
}

// A warp's share of an item (its rows of n tiles from c's) by the formula as
// it stands: one value at a time in f32.  With an f16 cache the split terms of
// q and of the weights give the formula's results for finite values only
// (infinity times a term that is zero, or times terms of both signs, is NaN),
// so a share that came out NaN is done again here; its vectors, maxima and
// sums replace the first ones.  (A quantised cache holds no infinity, and a
// NaN is its group's scale.)
template <typename C>
__device__ __forceinline__ void PlainShare(const KvAttendParams& p, const Cursor<C>& c, int n, int warp, int lane,
                                           int64_t q_row, int queries, float* vec, float* maxima, float* sums) {
  constexpr int N = C::D / 32;  // values of a lane
  using Row = kvd::Pack<__half, N>;
#pragma unroll 1
  for (int qi = 0; qi < queries; ++qi) {
    const int64_t o = q_row + static_cast<int64_t>(qi) * C::D + lane * N;
    float x[N], acc[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      switch (p.type) {
        case ElemType::kF32: x[e] = static_cast<const float*>(p.q)[o + e]; break;
        case ElemType::kF16: x[e] = kvd::ToFloat(static_cast<const __half*>(p.q)[o + e]); break;
        case ElemType::kBF16: x[e] = kvd::ToFloat(static_cast<const __nv_bfloat16*>(p.q)[o + e]); break;
      }
      l += x[e] * 0.f;  // NaN with a NaN or an infinity in q
    }
    l = dev::WarpSum(l);
#pragma unroll 1
    for (int k = 0; k < n * C::R && l == l; ++k) {
      const int pos = c.span.base + (c.tile + k / C::R) * C::TILE + warp * C::R + k % C::R;
      if (pos < c.span.start || pos >= c.span.len) continue;
      const int page = kvd::PageOf(p.table, p.kv.n_pages, c.seq, pos >> p.kv.page_log2);
      if (page < 0) {
        l = kvd::Nan();
        break;
      }
      const int64_t at =
          kvd::CodeOffset(p.kv, page, c.head, pos & ((1 << p.kv.page_log2) - 1)) + lane * static_cast<int>(sizeof(Row));
      const Row kr = *reinterpret_cast<const Row*>(p.kv.k + at), vr = *reinterpret_cast<const Row*>(p.kv.v + at);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) dot += x[e] * __half2float(kr.v[e]);
      const float s = dev::WarpSum(dot) * (p.scale * kLog2e);
      const float now = fmaxf(m, s), ref = now == -INFINITY ? 0.f : now;
      const float alpha = Exp2(m - ref), w = Exp2(s - ref);
      m = now;
      l = l * alpha + w;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = acc[e] * alpha + w * __half2float(vr.v[e]);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) vec[qi * C::D + lane * N + e] = l == l ? acc[e] : l;
    if (lane == 0) {
      maxima[qi] = m;
      sums[qi] = l;
    }
  }
}

template <typename C>
__global__ void __launch_bounds__(C::THREADS, C::BLOCKS) KvAttendKernel(const KvAttendParams p) {
  constexpr int D = C::D;
  extern __shared__ __align__(128) char smem[];
  __shared__ float s_m[C::WARPS][8], s_l[C::WARPS][8], s_keep[8];
  __shared__ long long s_sum[C::WARPS], s_begin, s_item0[C::WARPS];
  __shared__ int s_seq, s_last;
  __shared__ Cursor<C> s_use[C::WARPS], s_fill[C::WARPS];
  __shared__ __align__(8) float s_bias[C::NG][3][8];
  __shared__ __align__(16) Places s_places[C::WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / p.kv.n_kv;
  const int chunks = (group + kKvMaxQueries - 1) / kKvMaxQueries;
  const int per_chunk = (group + chunks - 1) / chunks;
  const int items = p.kv.n_kv * chunks;

  dev::GridLaunchDependents();
  dev::GridWait();  // (launched before the stream's previous kernel has finished)
  // This block's share of the tiles: prefix sums of the conversations' tiles
  // (and their items' borders), a run of conversations per thread.
  const int run = (p.table.n_seq + C::THREADS - 1) / C::THREADS;
  long long mine = 0;
  for (int i = 0; i < run; ++i) {
    const int s = tid * run + i;
    if (s < p.table.n_seq) mine += static_cast<long long>(SpanOf<C>(p, s).tiles + C::BORDER) * items;
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
  for (int w = 0; w < C::WARPS; ++w) {
    if (w == warp) upto += total;
    total += s_sum[w];
  }
  const int blocks = static_cast<int>(min(static_cast<long long>(gridDim.x), (total + C::LEAST - 1) / C::LEAST));
  if (static_cast<int>(blockIdx.x) >= blocks) return;
  const long long first = ShareBegin(total, blockIdx.x, blocks);
  int left = static_cast<int>(ShareBegin(total, blockIdx.x + 1, blocks) - first);  // tiles to do
  if (first >= upto - mine && first < upto) {
    long long at = upto - mine;
    int s = tid * run;
    for (;; ++s) {
      const long long n = static_cast<long long>(SpanOf<C>(p, s).tiles + C::BORDER) * items;
      if (first < at + n) break;
      at += n;
    }
    s_seq = s;
    s_begin = at;
  }
  __syncthreads();
  Cursor<C> use;
  long long item0;  // the item's first tile
  use.seq = s_seq;
  use.span = SpanOf<C>(p, use.seq);
  {
    const long long in = first - s_begin;  // inside the conversation
    const int n = use.span.tiles + C::BORDER;
    const long long item = in < (1ll << 31) ? static_cast<uint32_t>(in) / static_cast<uint32_t>(n) : in / n;
    use.tile = static_cast<int>(in - item * n);
    use.head = static_cast<int>(item) / chunks;
    use.chunk = static_cast<int>(item) % chunks;
    item0 = first - use.tile;
    if (use.tile >= use.span.tiles) {  // the share begins in an item's border
      left -= n - use.tile;
      if (left <= 0) return;
      item0 += n;
      use.tile = use.span.tiles;
      use.Next(p, chunks, 0);
    }
  }

  const uint32_t ring = dev::SmemAddr(smem) + warp * C::RING;
  float* comb = reinterpret_cast<float*>(smem + C::WARPS * C::RING);
  float* mineq = comb + warp * (C::COMB / 4);
  const uint32_t q_smem = dev::SmemAddr(smem) + C::WARPS * C::RING + C::JOIN;
  const uint32_t k_lane = KLaneOffset<C>(lane), v_lane = VLaneOffset<C>(lane);
  // What changes with the item only is kept per warp in shared memory.
  if (lane == 0) {
    s_use[warp] = s_fill[warp] = use;
    s_item0[warp] = item0;
  }
  __syncwarp();
  Filler<C> fill;
  fill.at = &s_fill[warp];
  fill.left = left;
  fill.places = fill.place = dev::SmemAddr(&s_places[warp]);
  const int64_t lane_off = static_cast<int64_t>(lane / C::CPR) * p.kv.pos_stride + (lane % C::CPR) * 16;
  fill.Request(p, use, warp, lane);

  const uint32_t kslot = ring, vslot = ring + C::KSLOT;
  uint32_t bad_now = 0;  // the step's halves that have rows in range but no page
  const uint32_t magic = p.magic;
  const bool two_terms = p.type == ElemType::kF32;
  for (bool begin = true;; begin = false) {
    // ---- an item: its queries, as B fragments
    int n, lo, hi;  // tiles of the item that are this block's; the range, from this warp's first row
    float x[D / 4] = {};
    {
      const Cursor<C> c = s_use[warp];
      n = min(left, c.span.tiles - c.tile);
      lo = c.span.start - (c.span.base + c.tile * C::TILE + warp * C::R);
      hi = c.span.len - (c.span.base + c.tile * C::TILE + warp * C::R);
      const int qi = C::PACK ? g & 3 : g;
      if (qi < min(per_chunk, group - c.chunk * per_chunk)) {
        const int64_t o = c.seq * p.q_stride + (static_cast<int64_t>(c.head) * group + c.chunk * per_chunk + qi) * D;
        switch (p.type) {
          case ElemType::kF32: ReadQ<C>(x, static_cast<const float*>(p.q) + o, t); break;
          case ElemType::kF16: ReadQ<C>(x, static_cast<const __half*>(p.q) + o, t); break;
          case ElemType::kBF16: ReadQ<C>(x, static_cast<const __nv_bfloat16*>(p.q) + o, t); break;
        }
      }
    }
    if (begin) {  // the first steps' copies, while the queries are on their way
      fill.Batch(p, warp, lane, chunks);
      fill.template Issue<false>(p, kslot, lane, lane_off);
      fill.template Issue<true>(p, vslot, lane, lane_off);
      bad_now = fill.Pop();
    }
    // of columns 2 t, 2 t + 1: from products to scores in log2 units; largest
    // score; weights are 2^(score - ref); sum of this lane's weights
    float2 cs, m = Both(-INFINITY), ref = m, l = Both(0.f);
    float2 acc[D / 16][2];  // rows g and g + 8 of a tile
    int nu = 127 - 25;      // biased exponent of the power of two over the V scales seen
    {
      float bias[C::NG][C::QTILES];
      const float up = WriteQ<C>(q_smem, x, p.scale, two_terms, warp, lane, bias);
      if (C::QUANT && warp == 0 && t == 0) {
#pragma unroll
        for (int gp = 0; gp < C::NG; ++gp) {
#pragma unroll
          for (int n = 0; n < C::QTILES; ++n) s_bias[gp][n][g] = bias[gp][n];
        }
      }
      cs.x = __shfl_sync(0xFFFFFFFFu, up, 4 * (C::PACK ? (2 * t) & 3 : 2 * t));
      cs.y = __shfl_sync(0xFFFFFFFFu, up, 4 * (C::PACK ? (2 * t + 1) & 3 : 2 * t + 1));
      // (lanes that join the digits from the lower one have 256 times the product)
      if (C::QUANT && C::PACK && t >= 2) cs = Mul2(cs, Both(1.f / 256));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[i][0] = acc[i][1] = Both(0.f);
    }
    __syncthreads();

    // ---- its tiles
    left -= n + C::BORDER;  // (past the end where the share ends inside the item: what counts is whether any is left)
#pragma unroll 1
    for (int i = n; i > 0; --i, lo -= C::TILE, hi -= C::TILE) {
      const bool work = lo < C::R && hi > 0;
      const bool edge = lo > 0 || hi < C::R || bad_now != 0;

      // ---- scores (and the V scales)
      CopyWait<1>();
      __syncwarp();
      float2 s[C::MT][2];  // rows g and g + 8 of a tile, columns 2 t and 2 t + 1
      uint32_t vsc[C::MT][2];  // V scales of the lane's rows, one or two f16
      if (work) {
        const uint32_t kbase = kslot + k_lane, sbase = kslot + C::R * C::ROW + g * (2 * C::NG);
        const uint32_t qbase = q_smem + lane * 16;
        if (!C::QUANT) {
          float sum[C::MT][4];
#pragma unroll
          for (int k4 = 0; k4 < C::QWORDS / 4; ++k4) {
            const uint4 q = Lds128(qbase + k4 * 512);
            uint4 r = q;
            if (!C::PACK && two_terms) r = Lds128(qbase + (C::QWORDS / 4 + k4) * 512);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int ks = 2 * k4 + j;
#pragma unroll
              for (int mt = 0; mt < C::MT; ++mt) {
                uint32_t a[4];
                LdMatrix(a, Moved<C, false>(kbase, 16 * mt, 2 * ks));
                ks == 0 ? MmaFirst(sum[mt], a, q.x, q.y) : Mma(sum[mt], a, j == 0 ? q.x : q.z, j == 0 ? q.y : q.w);
                if (!C::PACK && two_terms) Mma(sum[mt], a, j == 0 ? r.x : r.z, j == 0 ? r.y : r.w);
              }
            }
          }
#pragma unroll
          for (int mt = 0; mt < C::MT; ++mt) {
            s[mt][0] = make_float2(sum[mt][0], sum[mt][1]);
            s[mt][1] = make_float2(sum[mt][2], sum[mt][3]);
          }
        } else {
          constexpr bool kU = C::KIND == KvType::kQ4;
          float2 d[C::MT][2];
#pragma unroll
          for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a = sbase + (16 * mt + 8 * i) * (2 * C::NG);
              const uint32_t k = C::NG == 2 ? Lds32(a) : Lds16(a);
              vsc[mt][i] = C::NG == 2 ? Lds32(a + C::SC) : Lds16(a + C::SC);
              d[mt][i] = __half22float2(BitsHalf(k));
            }
          }
#pragma unroll
          for (int gp = 0; gp < C::NG; ++gp) {
            const uint4 q0 = Lds128(qbase + gp * 512);
            const uint4 q1 = Lds128(qbase + (C::NG + gp) * 512);
            const uint4 q2 = C::PACK ? q1 : Lds128(qbase + (2 * C::NG + gp) * 512);
            float2 b0 = make_float2(kIntBias, kIntBias), b1 = b0, b2 = b0;
            if (kU) {
              b0 = *reinterpret_cast<const float2*>(&s_bias[gp][0][2 * t]);
              b1 = *reinterpret_cast<const float2*>(&s_bias[gp][1][2 * t]);
              b2 = *reinterpret_cast<const float2*>(&s_bias[gp][C::QTILES - 1][2 * t]);
            }
#pragma unroll
            for (int mt = 0; mt < C::MT; ++mt) {
              uint32_t a[2][4];
              KFragments<C>(a, kbase, mt, gp);
              auto product = [&](const uint4& q, const float2& b, float2 (&v)[2]) {
                int n[4];
                MmaIntFirst<kU>(n, a[0], q.x, q.y, kIntStart);
                MmaInt<kU>(n, a[1], q.z, q.w);
                const float2 less = make_float2(-b.x, -b.y);
                v[0] = Add2(make_float2(__int_as_float(n[0]), __int_as_float(n[1])), less);
                v[1] = Add2(make_float2(__int_as_float(n[2]), __int_as_float(n[3])), less);
              };
              float2 v[2], r[2];
              product(q0, b0, v);
              product(q1, b1, r);
#pragma unroll
              for (int i = 0; i < 2; ++i) v[i] = Fma2(r[i], Both(C::PACK ? 1.f / 65536 : 1.f / 256), v[i]);
              if (!C::PACK) {
                product(q2, b2, r);
#pragma unroll
                for (int i = 0; i < 2; ++i) v[i] = Fma2(r[i], Both(1.f / 65536), v[i]);
              }
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                s[mt][i] = gp == 0 ? Mul2(v[i], Both(d[mt][i].x)) : Fma2(v[i], Both(d[mt][i].y), s[mt][i]);
              }
            }
          }
        }
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
          if (C::PACK && C::QUANT) {  // lanes t < 2 hold the first digit, the others the second
            const float2 f = Both(t < 2 ? 1.f / 256 : 256.f);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 other = make_float2(__shfl_xor_sync(0xFFFFFFFFu, s[mt][i].x, 2),
                                               __shfl_xor_sync(0xFFFFFFFFu, s[mt][i].y, 2));
              s[mt][i] = Fma2(other, f, s[mt][i]);
            }
          }
          if (C::PACK && !C::QUANT && two_terms) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              s[mt][i].x += __shfl_xor_sync(0xFFFFFFFFu, s[mt][i].x, 2);
              s[mt][i].y += __shfl_xor_sync(0xFFFFFFFFu, s[mt][i].y, 2);
            }
          }
        }
      }
      __syncwarp();
      if (fill.count == 0) {
        if (fill.left > 0) {
          fill.Batch(p, warp, lane, chunks);
        } else {
          fill.have = 0;  // no more steps
        }
      }
      fill.template Issue<false>(p, kslot, lane, lane_off);
      CopyWait<1>();  // V
      __syncwarp();

      // ---- weights: 2^(score - ref) with ref a power of two over the largest,
      // so that a weight times its V scale is at most 2^14 and small ones stay
      // normal f16 numbers
      float2 alpha = Both(1.f);
      if (work) {
        if (edge) {
          asm volatile("" ::: "memory");  // a branch, not predicates: few steps come here
#pragma unroll
          for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = 16 * mt + 8 * i + g;
              if ((bad_now >> mt) & 1) s[mt][i] = Both(kvd::Nan());
              if (r < lo || r >= hi) {
                s[mt][i] = Both(-INFINITY);
                vsc[mt][i] = 0;  // a scale out of range may be anything
              }
            }
          }
        }
        if (C::QUANT) {
          __half2 top = BitsHalf(0);
#pragma unroll
          for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) top = __hmax2(top, __habs2(BitsHalf(vsc[mt][i])));
          }
          const uint32_t u = HalfBits(top);
          const uint32_t f16 = __reduce_max_sync(0xFFFFFFFFu, max(u & 0xFFFFu, u >> 16));
          const float d = __half2float(__ushort_as_half(static_cast<unsigned short>(f16)));
          nu = max(nu, min(static_cast<int>(__float_as_uint(d) >> 23), 127 + 16) + 1);
        }
        const float shift = C::QUANT ? static_cast<float>(nu - 127 - kWeightBits) : -static_cast<float>(kWeightBits);
        float2 top = s[0][0], now;
#pragma unroll
        for (int j = 1; j < 2 * C::MT; ++j) {
          top.x = fmaxf(top.x, s[j >> 1][j & 1].x);
          top.y = fmaxf(top.y, s[j >> 1][j & 1].y);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          top.x = fmaxf(top.x, __shfl_xor_sync(0xFFFFFFFFu, top.x, o));
          top.y = fmaxf(top.y, __shfl_xor_sync(0xFFFFFFFFu, top.y, o));
        }
        m.x = fmaxf(m.x, top.x * cs.x);
        m.y = fmaxf(m.y, top.y * cs.y);
        now.x = (m.x == -INFINITY ? 0.f : m.x) + shift;
        now.y = (m.y == -INFINITY ? 0.f : m.y) + shift;
        alpha = make_float2(Exp2(ref.x - now.x), Exp2(ref.y - now.y));
        ref.x = m.x == -INFINITY ? -INFINITY : now.x;
        ref.y = m.y == -INFINITY ? -INFINITY : now.y;
        l = Mul2(l, alpha);
        const float2 less = make_float2(-now.x, -now.y);
#pragma unroll
        for (int j = 0; j < 2 * C::MT; ++j) {
          const float2 e = Fma2(s[j >> 1][j & 1], cs, less);
          const float2 w = make_float2(Exp2(e.x), Exp2(e.y));
          s[j >> 1][j & 1] = w;
          l = Add2(l, w);
        }
      }

      // ---- values
      if (work) {
        if (!C::QUANT && edge) {  // what lies out of range may be anything, NaN too: zeros
#pragma unroll 1
          for (int i = lane; i < C::R * C::CPR; i += 32) {
            const int r = i / C::CPR;
            if (r < lo || r >= hi) Sts128Zero(vslot + ChunkAt<C, true>(r, i % C::CPR));
          }
          __syncwarp();
        }
        const uint32_t vbase = vslot + v_lane;
        // the term that the lane's columns take
        const float2 of_rest = Both(t >= 2 ? 1.f : 0.f), of_lead = Both(t >= 2 ? -1.f : 1.f);
#pragma unroll
        for (int gp = 0; gp < C::NG; ++gp) {
          uint32_t b[C::MT][2][C::PACK ? 1 : 2];
#pragma unroll
          for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float2 u = s[mt][i];
              if (C::QUANT) {
                const float2 d = __half22float2(BitsHalf(vsc[mt][i]));
                u = Mul2(u, Both(gp == 0 ? d.x : d.y));
              }
              // the first term is the leading 11 bits, the second the rest
              const float2 h = make_float2(__uint_as_float(__float_as_uint(u.x) & 0xFFFFE000u),
                                           __uint_as_float(__float_as_uint(u.y) & 0xFFFFE000u));
              if (C::PACK) {
                const float2 w = Fma2(u, of_rest, Mul2(h, of_lead));
                b[mt][i][0] = Transposed(PackHalf(w.x, w.y));
              } else {
                b[mt][i][0] = Transposed(PackHalf(h.x, h.y));
                b[mt][i][C::PACK ? 0 : 1] = Transposed(PackHalf(u.x - h.x, u.y - h.y));
              }
            }
          }
          if (C::QUANT) {
            float part[4][4];
#pragma unroll
            for (int kt = 0; kt < C::MT; ++kt) {
              uint32_t a[4][4];
              VFragments<C>(a, vbase, kt, gp, magic);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                kt == 0 ? MmaFirst(part[i], a[i], b[kt][0][0], b[kt][1][0])
                        : Mma(part[i], a[i], b[kt][0][0], b[kt][1][0]);
                if (!C::PACK) Mma(part[i], a[i], b[kt][0][C::PACK ? 0 : 1], b[kt][1][C::PACK ? 0 : 1]);
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                acc[4 * gp + i][c] = Fma2(acc[4 * gp + i][c], alpha, make_float2(part[i][2 * c], part[i][2 * c + 1]));
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              float part[4];
#pragma unroll
              for (int kt = 0; kt < C::MT; ++kt) {
                uint32_t a[4];
                LdMatrixT(a, Moved<C, true>(vbase, 16 * kt, 2 * i));
                kt == 0 ? MmaFirst(part, a, b[kt][0][0], b[kt][1][0]) : Mma(part, a, b[kt][0][0], b[kt][1][0]);
                if (!C::PACK) Mma(part, a, b[kt][0][C::PACK ? 0 : 1], b[kt][1][C::PACK ? 0 : 1]);
              }
#pragma unroll
              for (int c = 0; c < 2; ++c) acc[i][c] = Fma2(acc[i][c], alpha, make_float2(part[2 * c], part[2 * c + 1]));
            }
          }
        }
      }
      __syncwarp();
      fill.template Issue<true>(p, vslot, lane, lane_off);
      bad_now = fill.Pop();
    }

    // ---- the end of the item, or of this block's share of it
    {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l.x += __shfl_xor_sync(0xFFFFFFFFu, l.x, o);
        l.y += __shfl_xor_sync(0xFFFFFFFFu, l.y, o);
      }
      float2 any = l;  // NaN where one of the lane's results is
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float2 v = acc[i][c];
          if (C::PACK) {  // the two terms
            v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, 2);
            v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, 2);
          }
          if (!C::QUANT) any = Add2(any, v);
          const int value = C::QUANT ? 64 * (i >> 2) + 8 * g + 4 * c + (i & 3) : 16 * i + 8 * c + g;
          if (!C::PACK || t < 2) {
            mineq[2 * t * D + value] = v.x;
            mineq[(2 * t + 1) * D + value] = v.y;
          }
        }
      }
      if (g == 0 && (!C::PACK || t < 2)) {
        s_m[warp][2 * t] = ref.x;
        s_m[warp][2 * t + 1] = ref.y;
        s_l[warp][2 * t] = l.x;
        s_l[warp][2 * t + 1] = l.y;
      }
      if (!C::QUANT && __any_sync(0xFFFFFFFFu, !(any.x == any.x && any.y == any.y))) {
        const Cursor<C> c = s_use[warp];
        const int first = c.chunk * per_chunk;
        __syncwarp();
        PlainShare(p, c, n, warp, lane, c.seq * p.q_stride + (static_cast<int64_t>(c.head) * group + first) * D,
                   min(per_chunk, group - first), mineq, s_m[warp], s_l[warp]);
      }
      __syncthreads();
      const Cursor<C> use = s_use[warp];
      const long long item0 = s_item0[warp];
      const bool whole = use.tile == 0 && n == use.span.tiles;
      const int queries = min(per_chunk, group - use.chunk * per_chunk);
      const int64_t out = use.seq * p.out_stride + (static_cast<int64_t>(use.head) * group + use.chunk * per_chunk) * D;
      const bool past = static_cast<int64_t>(max(p.lens[use.seq], 0)) >
                        (static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2);
      // The warps' shares joined: values 4 i .. 4 i + 3 of the item's queries.
      auto join = [&](int i, float& sum, float& top) {
        const int q = 4 * i / D;
        top = s_m[0][q];
#pragma unroll
        for (int w = 1; w < C::WARPS; ++w) top = fmaxf(top, s_m[w][q]);
        const float ref = top == -INFINITY ? 0.f : top;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) {
          AddScaled(v, Exp2(s_m[w][q] - ref), reinterpret_cast<const float4*>(comb + w * (C::COMB / 4))[i]);
          sum += Exp2(s_m[w][q] - ref) * s_l[w][q];
        }
        return v;
      };
      auto put = [&](int i, const float4& v, float sum) {
        const float f = sum != 0.f ? 1.f / sum : 0.f;  // nothing in range: zero
        float y[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = past ? kvd::Nan() : y[e];
        switch (p.type) {
          case ElemType::kF32: kvd::Store4(static_cast<float*>(p.out) + out + 4 * i, y); break;
          case ElemType::kF16: kvd::Store4(static_cast<__half*>(p.out) + out + 4 * i, y); break;
          case ElemType::kBF16: kvd::Store4(static_cast<__nv_bfloat16*>(p.out) + out + 4 * i, y); break;
        }
      };
      const int vecs = queries * D / 4;
      bool finish = whole;
      if (!whole) {
        // This block's record: one for an item that began in an earlier block,
        // one for an item that begins here.  Blocks b0 .. b1 hold the parts.
        const int b0 = ShareOf(item0, total, blocks), b1 = ShareOf(item0 + use.span.tiles - 1, total, blocks);
        const int record_size = KvRecordFloats(per_chunk, D), ms = per_chunk * D, ls = ms + per_chunk;
        float* records = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + kKvMaxBlocks * 4);
        auto record = [&](int b) { return records + static_cast<int64_t>(2 * b + (b == b0 ? 1 : 0)) * record_size; };
        // (one item at most begins in a block and goes on past it, so the block numbers its counter)
        unsigned* count = static_cast<unsigned*>(p.workspace) + b0;
        float* rec = record(blockIdx.x);
        for (int i = tid; i < vecs; i += C::THREADS) {
          float sum, top;
          reinterpret_cast<float4*>(rec)[i] = join(i, sum, top);
          if (i % (D / 4) == 0) {
            rec[ms + i / (D / 4)] = top;
            rec[ls + i / (D / 4)] = sum;
          }
        }
        __syncthreads();
        if (tid == 0) s_last = AddAcqRel(count, 1u) == static_cast<unsigned>(b1 - b0);
        __syncthreads();
        finish = s_last != 0;
        if (finish && tid == 0) *count = 0;
        constexpr int kFew = 4;
        if (finish && b1 - b0 < kFew) {
          // Few records: every thread reads what it needs of all of them at
          // once.  Against the join below: one conversation of 16 / 8 heads to
          // 300 in f16 7.5 and 8.5 us, of 32 / 8 to 500 in 8 bits 9.1 and 10.0,
          // 64 to 4096 in 4 bits 56.3 and 57.6.  (Up to eight records so: 8 of
          // 64 / 8 heads to 1000 in f16 11.5 us against 13.2, but 11.1 against
          // 10.8 for one of 16 / 8 to 2851, for the registers it takes.)
          finish = false;
          for (int i = tid; i < vecs; i += C::THREADS) {
            const int q = 4 * i / D;
            float top = -INFINITY, m_[kFew], l_[kFew];
            float4 v[kFew];
#pragma unroll
            for (int n = 0; n < kFew; ++n) {
              m_[n] = -INFINITY;
              l_[n] = 0.f;
              v[n] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (b0 + n <= b1) {
                const float* r = record(b0 + n);
                m_[n] = __ldcg(r + ms + q);
                l_[n] = __ldcg(r + ls + q);
                v[n] = __ldcg(reinterpret_cast<const float4*>(r) + i);
              }
            }
#pragma unroll
            for (int n = 0; n < kFew; ++n) top = fmaxf(top, m_[n]);
            const float ref = top == -INFINITY ? 0.f : top;
            float4 sumv = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < kFew; ++n) {
              const float f = Exp2(m_[n] - ref);
              AddScaled(sumv, f, v[n]);
              sum += f * l_[n];
            }
            put(i, sumv, sum);
          }
        }
        if (finish) {
          // The last block joins all records, BATCH of them at a time: their
          // factors under the largest maximum so far into the join area, a
          // query per warp and a record per lane; then warp w adds up records
          // w, w + WARPS, ... in that order, a few of them in flight.
          float* factor = comb;  // [query][record of the batch]
          constexpr int kVec = C::QUERIES * D / 128, kFlight = 8 / kVec;  // float4 of a lane; records in flight
          float4 v[kVec];
#pragma unroll
          for (int k = 0; k < kVec; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int c0 = b0; c0 <= b1; c0 += C::BATCH) {
            const int c1 = min(c0 + C::BATCH - 1, b1);
            for (int q = warp; q < queries; q += C::WARPS) {
              const float before = c0 == b0 ? -INFINITY : s_m[0][q];
              float top = before, sum = 0.f;  // the lane's
              for (int b = c0 + lane; b <= c1; b += 64) {  // (a second record per lane at once)
                const bool two = b + 32 <= c1;
                const float *r = record(b) + q, *r2 = record(two ? b + 32 : b) + q;
                const float ma = __ldcg(r + ms), mb = __ldcg(r2 + ms), la = __ldcg(r + ls), lb = __ldcg(r2 + ls);
                const float now = fmaxf(top, fmaxf(ma, mb)), ref = now == -INFINITY ? 0.f : now;
                sum = sum * Exp2(top - ref) + Exp2(ma - ref) * la + (two ? Exp2(mb - ref) * lb : 0.f);
                top = now;
                factor[q * C::BATCH + b - c0] = ma;
                if (two) factor[q * C::BATCH + b + 32 - c0] = mb;
              }
              const float all = dev::WarpMax(top), ref = all == -INFINITY ? 0.f : all;
              sum = dev::WarpSum(sum * Exp2(top - ref));
              for (int b = lane; b <= c1 - c0; b += 32) {  // (the lane's own: b and b + 32 keep their lane)
                factor[q * C::BATCH + b] = Exp2(factor[q * C::BATCH + b] - ref);
              }
              const float keep = Exp2(before - ref), was = c0 == b0 ? 0.f : s_l[0][q];
              __syncwarp();
              if (lane < C::WARPS) {
                s_m[lane][q] = all;
                s_l[lane][q] = lane == 0 ? was * keep + sum : 0.f;
              }
              if (lane == 0) s_keep[q] = keep;
            }
            __syncthreads();
            if (c0 != b0) {
#pragma unroll
              for (int k = 0; k < kVec; ++k) {
                const int q = D == 128 ? k : 2 * k + (lane >> 4);
                const float f = q < queries ? s_keep[q] : 0.f;
                v[k] = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
              }
            }
            for (int b = c0 + warp; b <= c1; b += C::WARPS * kFlight) {
              float4 r[kFlight][kVec];
#pragma unroll
              for (int n = 0; n < kFlight; ++n) {
#pragma unroll
                for (int k = 0; k < kVec; ++k) {
                  const int q = D == 128 ? k : 2 * k + (lane >> 4);
                  if (b + n * C::WARPS <= c1 && q < queries) {
                    r[n][k] = __ldcg(reinterpret_cast<const float4*>(record(b + n * C::WARPS)) + 32 * k + lane);
                  }
                }
              }
#pragma unroll
              for (int n = 0; n < kFlight; ++n) {
#pragma unroll
                for (int k = 0; k < kVec; ++k) {
                  const int q = D == 128 ? k : 2 * k + (lane >> 4);
                  if (b + n * C::WARPS <= c1 && q < queries) {
                    AddScaled(v[k], factor[q * C::BATCH + b - c0 + n * C::WARPS], r[n][k]);
                  }
                }
              }
            }
            __syncthreads();  // the factors have been read
          }
#pragma unroll
          for (int k = 0; k < kVec; ++k) reinterpret_cast<float4*>(mineq)[32 * k + lane] = v[k];
          __syncthreads();
        }
      }
      if (finish) {
        for (int i = tid; i < vecs; i += C::THREADS) {
          float sum, top;
          const float4 v = join(i, sum, top);
          put(i, v, sum);
        }
      }
      if (left > 0) {
        Cursor<C> c = use;
        c.Next(p, chunks, n);
        __syncwarp();
        if (lane == 0) {
          s_use[warp] = c;
          s_item0[warp] = item0 + use.span.tiles + C::BORDER;
        }
      }
      __syncthreads();  // the next item writes the join area again
    }
    if (left <= 0) break;
  }
  CopyWait<0>();
}

// Blocks of the kernel that the current device holds at once.
template <typename C>
int Resident() {
  static std::atomic<int> resident[64];
  int dev = 0;
  RPGB_CUDA(cudaGetDevice(&dev));
  RPGB_CHECK(dev < 64, "kv: device %d", dev);
  int grid = resident[dev].load(std::memory_order_acquire);
  if (grid == 0) {
    int sms = 0, per = 0;
    RPGB_CUDA(cudaFuncSetAttribute(KvAttendKernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    RPGB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    RPGB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, KvAttendKernel<C>, C::THREADS, C::SMEM));
    RPGB_CHECK(per > 0, "kv: the attend kernel does not fit device %d", dev);
    grid = sms * per < C::MAXBLOCKS ? sms * per : C::MAXBLOCKS;
    resident[dev].store(grid, std::memory_order_release);
  }
  return grid;
}

template <typename C>
void Launch(const KvAttendParams& p, int chunks, cudaStream_t s) {
  int grid = Resident<C>();
  // no more blocks than tiles there can be
  const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
  const int64_t tiles = ((cap + 15) / C::TILE + 1 + C::BORDER) * p.kv.n_kv * chunks;
  if (tiles < grid && tiles * p.table.n_seq < grid) grid = static_cast<int>(tiles * p.table.n_seq);
  KvAttendParams a = p;
  a.magic = kvd::kMagic;
  a.page16 = static_cast<uint32_t>(p.kv.page_stride / 16);
  a.head16 = static_cast<uint32_t>(p.kv.head_stride / 16);
  a.pos16 = static_cast<uint32_t>(p.kv.pos_stride / 16);
  a.spage16 = static_cast<uint32_t>(p.kv.scale_page_stride / 16);
  a.shead16 = static_cast<uint32_t>(p.kv.scale_head_stride / 16);
  LaunchKernelArgs(reinterpret_cast<const void*>(KvAttendKernel<C>), dim3(grid), dim3(C::THREADS), C::SMEM, s, true, a);
}

// Blocks of four warps that share an item, or of one.  With about as many
// items as warps that run at once, a warp for itself needs no barriers and
// joins less; with few, a warp's records are many.  32 / 8 heads, four warps
// and one: 128 conversations to 100 positions in 8 bits 20.3 and 15.3 us, to
// 2000 70 and 67, 96 to 400 25.0 and 23.1, 64 to 400 18.4 and 18.6, 32 to 100
// 9.2 and 12.7.  In f16, where a step is shorter, 220 to 100 25.5 and 23.1, to
// 400 47.0 and 47.7, to 2000 172 and 181, 128 to 400 31.7 and 33.1.  So half
// the running warps' number of items is the border for codes, and their whole
// number for f16.  Other layouts, 220 conversations of 40 / 8 heads: in 8 bits
// to 400 58 and 38, to 2000 130 and 113, in f16 to 400 56 and 50, to 2000 182
// and 183; 96 in 4 bits to 400 26 and 23; 192 of 24 / 4 heads of 64 in 8 bits
// to 400 18.3 and 17.8, 320 25 and 22.  Near the border short conversations
// would take one warp earlier (160 to 100 of 8 / 8 heads of 64 in f16 15.3 and
// 10.3) and long ones later (192 to 2000 of 24 / 4 in f16 45.5 and 49.4).
template <int D, KvType KIND, bool PACK>
void ByItems(const KvAttendParams& p, int chunks, cudaStream_t s) {
  using One = Cfg<D, KIND, PACK, 1>;
  if (static_cast<int64_t>(p.table.n_seq) * p.kv.n_kv * chunks >= Resident<One>() / (One::QUANT ? 2 : 1)) {
    Launch<One>(p, chunks, s);
  } else {
    Launch<Cfg<D, KIND, PACK, 4>>(p, chunks, s);
  }
}
template <int D, KvType KIND>
void ByQueries(const KvAttendParams& p, cudaStream_t s) {
  const int group = p.n_heads / p.kv.n_kv, chunks = (group + kKvMaxQueries - 1) / kKvMaxQueries;
  if (group <= 4) {
    ByItems<D, KIND, true>(p, chunks, s);
  } else {
    ByItems<D, KIND, false>(p, chunks, s);
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

int64_t KvAttendWorkspace(int n_heads, int n_kv, int head_dim) {
  const int group = n_heads / n_kv, chunks = (group + kKvMaxQueries - 1) / kKvMaxQueries;
  return kKvMaxBlocks * (4 + 8ll * KvRecordFloats((group + chunks - 1) / chunks, head_dim));
}

void LaunchKvAttend(const KvAttendParams& p, cudaStream_t s) {
  p.kv.head_dim == 64 ? ByKind<64>(p, s) : ByKind<128>(p, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(1);
}

}  // namespace rpgb
