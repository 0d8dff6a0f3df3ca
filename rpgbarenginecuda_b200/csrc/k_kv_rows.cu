// k_kv_rows.cu -- attention of several rows that read one page list: new tokens
// of a conversation, or the conversations of a group over what they share.
//
// Row r, query head h: o = sum_j w_j V_j / sum_j w_j, w_j = 2^(s_j - ref), over the
// positions j that the row sees, s_j = bend(scale q . K_j) log2(e), ref a bound that
// follows the largest score (it moves when a weight would pass 2^15, by as much as
// brings it to 2^7; the result so far is scaled then).  Sums and results are f32.
// Where a call also has attention over other positions (own, own_lse) the two are
// added with the weights 2^lse.
//
// Rows times the heads of a KV head are the rows of two 128-row tiles, so every
// position is read once for up to 256 rows, and both products are tcgen05 ones:
// S = Q K^T from shared memory, O += P V with P in tensor memory (in the columns
// that had S).  An item is such a pair of tiles and the positions that any of its
// rows sees, in steps of 64.  All items' steps are dealt to one block an SM in equal
// shares, whatever the lists' lengths; what begins or ends inside a block's share
// leaves its result, reference and sum as a record, and RowsJoinKernel adds the
// records of an item up in block order (no atomics: calls repeat bit by bit).
//
// Operands of the products are f16.  f16 queries go in as they are, bf16 and f32
// ones times a power of two a row; an f32 row is two f16 terms, hi + lo, which leave
// 2^-22 of it, as are its weights: errors of 6e-7 of the largest value (2^-11 with
// one term).  Codes are exact in f16; K's scale
// multiplies the scores and V's the weights, per 64-value group.  Rows where
// infinities or NaN of an f16 cache reach the result are worked out again one by
// one (PlainRow): a product with a tile's other columns would spread them.
//
// Warps: 8 or 16 have the softmax, one issues the products, one deals items, two
// copy (f16 pages by TMA; codes by cp.async, spread to f16 on the way from one
// place in shared memory to another).  Registers are shared out between them
// by setmaxnreg.
//
// What bounds it: 4 prompts of 4096 over f16, 32 heads of 8 KV heads, bf16: 427 us,
// 720 TFLOP/s of the pairs that are seen.  A step of a tile takes its softmax warps
// some 1400 cycles (exponentials 700 of them, 16 a cycle an SM; reading the scores
// 250, the largest 230, storing weights 80), the two tiles of a block run side by
// side on the same four schedulers, and an item's beginning and end add 400 a step
// at 18 steps an item; the tensor cores are at 40 %.  Over codes of 128 values a
// tile's products and its softmax take turns (one buffer of scores: two groups with
// scales of their own fill the columns), 16 prompts of 1024 over 8 bits 308 us; four
// copying warps and a thread per row gave 298 there and 171 in place of 145 for 6
// prompts of 1501 over 4 bits.  With few steps a block it is what a launch costs: the
// pair of kernels 4 us, the plan 1.6, the roles' first instructions 3.
//
// Tried and not kept, 4 prompts of 4096 at the time: a part of the exponentials as
// polynomials, weights in two halves so that their product begins earlier, results
// through shared memory for whole lines (each slower); mixed f32 + f16 additions for
// the sum (423 -> 422).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "common.h"
#include "kv_dev.cuh"
#include "launch.h"
#include "tc_dev.cuh"

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
struct Bounds {
  int start, end, prefix;  // as the caller gives them
  __device__ __forceinline__ void Load(const KvRowsParams& p, int row) {
    start = p.starts != nullptr ? p.starts[row] : 0;
    end = p.ends[row];
    prefix = p.prefix != nullptr ? p.prefix[row] : 0;
  }
};
__device__ __forceinline__ Seen SeenBy(const KvRowsParams& p, const Bounds& b) {
  const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
  Seen s;
  s.start = max(b.start, 0);
  int64_t end = max(b.end, 0);
  if (p.prefix != nullptr) end = min(end, static_cast<int64_t>(max(b.prefix, 0)));
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

// What scores are bent by, in units of log2.
struct Bend {
  float rate, cap, slope;
  bool capped, biased;
  __device__ __forceinline__ explicit Bend(const KvRowsParams& p, float slope_)
      : rate(p.cap > 0.f ? -2.f * kLog2e / p.cap : 0.f), cap(p.cap * kLog2e), slope(slope_ * kLog2e), capped(p.cap > 0.f),
        biased(p.slopes != nullptr) {}
  // cap tanh(x / cap) of a score of the formula: tanh |t| = (1 - e) / (1 + e) with e = exp(-2 |t|)
  __device__ __forceinline__ float Capped(float x) const {
    const float e = Exp2(fabsf(x) * rate);
    return copysignf(cap * __fdividef(1.f - e, 1.f + e), x);
  }
  __device__ __forceinline__ float operator()(float x, int distance) const {
    x = capped ? Capped(x) : x * kLog2e;
    return biased ? x - slope * fabsf(static_cast<float>(distance)) : x;
  }
};

// One row by the formula, a position at a time, by a warp.
template <int D, KvType KIND>
__device__ __forceinline__ void PlainRow(const KvRowsParams& p, int table_row, int head, int64_t q_at, float slope, int pos,
                                         int from, int to, float (&acc)[D / 32], float& m, float& l) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const Bend bend(p, slope);
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
    const float s = bend(dev::WarpSum(dot) * p.scale, pos - at);
    const float now = fmaxf(m, s), ref = now == -INFINITY ? 0.f : now;
    const float alpha = Exp2(m - ref), w = Exp2(s - ref);
    m = now;
    l = l * alpha + w;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = acc[e] * alpha + w * v[e];
  }
}


// ------------------------------------------------------------------ shapes

constexpr int kTileRows = 128;            // rows of a tile: the lanes of tensor memory
constexpr int kItemRows = 2 * kTileRows;  // two tiles share the positions that pass through
constexpr int kLoadWarps = 2;
constexpr int kMaxBlocks = 160;
constexpr int kItems = 4;    // items described ahead
constexpr int kNotes = 8;    // steps whose bad pages are held
constexpr int kLeast = 2;    // steps that a block is started for
constexpr int kHeadroom = 15, kSlack = 8;  // weights are at most 2^15, and 2^7 when their reference was set

template <int D_, KvType KIND_, bool TWO_>
struct Cfg {
  static constexpr int D = D_;
  static constexpr KvType KIND = KIND_;
  static constexpr bool QUANT = KIND != KvType::kF16;
  static constexpr bool TWO = TWO_;  // q and weights in two f16 terms (f32 activations)
  static constexpr int TERMS = TWO ? 2 : 1;
  // Warps of the softmax: four to a tile and half.  Over codes with one term two
  // threads share a row, half of the positions and half of the values each: what a
  // thread does in turn is what bounds a step there (16 prompts
  // of 1024 over 8 bits 324 -> 308 us, 6 of 1501 over 4 bits 171 -> 145; 64 rows over
  // a prefix of 4096, few steps a block, lose, 60 -> 65).  An f16 cache
  // keeps a thread per row (4 prompts of 4096 423 us; 473 with two, whose exchange of
  // the row's largest score costs more than the shorter turn gives).  With two terms
  // the row's result stays in registers, which takes all of one thread's.
  static constexpr int HALVES = QUANT && !TWO ? 2 : 1;
  static constexpr int SOFT = 8 * HALVES, MMA = SOFT, DEAL = SOFT + 1, LOAD = SOFT + 2, WARPS = LOAD + kLoadWarps;
  static constexpr int THREADS = 32 * WARPS;
  // Registers a thread at launch, and how the groups of four warps share them.
  static constexpr int REGS = HALVES == 1 ? 168 : 96, SOFT_REGS = HALVES == 1 ? 216 : 104, OTHER_REGS = HALVES == 1 ? 72 : 64;
  static_assert(32 * SOFT * SOFT_REGS + 128 * OTHER_REGS <= REGS * THREADS, "registers");
  // Positions of a step.  With 128 a tile's scores take all of its 128 columns of
  // tensor memory and the softmax waits for every product (4 prompts of 4096 over
  // f16 460 us, 423 with 64 and two buffers).
  static constexpr int KT = 64;
  static constexpr int NG = QUANT ? D / kKvGroup : 1;
  static constexpr int COLS = KT / HALVES, DIMS = D / HALVES;  // positions and values of a thread
  static constexpr int BOX = D / 64;                  // 128-byte columns of a tile of f16
  static constexpr int QTERM = BOX * kTileRows * 128, QTILE = TERMS * QTERM;
  static constexpr int PLANE = BOX * KT * 128;
  // Buffers for a tile's scores: 128 columns of tensor memory are there, and a step
  // takes 64 for each group of values that has its own scale.
  static constexpr int BUFS = NG == 1 ? 2 : 1;
  static constexpr int STAGES = QUANT ? (TWO && D == 128 ? 2 : 3) : (TWO ? 3 : 4);
  static constexpr int SCALES = BUFS == 2 ? 8 : 4;  // steps whose scales are held, as they come and as f32
  static constexpr int LAG = QUANT && !TWO ? 4 : 2;  // copies of codes begun before the oldest is waited for
  static constexpr int ROW = KIND == KvType::kF16 ? 2 * D : (KIND == KvType::kQ8 ? D : D / 2);
  static constexpr int CPR = ROW / 16;
  static constexpr int PER = KT * CPR / (32 * kLoadWarps);  // 16-byte pieces of a thread
  static constexpr int RAW = QUANT ? KT * ROW : 0;
  static constexpr int SCALE = QUANT ? 2 * KT * NG * 2 : 0;  // scales of a step: K, then V
  static constexpr int NOTE = 2 * SCALE;                     // the same as f32, [K or V][group][position]
  // Steps that the beginning and end of an item (its queries, its result) count
  // for when the work is dealt.  Codes, 16 prompts of 1024 with 1, 2, 3 and 4: 318,
  // 307, 309, 318 us; f16, 4 of 4096 with 4, 8 and 12: 430, 418, 431; two terms, a
  // prompt of 2811 with 3, 5, 7 and 10: 138, 129, 122, 125.
  static constexpr int BORDER = TWO ? 7 : (QUANT ? 2 : 8);
  static constexpr int SMEM = 1024 + 2 * QTILE + 2 * STAGES * PLANE + (LAG + 1) * RAW + SCALES * (SCALE + NOTE);
  static_assert(SMEM <= 226 * 1024, "shared memory");
};

struct Item {
  int table_row, row0, n_tok, head, chunk;
  int base, lo, hi;      // first position of step 0; positions that any row may see
  int step0, steps;      // 0: no more items
  int first_prefix;
  bool begins, ends;
};
// A piece that begins an item that further blocks end.
struct Job {
  int row0, n_tok, head, chunk, last, pad[3];
};

__host__ __device__ constexpr int64_t RecordFloats(int d) { return static_cast<int64_t>(kItemRows) * (d + 2); }
constexpr int64_t kJobBytes = kMaxBlocks * static_cast<int64_t>(sizeof(Job));

// Query heads of a KV head in chunks of at most kItemRows.
struct Split {
  int group, chunks, per, tokens, items;  // of a chunk; tokens of an item; items of a slot
  __device__ __forceinline__ explicit Split(const KvRowsParams& p) {
    group = p.n_heads / p.kv.n_kv;
    chunks = (group + kItemRows - 1) / kItemRows;
    per = (group + chunks - 1) / chunks;
    tokens = kItemRows / per;
    items = p.kv.n_kv * chunks;
  }
};

// Slots number the items of a head: list s begins at slot rows[s] / tokens + s,
// which leaves room for all its pieces whatever the lists before it hold.
__device__ __forceinline__ int SlotOf(const KvRowsParams& p, const Split& sp, int list) {
  return RowBegin(p, list) / sp.tokens + list;
}
template <typename C>
struct Slots {
  int list = 0;
  __device__ __forceinline__ void Seek(const KvRowsParams& p, const Split& sp, int slot) {
    int lo = 0, hi = p.n_lists - 1;
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      SlotOf(p, sp, mid) <= slot ? lo = mid : hi = mid - 1;
    }
    list = lo;
  }
  // Item of the slot (head and steps taken are the caller's); returns its steps, 0 where there is none.
  __device__ __forceinline__ int Get(const KvRowsParams& p, const Split& sp, int slot, Item& it) {
#pragma unroll 1
    while (list + 1 < p.n_lists && SlotOf(p, sp, list + 1) <= slot) ++list;
    const int begin = RowBegin(p, list), end = RowEnd(p, list);
    const int64_t j = slot - (begin / sp.tokens + list), row0 = begin + j * sp.tokens;
    if (j < 0 || row0 >= end) return 0;
    it.table_row = TableRow(p, list);
    it.row0 = static_cast<int>(row0);
    it.n_tok = min(sp.tokens, end - it.row0);
    const int64_t cap = static_cast<int64_t>(p.table.max_pages) << p.kv.page_log2;
    it.first_prefix = 0;
    if (p.prefix != nullptr) {
      it.first_prefix = max(p.prefix[begin], 0);
      it.lo = 0;
      it.hi = static_cast<int>(min(static_cast<int64_t>(it.first_prefix), cap));
    } else {
      it.lo = p.starts != nullptr ? max(p.starts[it.row0], 0) : 0;
      it.hi = static_cast<int>(min(static_cast<int64_t>(max(p.ends[it.row0 + it.n_tok - 1], 0)), cap));
    }
    if (it.lo >= it.hi) it.lo = it.hi = 0;
    // (an f16 cache's steps begin where pages of as many positions do)
    it.base = it.lo & ~(!C::QUANT && 1 << p.kv.page_log2 >= C::KT ? C::KT - 1 : 15);
    return max(1, (it.hi - it.base + C::KT - 1) / C::KT);
  }
};

// Block b of n has steps [total b / n, total (b + 1) / n), the borders of items
// counted; ShareOf is the block that has step x.
__device__ __forceinline__ int ShareOf(long long x, long long total, int n) {
  return static_cast<int>(((x + 1) * n - 1) / total);
}

// ------------------------------------------------------------------ instructions

__device__ __forceinline__ uint32_t Swz(int row, int chunk) {
  return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4));
}
__device__ __forceinline__ void CopyAsync16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void CopyCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void CopyWait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Bounded wait; one small loop (kernels.cuh's is unrolled, and there are many here).
__device__ __forceinline__ bool Wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 0; i < 1u << 16; ++i) {
    if (dev::MbarTryWait(bar, parity)) return true;
  }
  return false;
}
// Positions at .. of a head's page, from its `box`th 64 values on: as many as the map's boxes have.
__device__ __forceinline__ void LoadTile(void* dst, const CUtensorMap* map, int at, int box, int head, int page,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::
          "r"(dev::SmemAddr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(at), "r"(box), "r"(head), "r"(page), "r"(dev::SmemAddr(bar))
      : "memory");
}
__device__ __forceinline__ void TmemLoad32(uint32_t a, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
__device__ __forceinline__ void TmemLoadWait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void TmemStore32(uint32_t a, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Operands in shared memory as the low words of their descriptors; the high
// word is the same for all: 1024 bytes between groups of eight 128-byte rows,
// version 1, the 128-byte swizzle.  One thread issues a product in about 115
// cycles where it works out 64-bit descriptors, loops and branches for each,
// which is twice what the product takes; unrolled and with 32-bit sums it keeps
// up.
constexpr uint32_t kDescHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
// A tile whose rows are 128 bytes along the sum (q and K).
__device__ __forceinline__ uint32_t DescRows(uint32_t a) { return a >> 4 | 1u << 16; }
// V: the sum runs over rows, and the next 64 values are `box` bytes on.
__device__ __forceinline__ uint32_t DescV(uint32_t a, int box) { return a >> 4 | static_cast<uint32_t>(box >> 4) << 16; }
// Products are issued by one elected lane of a warp that stays together: their
// operands are in uniform registers then.  In a branch of one lane each of them
// waits for its operands to be moved there (4 prompts of 4096 over f16 561 -> 433 us,
// 16 of 1024 over 8 bits 330 -> 307).
__device__ __forceinline__ void MmaSs(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\telect.sync _|e, 0xFFFFFFFF;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(kDescHigh)
      : "memory");
}
// A in tensor memory.
__device__ __forceinline__ void MmaTs(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b;\n\telect.sync _|e, 0xFFFFFFFF;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void Commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xFFFFFFFF;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(dev::SmemAddr(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t PackHalf(float lo, float hi) { return kvd::HalfBits(__floats2half2_rn(lo, hi)); }

// ------------------------------------------------------------------ kernel

struct Bars {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], q_full[2];  // [tile][buffer], [tile]
  uint64_t item_full[kItems], item_empty[kItems], fin;
  uint64_t pair[8];  // of the two warps that have the halves of 32 rows
};

// The ring of items, as a reader sees it.
struct Reader {
  int n = 0;
  __device__ __forceinline__ bool Next(Bars& b, const Item* items, Item& it, int lane) {
    const int i = n % kItems;
    if (!__all_sync(0xFFFFFFFFu, Wait(&b.item_full[i], (n / kItems) & 1))) return false;
    it = items[i];
    __syncwarp();
    if (lane == 0) tc::MbarArrive(&b.item_empty[i]);
    ++n;
    return it.steps > 0;
  }
};

template <typename C>
__device__ __forceinline__ float* RecordOf(const KvRowsParams& p, int block, bool begins) {
  return reinterpret_cast<float*>(static_cast<char*>(p.workspace) + kJobBytes) +
         (2 * block + (begins ? 1 : 0)) * RecordFloats(C::D);
}

// The same for those that go on reading the item where it is, until they let go of it.
struct Holder {
  int n = 0;
  __device__ __forceinline__ const Item* Next(Bars& b, const Item* items) {
    const int i = n % kItems;
    if (!__all_sync(0xFFFFFFFFu, Wait(&b.item_full[i], (n / kItems) & 1))) return nullptr;
    ++n;
    return items + i;
  }
  static __device__ __forceinline__ void Release(Bars& b, const Item* items, const Item* it, int lane) {
    __syncwarp();
    if (lane == 0) tc::MbarArrive(&b.item_empty[it - items]);
  }
};

// How a row's result and what was found elsewhere add up.
struct Join {
  float f = 0.f, g = 0.f;  // of this result, of the other
  __device__ __forceinline__ Join(const KvRowsParams& p, int64_t row_head, float ref, float l) {
    f = l != 0.f ? 1.f / l : 0.f;
    if (p.own != nullptr) {
      const float a = ref + log2f(l), b = p.own_lse[row_head];
      const float top = fmaxf(a, b), base = top == -INFINITY ? 0.f : top;
      const float wa = exp2f(a - base), wb = exp2f(b - base), sum = wa + wb;
      f = sum != 0.f ? f * (wa / sum) : 0.f;
      g = sum != 0.f ? wb / sum : 0.f;
    }
  }
};

// 32 values of an output row.
__device__ __forceinline__ void Put32(const KvRowsParams& p, int64_t at, const float* y) {
  if (p.type == ElemType::kF32) {
    uint4* o = reinterpret_cast<uint4*>(static_cast<float*>(p.out) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = make_uint4(__float_as_uint(y[4 * i]), __float_as_uint(y[4 * i + 1]), __float_as_uint(y[4 * i + 2]),
                        __float_as_uint(y[4 * i + 3]));
    }
  } else {
    uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at);
    uint32_t w[16];
    if (p.type == ElemType::kF16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = PackHalf(y[2 * i], y[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

// A thread's values of a query row into the tile, the sign of the softmax scale
// in them: f16 ones as they are, others times 2^-e (the row's largest value in
// [2^12, 2^13)) as f16 terms.  `most_of` makes the largest magnitude that of the
// whole row.  Returns the factor from products to scores, NaN for a row that is
// not finite.
template <typename C, typename T, typename F>
__device__ __forceinline__ float WriteQ(const KvRowsParams& p, int64_t at, bool there, char* tile, int row, int chunk0,
                                        F most_of) {
  constexpr bool kF32 = sizeof(T) == 4, kF16 = std::is_same<T, __half>::value;
  constexpr int kChunks = C::DIMS / 8;
  kvd::Raw8<T> q[kChunks];  // all on their way at once
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (there) {
      q[c].Load(static_cast<const T*>(p.q) + at + 8 * (chunk0 + c));
    } else {
#pragma unroll
      for (int i = 0; i < kvd::Raw8<T>::N; ++i) q[c].w[i] = make_uint4(0, 0, 0, 0);
    }
  }
  // the bits of the largest magnitude: those of infinity and NaN are above all others
  uint32_t most = 0;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
#pragma unroll
    for (int i = 0; i < kvd::Raw8<T>::N; ++i) {
      for (const uint32_t w : {q[c].w[i].x, q[c].w[i].y, q[c].w[i].z, q[c].w[i].w}) {
        most = kF32 ? max(most, w & 0x7FFFFFFFu) : __vmaxu2(most, w & 0x7FFF7FFFu);
      }
    }
  }
  if (!kF32) most = max(most & 0xFFFFu, most >> 16) << 16;
  most = most_of(most);
  const bool finite = most < (kF16 ? 0x7C000000u : 0x7F800000u);
  const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0;
  float f0 = 1.f, f1 = 1.f;
  if (!kF16) {
    const int e = most > 0 && finite ? max(static_cast<int>(most >> 23), 1) - 127 - 12 : 0;
    // 2^-e in two factors: each is a normal number
    f0 = __uint_as_float(static_cast<uint32_t>(127 - e / 2) << 23);
    f1 = __uint_as_float(static_cast<uint32_t>(127 - (e - e / 2)) << 23);
  }
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    uint32_t hi[4], lo[4];
    if (kF16) {
      const uint4 w = q[c].w[0];
      hi[0] = w.x ^ sign;
      hi[1] = w.y ^ sign;
      hi[2] = w.z ^ sign;
      hi[3] = w.w ^ sign;
    } else {
      float x[8];
      q[c].Floats(x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = __fmul2_rn(__fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(f0, f0)), make_float2(f1, f1));
        hi[i] = PackHalf(y.x, y.y);
        if (C::TWO) {
          const float2 h = __half22float2(kvd::BitsHalf(hi[i]));
          lo[i] = PackHalf(y.x - h.x, y.y - h.y) ^ sign;
        }
        hi[i] ^= sign;
      }
    }
    char* dst = tile + ((chunk0 + c) >> 3) * (kTileRows * 128) + Swz(row, (chunk0 + c) & 7);
    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (C::TWO) *reinterpret_cast<uint4*>(dst + C::QTERM) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  return finite ? fabsf(p.scale) / f0 / f1 : kvd::Nan();
}

// A row of an item, as the thread that has it sees it.
struct RowState {
  const Item* it;
  int note0;  // steps before the item
  int row, qh;
  Bounds bounds;
  Seen seen;
  float cs, slope;  // scores (in units of log2 where they are not capped) are products times cs
  int pos;
  bool valid, active, is_nan;  // active: some row of the warp is valid
};

// An f16 cache's planes, in boxes of 16 positions and 64 values and, where pages hold them, of whole steps.
struct Maps {
  CUtensorMap k, v, step_k, step_v;
};

template <typename C>
__global__ void __launch_bounds__(C::THREADS, 1) RowsKernel(const __grid_constant__ Maps maps,
                                                            const KvRowsParams p, uint32_t magic) {
  using namespace tc;
  constexpr int D = C::D, KT = C::KT;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ Item items[kItems];
  __shared__ uint32_t s_tmem, s_bad[kNotes], s_pair[2][2][2 * kTileRows];
  __shared__ int2 s_seen[kLoadWarps][C::SCALES];  // a warp's own notes of what a step's rows see
  __shared__ long long s_part[C::THREADS / 32], s_before;
  __shared__ int s_slot;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* s_q = smem;
  char* s_k = s_q + 2 * C::QTILE;
  char* s_v = s_k + C::STAGES * C::PLANE;
  char* s_raw = s_v + C::STAGES * C::PLANE;
  char* s_scale = s_raw + (C::LAG + 1) * C::RAW;
  char* s_note = s_scale + C::SCALES * C::SCALE;
  const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
  const Split sp(p);

  if (warp == 0) TmemAlloc(&s_tmem, 512u);
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      dev::MbarInit(&bars.k_full[i], C::QUANT ? kLoadWarps : 1);
      dev::MbarInit(&bars.v_full[i], C::QUANT ? kLoadWarps : 1);
      dev::MbarInit(&bars.k_empty[i], 1);
      dev::MbarInit(&bars.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      for (int b = 0; b < 2; ++b) {
        dev::MbarInit(&bars.s_full[i][b], 1);
        dev::MbarInit(&bars.pv_done[i][b], 1);
        dev::MbarInit(&bars.p_full[i][b], C::SOFT / 2);
      }
      dev::MbarInit(&bars.q_full[i], C::SOFT / 2);
    }
    for (int i = 0; i < kItems; ++i) {
      dev::MbarInit(&bars.item_full[i], 1);
      dev::MbarInit(&bars.item_empty[i], C::SOFT + kLoadWarps + 1);
    }
    dev::MbarInit(&bars.fin, 1);
    for (int i = 0; i < 8; ++i) dev::MbarInit(&bars.pair[i], 2);
    dev::MbarInitFence();
  }
  dev::GridLaunchDependents();
  dev::GridWait();

  // ---- this block's share of the steps: a run of slots per thread, their steps added up
  const int n_slots = p.n_rows / sp.tokens + p.n_lists;
  const int run = (n_slots + C::THREADS - 1) / C::THREADS;
  const int slot_lo = min(tid * run, n_slots), slot_hi = min(slot_lo + run, n_slots);
  long long mine = 0;
  {
    Slots<C> sl;
    Item it;
    if (slot_lo < slot_hi) sl.Seek(p, sp, slot_lo);
#pragma unroll 1
    for (int i = slot_lo; i < slot_hi; ++i) {
      const int steps = sl.Get(p, sp, i, it);
      mine += steps > 0 ? steps + C::BORDER : 0;
    }
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_part[warp] = incl;
  FenceBeforeSync();
  __syncthreads();
  FenceAfterSync();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, s_tmem, 0);
  long long before = incl - mine, per_head = 0;
#pragma unroll 1
  for (int w = 0; w < C::THREADS / 32; ++w) {
    if (w < warp) before += s_part[w];
    per_head += s_part[w];
  }
  const long long total = per_head * sp.items;
  const int blocks = static_cast<int>(min(static_cast<long long>(gridDim.x), max(total / kLeast, 1ll)));
  const int block = blockIdx.x;
  const long long x0 = block < blocks ? total * block / blocks : total;
  const long long x1 = block < blocks ? total * (block + 1) / blocks : total;
  const long long rem = per_head > 0 ? x0 % per_head : 0;
  if (x0 < x1 && before <= rem && rem < before + mine) {
    s_slot = slot_lo;
    s_before = before;
  }
  __syncthreads();
  if (warp >= C::SOFT) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
    if (warp == C::DEAL) {
      // ---- items of this block, in order
      Job job{};
      Slots<C> sl;
      int n = 0, slot = 0, hc = 0;
      long long x = x0, skip = 0;
      if (x0 < x1) {
        slot = s_slot;
        skip = rem - s_before;  // steps of the run to leave out
        hc = static_cast<int>(x0 / per_head);
        sl.Seek(p, sp, slot);
      }
      bool ok = true;
#pragma unroll 1
      for (bool more = true; more && ok;) {
        Item it;
        it.steps = 0;
        it.n_tok = 0;
        if (x < x1) {
          const int steps = sl.Get(p, sp, slot, it);
          const int weight = steps > 0 ? steps + C::BORDER : 0;
          if (steps <= skip) {  // nothing of it, or its border alone
            x += weight > skip ? weight - skip : 0;
            skip -= min(skip, static_cast<long long>(weight));
            it.steps = -1;
          } else {
            it.step0 = static_cast<int>(skip);
            it.steps = static_cast<int>(min(static_cast<long long>(steps) - skip, x1 - x));
            it.head = hc / sp.chunks;
            it.chunk = hc % sp.chunks;
            it.begins = it.step0 == 0;
            it.ends = it.step0 + it.steps == steps;
            if (it.begins && !it.ends) {
              job.row0 = it.row0;
              job.n_tok = it.n_tok;
              job.head = it.head;
              job.chunk = it.chunk;
              job.last = min(max(ShareOf(x + steps - 1, total, blocks), block), blocks - 1);
            }
            x += it.steps + (it.ends ? C::BORDER : 0);
            skip = 0;
          }
          if (++slot == n_slots) {
            slot = 0;
            ++hc;
            sl.list = 0;
          }
          if (it.steps < 0) continue;
        } else {
          more = false;
        }
        const int i = n % kItems;
        if (n >= kItems) ok = __all_sync(0xFFFFFFFFu, Wait(&bars.item_empty[i], (n / kItems - 1) & 1));
        if (!ok) break;
        if (lane == 0) {
          items[i] = it;
          MbarArrive(&bars.item_full[i]);
        }
        __syncwarp();
        ++n;
        // its queries on their way into L2, an item or more before they are read
        const int size = p.type == ElemType::kF32 ? 4 : 2;
        const int heads = it.steps > 0 ? min(sp.per, sp.group - it.chunk * sp.per) : 0;
        const int lines = (heads * D * size + 127) / 128;
#pragma unroll 1
        for (int k = lane; k < it.n_tok * lines; k += 32) {
          const int64_t at = (it.row0 + k / lines) * p.q_stride + static_cast<int64_t>(it.head * sp.group + it.chunk * sp.per) * D;
          asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(p.q) + at * size + k % lines * 128));
        }
      }
      if (lane == 0) static_cast<Job*>(p.workspace)[block] = job;
    } else if (warp == C::MMA) {
      // ---- products: per step and tile S = Q K^T, and O += P V of the step before.
      // With two buffers the scores come first, so that they are there when the
      // softmax is done with those before; their buffer had the weights of two
      // steps ago, whose product is issued.
      {
        constexpr uint32_t id_s = InstrDesc(128, KT);
        constexpr uint32_t id_o = InstrDesc(128, C::NG == 1 ? D : 64) | 1u << 16;  // (V: values contiguous)
        const uint32_t a_q = dev::SmemAddr(s_q), a_k = dev::SmemAddr(s_k), a_v = dev::SmemAddr(s_v);
        int n = 0;
        uint32_t q_parity = 0;
        int c = 0, ct0 = 0, ct1 = 0;  // steps so far, and those of each tile
        bool ok = true;
#pragma unroll 1
        while (ok) {
          const int i = n % kItems;
          if (!__all_sync(0xFFFFFFFFu, Wait(&bars.item_full[i], (n / kItems) & 1))) break;
          const int steps = __shfl_sync(0xFFFFFFFFu, items[i].steps, 0);
          const int rows = __shfl_sync(0xFFFFFFFFu, items[i].n_tok * sp.per, 0);
          if (lane == 0) MbarArrive(&bars.item_empty[i]);
          __syncwarp();
          ++n;
          if (steps <= 0) break;
          const int tiles = rows > kTileRows ? 2 : 1;
#pragma unroll 1
          for (int j = 0; j <= steps && ok; ++j) {
            auto pv = [&](int t) {
              const int n = c + j - 1, st = n % C::STAGES, nt = (t == 0 ? ct0 : ct1) + j - 1, buf = nt % C::BUFS;
              ok = __all_sync(0xFFFFFFFFu, (t > 0 || Wait(&bars.v_full[st], (n / C::STAGES) & 1)) &&
                                               Wait(&bars.p_full[t][buf], (nt / C::BUFS) & 1));
              if (!ok) return;
              FenceAfterSync();
              const uint32_t o = tmem + 256 + t * 128, w = tmem + t * 128 + buf * 64;
              // with two terms every step's product starts anew (it is added up in registers)
              const bool going_on = !C::TWO && j > 1;
#pragma unroll
              for (int g = 0; g < C::NG; ++g) {
#pragma unroll
                for (int term = C::TERMS - 1; term >= 0; --term) {
                  const uint32_t v = DescV(a_v + st * C::PLANE + g * (KT * 128), KT * 128);
                  const uint32_t a = w + (g * C::TERMS + term) * (KT / 2), d = o + 64 * g;
#pragma unroll
                  for (int k = 0; k < KT / 16; ++k) {
                    MmaTs(d, a + 8 * k, v + k * (2048 >> 4), id_o, k > 0 || term < C::TERMS - 1 || going_on);
                  }
                }
              }
              Commit(&bars.pv_done[t][buf]);
              if (t == tiles - 1) Commit(&bars.v_empty[st]);
            };
            auto qk = [&](int t) {
              const int n = c + j, st = n % C::STAGES, buf = ((t == 0 ? ct0 : ct1) + j) % C::BUFS;
              ok = __all_sync(0xFFFFFFFFu, (j > 0 || Wait(&bars.q_full[t], q_parity >> t & 1)) &&
                                               (t > 0 || Wait(&bars.k_full[st], (n / C::STAGES) & 1)));
              if (!ok) return;
              if (j == 0) q_parity ^= 1u << t;
              FenceAfterSync();
              // (second terms first: the sums that the tensor cores cut short are small then)
#pragma unroll
              for (int term = C::TERMS - 1; term >= 0; --term) {
#pragma unroll
                for (int box = 0; box < C::BOX; ++box) {
                  const uint32_t d = tmem + t * 128 + (C::NG == 2 ? 64 * box : 64 * buf);
                  const uint32_t q = DescRows(a_q + t * C::QTILE + term * C::QTERM + box * (kTileRows * 128));
                  const uint32_t kk = DescRows(a_k + st * C::PLANE + box * (KT * 128));
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    MmaSs(d, q + 2 * k, kk + 2 * k, id_s, k > 0 || term < C::TERMS - 1 || (C::NG == 1 && box > 0));
                  }
                }
              }
              Commit(&bars.s_full[t][buf]);
              if (t == tiles - 1) Commit(&bars.k_empty[st]);
            };
            // With two terms both tiles' scores come first (a prompt of 40 24.9 us, not
            // 25.6); with one, a tile's products together (4 of 4096 430 us, not 440).
            if constexpr (C::BUFS == 2 && C::TWO) {
#pragma unroll 1
              for (int t = 0; t < tiles && ok && j < steps; ++t) qk(t);
#pragma unroll 1
              for (int t = 0; t < tiles && ok && j > 0; ++t) pv(t);
            } else {
#pragma unroll 1
              for (int t = 0; t < tiles && ok; ++t) {
                if (C::BUFS == 2 && j < steps) qk(t);
                if (ok && j > 0) pv(t);
                if (C::BUFS == 1 && ok && j < steps) qk(t);
              }
            }
          }
          c += steps;
          ct0 += steps;
          if (tiles == 2) ct1 += steps;
        }
        Commit(&bars.fin);  // no product is under way when the block ends
        Wait(&bars.fin, 0);
      }
      __syncwarp();
    } else {
      // ---- copies
      const int lt = tid - 32 * C::LOAD, lw = lt >> 5;
      const int mask = (1 << p.kv.page_log2) - 1;
      int begun = 0, ended = 0;  // copies: of codes 2 n is K's of step n and 2 n + 1 V's, of f16 n is step n's
      bool ok = true;
      asm volatile("fence.proxy.async.global;" ::: "memory");  // (what kernels before this one stored is read by copies)
      const uint32_t a_raw = dev::SmemAddr(s_raw), a_scale = dev::SmemAddr(s_scale);
      const int c0 = lt % C::CPR, r0 = lt / C::CPR;  // piece and first row of this thread
      constexpr int kRowStep = 32 * kLoadWarps / C::CPR;
      // The oldest copy of codes has arrived: spread them to f16, tell the products.
      auto finish = [&]() {
        const int step = ended >> 1, st = step % C::STAGES;
        const bool v = ended & 1;
        if (!__all_sync(0xFFFFFFFFu, Wait(v ? &bars.v_empty[st] : &bars.k_empty[st], ((step / C::STAGES) & 1) ^ 1))) {
          ok = false;
          return;
        }
        const char* raw = s_raw + ended % (C::LAG + 1) * C::RAW + lt * 16;
        char* dst = (v ? s_v : s_k) + st * C::PLANE;
#pragma unroll 2
        for (int i = 0; i < C::PER; ++i) {
          const int r = r0 + i * kRowStep;
          const uint4 w = *reinterpret_cast<const uint4*>(raw + i * (32 * kLoadWarps * 16));
          constexpr int kHalves = C::KIND == KvType::kQ8 ? 1 : 2;  // runs of 16 values
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            kvd::Codes16<C::KIND> code;
            if (C::KIND == KvType::kQ8) {
              code.w[0] = w.x;
              code.w[1] = w.y;
              code.w[C::KIND == KvType::kQ8 ? 2 : 0] = w.z;
              code.w[C::KIND == KvType::kQ8 ? 3 : 0] = w.w;
            } else {
              code.w[0] = h == 0 ? w.x : w.z;
              code.w[1] = h == 0 ? w.y : w.w;
            }
            uint32_t y[8];
            code.Pairs(y, magic);
            const int u = (c0 * kHalves + h) * 2;  // 8-value chunk of the row
            char* d = dst + (u >> 3) * (KT * 128);
            *reinterpret_cast<uint4*>(d + Swz(r, u & 7)) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4*>(d + Swz(r, (u & 7) + 1)) = make_uint4(y[4], y[5], y[6], y[7]);
          }
        }
        if (!v) {
          // the scales that this warp copied, group after group; 0 where no row sees the position
          __syncwarp();
          const int2 seen = s_seen[lw][step % C::SCALES];
          const __half* h = reinterpret_cast<const __half*>(s_scale + step % C::SCALES * C::SCALE + lw * (C::SCALE / 2));
          float* f = reinterpret_cast<float*>(s_note + step % C::SCALES * C::NOTE + lw * (C::NOTE / 2));
#pragma unroll 1
          for (int i = lane; i < KT * C::NG; i += 32) {
            const int pos = i / C::NG;
            f[i % C::NG * KT + pos] = pos >= seen.x && pos < seen.y ? __half2float(h[i]) : 0.f;
          }
        }
        dev::FenceProxyAsync();
        __syncwarp();
        if (lane == 0) MbarArrive(v ? &bars.v_full[st] : &bars.k_full[st]);
        ++ended;
      };
      Reader rd;
      Item it;
#pragma unroll 1
      while (ok && rd.Next(bars, items, it, lane)) {
        // lane g has to do with positions 16 g .. 16 g + 15 of a step: their page
        auto lookup = [&](int pos) {
          return lane < KT / 16 && pos + 16 > it.lo && pos < it.hi
                     ? p.table.pages[it.table_row * p.table.stride + (pos >> p.kv.page_log2)]
                     : -1;
        };
        int next = lookup(it.base + it.step0 * KT + 16 * lane);
#pragma unroll 1
        for (int j = 0; j < it.steps && ok; ++j) {
          const int pos0 = it.base + (it.step0 + j) * KT, at = pos0 + 16 * lane;
          const int page = next;
          if (j + 1 < it.steps) next = lookup(at + KT);
          const bool used = lane < KT / 16 && at + 16 > it.lo && at < it.hi;
          const bool there = used && static_cast<unsigned>(page) < static_cast<unsigned>(p.kv.n_pages);
          const uint32_t have = __ballot_sync(0xFFFFFFFFu, there);
          const uint32_t bad = __ballot_sync(0xFFFFFFFFu, used && !there);
          const int64_t off = there ? kvd::CodeOffset(p.kv, page, it.head, at & mask) : 0;
          if (lt == 0) s_bad[(C::QUANT ? begun >> 1 : begun) % kNotes] = bad;
          if (C::QUANT && lane == 0) s_seen[lw][(begun >> 1) % C::SCALES] = make_int2(it.lo - pos0, it.hi - pos0);
          if (!C::QUANT) {
            // By TMA: whole steps where a page holds them, or else 16 positions and 64
            // values at a time.  One warp has K, the other V.  (A lane takes some 100
            // cycles for each copy: 128 conversations over 4 prefixes of 16384 in pages
            // of 64 122 us with 16 copies a step, 117 with two.)
            const uint32_t full = __ballot_sync(0xFFFFFFFFu, there && at >= it.lo && at + 16 <= it.hi);
            constexpr uint32_t kAll = (1u << KT / 16) - 1;
            const bool v = lw != 0;
            const int st = begun % C::STAGES, g = lane / C::BOX, box = lane % C::BOX;
            const int pg = __shfl_sync(0xFFFFFFFFu, page, g & 31), in = (pos0 + 16 * g) & mask;
            uint64_t *empty = v ? &bars.v_empty[st] : &bars.k_empty[st], *whole = v ? &bars.v_full[st] : &bars.k_full[st];
            if (!__all_sync(0xFFFFFFFFu, Wait(empty, ((begun / C::STAGES) & 1) ^ 1))) {
              ok = false;
              break;
            }
            char* dst = (v ? s_v : s_k) + st * C::PLANE;
            const uint32_t take = v ? full : have;
            uint32_t rest = v ? kAll & ~full : 0;
            if (rest != 0) {
              // V of positions that no row sees may hold anything, and zero times NaN is NaN: zeros instead
#pragma unroll 1
              while (rest != 0) {
                const int q = __ffs(rest) - 1;
                rest &= rest - 1;
                const char* src = p.kv.v + __shfl_sync(0xFFFFFFFFu, off, q);
#pragma unroll 1
                for (int i = lane; i < 16 * C::CPR; i += 32) {
                  const int r = i / C::CPR, c = i % C::CPR, pos = pos0 + 16 * q + r;
                  const bool seen = ((have >> q) & 1) && pos >= it.lo && pos < it.hi;
                  CopyAsync16(dev::SmemAddr(dst + (c >> 3) * (KT * 128) + Swz(16 * q + r, c & 7)),
                              seen ? src + r * p.kv.pos_stride + c * 16 : p.kv.v, seen);
                }
              }
              CopyCommit();
              CopyWait<0>();
              dev::FenceProxyAsync();
            }
            __syncwarp();
            if (lane == 0) dev::MbarExpectTx(whole, __popc(take) * (C::BOX * 2048));  // (an arrival too)
            __syncwarp();
            if (take == kAll && (1 << p.kv.page_log2) >= KT && (pos0 & (KT - 1)) == 0) {
              if (lane == 0) LoadTile(dst, v ? &maps.step_v : &maps.step_k, pos0 & mask, 0, it.head, pg, whole);
            } else if (lane < KT / 16 * C::BOX && ((take >> g) & 1)) {
              LoadTile(dst + box * (KT * 128) + g * 2048, v ? &maps.v : &maps.k, in, box, it.head, pg, whole);
            }
            ++begun;
          } else {
#pragma unroll 1
            for (int v = 0; v < 2 && ok; ++v) {
              const char* plane = (v ? p.kv.v : p.kv.k) + c0 * 16;
              const uint32_t dst = a_raw + begun % (C::LAG + 1) * C::RAW + lt * 16;
              // 16 positions at a time: rows r0 + k * kRowStep of them are this thread's
#pragma unroll 1
              for (int g = 0; g < KT / 16; ++g) {
                const char* src = plane + __shfl_sync(0xFFFFFFFFu, off, g);
                const bool have_g = (have >> g) & 1;
                const int first = pos0 + 16 * g;
                auto copy = [&](uint32_t to, int r) {
                  const bool in = have_g && first + r >= it.lo && first + r < it.hi;
                  CopyAsync16(to, in ? src + r * p.kv.pos_stride : plane, in);
                };
                if (kRowStep > 16) {  // (a thread has rows of every other sixteen)
                  constexpr int kSkip = kRowStep > 16 ? kRowStep / 16 : 1;
                  if ((r0 >> 4) == g % kSkip) copy(dst + g / kSkip * (32 * kLoadWarps * 16), r0 & 15);
                } else {
#pragma unroll
                  for (int k = 0; k < 16 / kRowStep; ++k) copy(dst + g * (16 * C::ROW) + k * (kRowStep * C::ROW), r0 + k * kRowStep);
                }
              }
              if (v == 0) {
                // scales of K and V: 16 positions are dense, 2 NG 16-byte pieces
                constexpr int kPer = 2 * C::NG;
                const int i = lane / kPer % (KT / 16);
                const int64_t so = there ? kvd::ScaleOffset(p.kv, page, it.head, at & mask) : 0;
                const int64_t o = __shfl_sync(0xFFFFFFFFu, so, i) + lane % kPer * 16;
                if (lane < KT / 16 * kPer) {
                  const bool in = (have >> i) & 1;
                  const char* src = lw == 0 ? p.kv.k_scale : p.kv.v_scale;
                  CopyAsync16(a_scale + (begun >> 1) % C::SCALES * C::SCALE + lw * (C::SCALE / 2) + lane * 16, in ? src + o : src, in);
                }
              }
              CopyCommit();
              ++begun;
              if (begun - ended > C::LAG) {
                CopyWait<C::LAG>();
                finish();
              }
            }
          }
        }
      }
      if (C::QUANT) {
        CopyWait<0>();
        while (ok && ended < begun) finish();
      } else if (begun > 0) {
        // copies that nobody waits for any more have landed before the block ends
        for (int n = max(0, begun - C::STAGES); n < begun; ++n) {
          const int st = n % C::STAGES;
          Wait(lw != 0 ? &bars.v_full[st] : &bars.k_full[st], (n / C::STAGES) & 1);
        }
      }
    }
  } else {
    // ---- softmax: a thread per row, or two
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFT_REGS));
    const int t = warp / (4 * C::HALVES), half = C::HALVES == 2 ? (warp >> 2) & 1 : 0;
    const int in_tile = (warp & 3) * 32 + lane, r = t * kTileRows + in_tile;
    const int col0 = half * C::COLS, dim0 = half * C::DIMS;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t a_t = lanes + t * 128, a_o = lanes + 256 + t * 128 + dim0;
    uint32_t pair_parity = 0;
    int c = 0, note = 0;  // steps so far, of this tile and all
    bool ok = true;
    // What the thread with the row's other half has in its place.
    auto other = [&](uint32_t v) -> uint32_t {
      uint32_t* place = s_pair[pair_parity][t];
      place[half * kTileRows + in_tile] = v;
      FenceBeforeSync();  // (what either has read of tensor memory, the other may write over)
      __syncwarp();
      uint64_t* bar = &bars.pair[t * 4 + (warp & 3)];
      if (lane == 0) MbarArrive(bar);
      if (!__all_sync(0xFFFFFFFFu, Wait(bar, pair_parity))) ok = false;
      FenceAfterSync();
      pair_parity ^= 1;
      return place[(half ^ 1) * kTileRows + in_tile];
    };
    Holder rd;
    const Item* first_item = items;
    // The next item that this tile has rows of, and what the thread has to know of its row.
    auto next_item = [&](RowState& w) {
      for (;;) {
        w.it = rd.Next(bars, items);
        if (w.it == nullptr) return false;
        w.note0 = note;
        note += w.it->steps;
        if (w.it->steps <= 0) return false;
        if (t == 0 || w.it->n_tok * sp.per > kTileRows) break;
        Holder::Release(bars, first_item, w.it, lane);
      }
      const int tok = r / sp.per, g = r - tok * sp.per + w.it->chunk * sp.per;
      w.valid = tok < w.it->n_tok && g < sp.group;
      w.active = __any_sync(0xFFFFFFFFu, w.valid);
      w.row = w.it->row0 + tok;
      w.qh = w.it->head * sp.group + g;
      w.seen = Seen{0, 0, false};
      w.cs = w.slope = 0.f;
      w.pos = 0;
      w.is_nan = false;
      if (w.valid) {  // (on their way while the queries are read)
        w.bounds.Load(p, w.row);
        if (p.slopes != nullptr) {
          w.slope = p.slopes[w.qh];
          w.pos = p.pos[w.row];
        }
      }
      return true;
    };
    auto write_q = [&](RowState& w) {
      if (w.active) {
        const int64_t q_at = w.row * p.q_stride + static_cast<int64_t>(w.qh) * D;
        char* tile = s_q + t * C::QTILE;
        auto most_of = [&](uint32_t most) { return C::HALVES == 2 ? max(most, other(most)) : most; };
        if (C::TWO) {
          w.cs = WriteQ<C, float>(p, q_at, w.valid, tile, in_tile, dim0 / 8, most_of);
        } else {
          w.cs = p.type == ElemType::kF16 ? WriteQ<C, __half>(p, q_at, w.valid, tile, in_tile, dim0 / 8, most_of)
                                          : WriteQ<C, __nv_bfloat16>(p, q_at, w.valid, tile, in_tile, dim0 / 8, most_of);
        }
      }
      if (w.valid) {
        w.seen = SeenBy(p, w.bounds);
        const Seen& s = w.seen;
        w.is_nan = s.past || (s.start < s.end && (s.start < w.it->lo || s.end > w.it->hi)) || !(w.cs == w.cs) ||
                   (p.prefix != nullptr && w.bounds.prefix > w.it->first_prefix);
        if (!(p.cap > 0.f)) w.cs = fmaxf(w.cs * kLog2e, 1e-37f);  // (a scale of 0: minus infinity times it is to stay)
      }
      dev::FenceProxyAsync();
      __syncwarp();
      if (lane == 0) MbarArrive(&bars.q_full[t]);
    };
    RowState now{};  // (nothing, before the first item)
    bool more = true;
#pragma unroll 1
    while (ok && more) {
      const int steps = now.it != nullptr ? now.it->steps : 0, note0 = now.note0, row = now.row, qh = now.qh;
      const Seen seen = now.seen;
      const float cs = now.cs, slope = now.slope;
      const int pos = now.pos;
      const bool valid = now.valid, active = now.active;
      bool nan_row = now.is_nan;
      const Bend bend(p, slope);
      float m = -INFINITY, ref = -INFINITY, l = 0.f;
      int nu = C::QUANT ? -30 : 0;
      float2 acc[C::TWO ? D / 2 : 1];  // the result of the steps before the last
      if (C::TWO) {
#pragma unroll
        for (int i = 0; i < D / 2; ++i) acc[i % (C::TWO ? D / 2 : 1)] = make_float2(0.f, 0.f);
      }
      auto ProductsDone = [&]() {  // those with V of the last step
        if (!__all_sync(0xFFFFFFFFu, Wait(&bars.pv_done[t][(c - 1) % C::BUFS], ((c - 1) / C::BUFS) & 1))) return false;
        FenceAfterSync();
        return true;
      };
      // Softmax of a step's scores, weights into tensor memory.  EDGE: some row of the warp does not see all positions.
      auto step = [&](auto edge, int j, int from, int to, int pos0, const float* scales) {
        constexpr bool EDGE = decltype(edge)::value;
        const uint32_t a_s = a_t + c % C::BUFS * 64;
        if (C::TWO && j > 0) {
          if (!ProductsDone()) return false;  // (they came before these scores)
#pragma unroll
          for (int k = 0; k < D; k += 32) {
            uint32_t o[32];
            TmemLoad32(a_o + k, o);
            TmemLoadWait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2& a = acc[(k / 2 + i) % (C::TWO ? D / 2 : 1)];
              a = __fadd2_rn(a, make_float2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])));
            }
          }
        }
        float2 s[C::COLS / 2];
        uint32_t* u = reinterpret_cast<uint32_t*>(s);
        if (C::NG == 2) {
          // the parts of the two groups, each times its scale
#pragma unroll
          for (int h = 0; h < C::COLS; h += 16) {
            uint32_t b[16];
            TmemLoad16(a_s + col0 + h, *reinterpret_cast<uint32_t(*)[16]>(u + h));
            TmemLoad16(a_s + 64 + col0 + h, b);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 d0 = *reinterpret_cast<const float4*>(scales + col0 + h + i);
              const float4 d1 = *reinterpret_cast<const float4*>(scales + KT + col0 + h + i);
              float2 &x = s[(h + i) / 2], &y = s[(h + i) / 2 + 1];
              const float2 bx = make_float2(__uint_as_float(b[i]), __uint_as_float(b[i + 1]));
              const float2 by = make_float2(__uint_as_float(b[i + 2]), __uint_as_float(b[i + 3]));
              x = __ffma2_rn(bx, make_float2(d1.x, d1.y), __fmul2_rn(x, make_float2(d0.x, d0.y)));
              y = __ffma2_rn(by, make_float2(d1.z, d1.w), __fmul2_rn(y, make_float2(d0.z, d0.w)));
            }
          }
        } else {
#pragma unroll
          for (int h = 0; h < C::COLS; h += 32) TmemLoad32(a_s + col0 + h, u + h);
          TmemLoadWait();
          if (C::QUANT) {
#pragma unroll
            for (int i = 0; i < C::COLS; i += 4) {
              const float4 d = *reinterpret_cast<const float4*>(scales + col0 + i);
              s[i / 2] = __fmul2_rn(s[i / 2], make_float2(d.x, d.y));
              s[i / 2 + 1] = __fmul2_rn(s[i / 2 + 1], make_float2(d.z, d.w));
            }
          }
        }
        if (bend.capped) {
#pragma unroll
          for (int i = 0; i < C::COLS; ++i) u[i] = __float_as_uint(bend.Capped(__uint_as_float(u[i]) * cs));
        }
        if (bend.biased) {
          const float first = static_cast<float>(pos - pos0 - col0), f = bend.capped ? 1.f : cs;
#pragma unroll
          for (int i = 0; i < C::COLS; ++i) {
            u[i] = __float_as_uint(__uint_as_float(u[i]) * f - bend.slope * fabsf(first - static_cast<float>(i)));
          }
        }
        if (EDGE) {
#pragma unroll
          for (int i = 0; i < C::COLS; ++i) {
            if (i < from || i >= to) u[i] = __float_as_uint(-INFINITY);
          }
        }
        float2 top = s[0], top2 = s[1];
#pragma unroll
        for (int i = 2; i + 3 < C::COLS / 2; i += 4) {  // (three at a time is one instruction)
          top.x = fmaxf(fmaxf(top.x, s[i].x), s[i + 1].x);
          top.y = fmaxf(fmaxf(top.y, s[i].y), s[i + 1].y);
          top2.x = fmaxf(fmaxf(top2.x, s[i + 2].x), s[i + 3].x);
          top2.y = fmaxf(fmaxf(top2.y, s[i + 2].y), s[i + 3].y);
        }
        static_assert(C::COLS / 2 % 4 == 0, "two pairs are left");
        top.x = fmaxf(fmaxf(top.x, s[C::COLS / 2 - 2].x), s[C::COLS / 2 - 1].x);
        top.y = fmaxf(fmaxf(top.y, s[C::COLS / 2 - 2].y), s[C::COLS / 2 - 1].y);
        float mx = fmaxf(fmaxf(top.x, top.y), fmaxf(top2.x, top2.y));
        if (C::HALVES == 2) {
          mx = fmaxf(mx, __uint_as_float(other(__float_as_uint(mx))));
          if (!ok) return false;
        }
        const float to_log2 = bend.capped || bend.biased ? 1.f : cs;
        if (C::QUANT) {
          // an exponent over the step's V scales
          const float* vs = scales + C::NG * KT;
          float most = 0.f;
#pragma unroll
          for (int i = 0; i < KT * C::NG / 32; ++i) most = fmaxf(most, fabsf(vs[32 * i + lane]));
          most = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most)));
          nu = max(nu, static_cast<int>(__float_as_uint(most) >> 23) - 126);
        }
        m = fmaxf(m, mx * to_log2);
        const float over = m + static_cast<float>(nu);
        const bool grow = over > ref + static_cast<float>(kHeadroom);
        float alpha = 1.f;
        bool rescale = false;
        if (__any_sync(0xFFFFFFFFu, grow)) {
          const float now = grow ? over - static_cast<float>(kHeadroom - kSlack) : ref;
          if (grow && ref != -INFINITY) alpha = exp2f(ref - now);
          ref = now;
          l *= alpha;
          rescale = __any_sync(0xFFFFFFFFu, alpha != 1.f);
        }
        if (rescale && C::TWO) {
#pragma unroll
          for (int i = 0; i < D / 2; ++i) {
            float2& a = acc[i % (C::TWO ? D / 2 : 1)];
            a = __fmul2_rn(a, make_float2(alpha, alpha));
          }
        }
        if (rescale && !C::TWO && j > 0) {
          if (!ProductsDone()) return false;
#pragma unroll 1
          for (int k = 0; k < C::DIMS; k += 32) {
            uint32_t o[32];
            TmemLoad32(a_o + k, o);
            TmemLoadWait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            TmemStore32(a_o + k, o);
          }
        }
        const float less = ref == -INFINITY ? 0.f : -ref;
        const float2 f2 = make_float2(to_log2, to_log2), less2 = make_float2(less, less);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int h = 0; h < C::COLS; h += 32) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2& x = s[h / 2 + i];
            x = __ffma2_rn(x, f2, less2);
            x = make_float2(Exp2(x.x), Exp2(x.y));
            if (C::TWO || C::QUANT) sum = __fadd2_rn(sum, x);
            if (!C::QUANT) {
              w[i] = PackHalf(x.x, x.y);
              // (weights of one term are added up as they are used)
              if (!C::TWO) sum = __fadd2_rn(sum, __half22float2(kvd::BitsHalf(w[i])));
            }
          }
          if (!C::QUANT) {
            TmemStore16(a_s + (col0 + h) / 2, w);
            if (C::TWO) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 x = s[h / 2 + i], f = __half22float2(kvd::BitsHalf(w[i]));
                w[i] = PackHalf(x.x - f.x, x.y - f.y);
              }
              TmemStore16(a_s + 32 + h / 2, w);
            }
          }
        }
        l += sum.x + sum.y;
        if (C::QUANT) {
          // times the scales of each group's values
          const float* vs = scales + C::NG * KT;
#pragma unroll
          for (int gp = 0; gp < C::NG; ++gp) {
#pragma unroll
            for (int h = 0; h < C::COLS; h += 32) {
              uint32_t w[16], w2[16];
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 d = *reinterpret_cast<const float4*>(vs + gp * KT + col0 + h + i);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int k = h + i + 2 * e, at = i / 2 + e;
                  float2 y = __fmul2_rn(s[k / 2], e == 0 ? make_float2(d.x, d.y) : make_float2(d.z, d.w));
                  if (EDGE) {  // (a scale that the row does not see may be NaN)
                    if (k < from || k >= to) y.x = 0.f;
                    if (k + 1 < from || k + 1 >= to) y.y = 0.f;
                  }
                  w[at] = PackHalf(y.x, y.y);
                  if (C::TWO) {
                    const float2 f = __half22float2(kvd::BitsHalf(w[at]));
                    w2[at] = PackHalf(y.x - f.x, y.y - f.y);
                  }
                }
              }
              TmemStore16(a_s + gp * C::TERMS * 32 + (col0 + h) / 2, w);
              if (C::TWO) TmemStore16(a_s + (gp * C::TERMS + 1) * 32 + h / 2, w2);
            }
          }
        }
        TmemStoreWait();
        FenceBeforeSync();
        return true;
      };
#pragma unroll 1
      for (int j = 0; j < steps; ++j) {
        if (!__all_sync(0xFFFFFFFFu, Wait(&bars.s_full[t][c % C::BUFS], (c / C::BUFS) & 1))) {
          ok = false;
          break;
        }
        FenceAfterSync();
        if (active) {
          const int pos0 = now.it->base + (now.it->step0 + j) * KT;
          const int from = min(max(seen.start - pos0, 0), KT), to = min(max(seen.end - pos0, 0), KT);  // columns seen
          const uint32_t bad = s_bad[(note0 + j) % kNotes];
          if (bad != 0 && from < to) {
            // columns from .. to - 1 in units of 16
            if (bad & ((2u << ((to - 1) >> 4)) - 1u) & ~((1u << (from >> 4)) - 1u)) nan_row = true;
          }
          const float* scales = reinterpret_cast<const float*>(s_note + (note0 + j) % C::SCALES * C::NOTE);
          const bool edge = __any_sync(0xFFFFFFFFu, valid && (from > 0 || to < KT));
          if (!(edge ? step(std::true_type(), j, from - col0, to - col0, pos0, scales)
                     : step(std::false_type(), j, from - col0, to - col0, pos0, scales))) {
            ok = false;
            break;
          }
        }
        __syncwarp();
        if (lane == 0) MbarArrive(&bars.p_full[t][c % C::BUFS]);
        ++c;
      }
      // The next item's queries go into the place of this one's (whose products
      // with K are done) before this one's result is taken, so that the tensor
      // cores have work meanwhile.  (With two terms the registers do not hold both.)
      RowState then{};
      more = ok && next_item(then);
      if (!C::TWO && more) write_q(then);
      // ---- the end of the item, or of this block's piece of it
      if (ok && steps > 0 && !__all_sync(0xFFFFFFFFu, Wait(&bars.pv_done[t][(c - 1) % C::BUFS], ((c - 1) / C::BUFS) & 1))) ok = false;
      FenceAfterSync();
      const int64_t row_head = static_cast<int64_t>(row) * p.n_heads + qh;
      const int64_t out = row * p.out_stride + static_cast<int64_t>(qh) * D;
      if (nan_row || !ok) l = kvd::Nan();  // (a wait that gave up is not to pass for a result)
      if (active) {
        const bool whole = now.it->begins && now.it->ends;
        float* rec = RecordOf<C>(p, block, now.it->begins);
        if (C::HALVES == 2) l += __uint_as_float(other(__float_as_uint(l)));
        const Join jn = valid && whole ? Join(p, row_head, ref, l) : Join(p, 0, 0.f, 0.f);
        float check = 0.f;
#pragma unroll (C::TWO ? D / 32 : 1)
        for (int k = 0; k < C::DIMS; k += 32) {
          uint32_t o[32];
          TmemLoad32(a_o + k, o);
          TmemLoadWait();
          float y[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            y[i] = __uint_as_float(o[i]);
            if (C::TWO) y[i] += reinterpret_cast<const float*>(acc)[(k + i) % (C::TWO ? D : 1)];
            check += y[i] * 0.f;
          }
          if (valid && whole) {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = l == 0.f ? 0.f : y[i] * jn.f;
            if (p.own != nullptr) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 w = *reinterpret_cast<const float4*>(p.own + row_head * D + dim0 + k + i);
                y[i] += jn.g * w.x;
                y[i + 1] += jn.g * w.y;
                y[i + 2] += jn.g * w.z;
                y[i + 3] += jn.g * w.w;
              }
            }
            Put32(p, out + dim0 + k, y);
          } else if (valid) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(y[i + e]);
              kvd::Store32(rec + r * D + dim0 + k + i, w);
            }
          }
        }
        if (valid && !whole && half == 0) {
          rec[kItemRows * D + r] = ref;
          rec[kItemRows * (D + 1) + r] = l;
        }
        if (!C::QUANT) {
          // infinities and NaN: such rows again, by the formula
          uint32_t bad = valid && !nan_row && ok && !(check + l * 0.f == 0.f);
          if (C::HALVES == 2) bad |= other(bad);  // (and the other half's values are written)
          uint32_t again = __ballot_sync(0xFFFFFFFFu, bad != 0 && half == 0 && ok);
          const int from = now.it->base + now.it->step0 * KT, to = from + steps * KT;
#pragma unroll 1
          while (again != 0) {
            const int w = __ffs(again) - 1;
            again &= again - 1;
            const int start = __shfl_sync(0xFFFFFFFFu, seen.start, w), end = __shfl_sync(0xFFFFFFFFu, seen.end, w);
            constexpr int N = D / 32;
            float acc[N], pm, pl;
            PlainRow<D, C::KIND>(p, now.it->table_row, now.it->head, __shfl_sync(0xFFFFFFFFu, row * p.q_stride + static_cast<int64_t>(qh) * D, w),
                                 __shfl_sync(0xFFFFFFFFu, slope, w), __shfl_sync(0xFFFFFFFFu, pos, w), max(start, from),
                                 min(end, to), acc, pm, pl);
            const int rr = __shfl_sync(0xFFFFFFFFu, r, w);
            const int64_t rh = __shfl_sync(0xFFFFFFFFu, row_head, w), oo = __shfl_sync(0xFFFFFFFFu, out, w);
            if (whole) {
              const Join jp(p, rh, pm, pl);
#pragma unroll
              for (int e = 0; e < N; ++e) {
                float y = pl == 0.f ? 0.f : acc[e] * jp.f;
                if (p.own != nullptr) y += jp.g * p.own[rh * D + lane * N + e];
                Put(p.out, p.type, oo + lane * N + e, y);
              }
            } else {
#pragma unroll
              for (int e = 0; e < N; ++e) rec[rr * D + lane * N + e] = acc[e];
              if (lane == 0) {
                rec[kItemRows * D + rr] = pm;
                rec[kItemRows * (D + 1) + rr] = pl;
              }
            }
          }
        }
      }
      FenceBeforeSync();  // (what was read of tensor memory, before the next item's products)
      if (now.it != nullptr) Holder::Release(bars, first_item, now.it, lane);
      if (C::TWO && more) write_q(then);
      now = then;
    }
  }
  __syncthreads();
  if (warp == 0) TmemDealloc(tmem, 512u);
}

// Joins the pieces of the items that several blocks had, in block order: block
// (b, y) the rows y, y + gridDim.y, ... (in units of 256 threads) of the item
// that begins in block b.  What bounds it is the pieces' way through L2, so
// eight of them are on their way at once.
constexpr int kJoinBlocks = 16;
template <typename C>
__global__ void __launch_bounds__(256) RowsJoinKernel(const KvRowsParams p) {
  constexpr int D = C::D, kVec = D / 4, kRows = 256 / kVec;  // threads of a row, rows of a block at once
  dev::GridLaunchDependents();
  dev::GridWait();
  const Job job = static_cast<const Job*>(p.workspace)[blockIdx.x];
  if (job.n_tok == 0) return;
  const Split sp(p);
  const int b0 = blockIdx.x, n = job.last - b0 + 1, i = threadIdx.x % kVec;
  for (int r = blockIdx.y * kRows + threadIdx.x / kVec; r < job.n_tok * sp.per; r += kJoinBlocks * kRows) {
    const int tok = r / sp.per, g = r - tok * sp.per + job.chunk * sp.per;
    if (g >= sp.group) continue;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kFlight = 8;
    for (int k0 = 0; k0 < n; k0 += kFlight) {
      float ref[kFlight], l[kFlight];
      float4 x[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        ref[k] = -INFINITY;
        l[k] = 0.f;
        if (k0 + k < n) {
          const float* q = RecordOf<C>(p, b0 + k0 + k, k0 + k == 0);
          ref[k] = q[kItemRows * D + r];
          l[k] = q[kItemRows * (D + 1) + r];
          x[k] = reinterpret_cast<const float4*>(q + r * D)[i];
        }
      }
      float now = top;
#pragma unroll
      for (int k = 0; k < kFlight; ++k) now = fmaxf(now, ref[k]);
      const float base = now == -INFINITY ? 0.f : now, keep = exp2f(top - base);
      v = make_float4(v.x * keep, v.y * keep, v.z * keep, v.w * keep);
      sum *= keep;
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        if (l[k] != 0.f) {
          const float f = exp2f(ref[k] - base);
          sum += f * l[k];
          v.x += f * x[k].x;
          v.y += f * x[k].y;
          v.z += f * x[k].z;
          v.w += f * x[k].w;
        }
      }
      top = now;
    }
    const int row = job.row0 + tok, qh = job.head * sp.group + g;
    const int64_t row_head = static_cast<int64_t>(row) * p.n_heads + qh;
    const Join jn(p, row_head, top, sum);
    float y[4] = {v.x * jn.f, v.y * jn.f, v.z * jn.f, v.w * jn.f};
    if (sum == 0.f) y[0] = y[1] = y[2] = y[3] = 0.f;
    if (p.own != nullptr) {
      const float4 w = reinterpret_cast<const float4*>(p.own + row_head * D)[i];
      y[0] += jn.g * w.x;
      y[1] += jn.g * w.y;
      y[2] += jn.g * w.z;
      y[3] += jn.g * w.w;
    }
    const int64_t out = row * p.out_stride + static_cast<int64_t>(qh) * D + 4 * i;
    switch (p.type) {
      case ElemType::kF32: kvd::Store4(static_cast<float*>(p.out) + out, y); break;
      case ElemType::kF16: kvd::Store4(static_cast<__half*>(p.out) + out, y); break;
      case ElemType::kBF16: kvd::Store4(static_cast<__nv_bfloat16*>(p.out) + out, y); break;
    }
  }
}

PFN_cuTensorMapEncodeTiled_v12000 Encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }
  });
  RPGB_CHECK(fn != nullptr, "kv: cuTensorMapEncodeTiled is unavailable");
  return fn;
}

// A plane of an f16 cache, [page][head][64 values][position][value] by its strides, in boxes of some positions and 64 values
// `columns` times.
CUtensorMap PlaneMap(const KvPages& kv, char* plane, int positions, int columns) {
  CUtensorMap m;
  const cuuint64_t dims[5] = {64, cuuint64_t{1} << kv.page_log2, static_cast<cuuint64_t>(kv.head_dim / 64),
                              static_cast<cuuint64_t>(kv.n_kv), static_cast<cuuint64_t>(kv.n_pages)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(kv.pos_stride), 128, static_cast<cuuint64_t>(kv.head_stride),
                                 static_cast<cuuint64_t>(kv.page_stride)};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(positions), static_cast<cuuint32_t>(columns), 1, 1};
  const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
  const CUresult r = Encode()(&m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, plane, dims, strides, box, steps,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RPGB_CHECK(r == CUDA_SUCCESS, "kv: tensor map encoding failed (%d)", static_cast<int>(r));
  return m;
}

template <typename C>
int Grid() {
  static std::atomic<int> grids[64];
  int dev = 0;
  RPGB_CUDA(cudaGetDevice(&dev));
  RPGB_CHECK(dev < 64, "kv: device %d", dev);
  int grid = grids[dev].load(std::memory_order_acquire);
  if (grid == 0) {
    int sms = 0;
    RPGB_CUDA(cudaFuncSetAttribute(RowsKernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    cudaFuncAttributes attr;
    RPGB_CUDA(cudaFuncGetAttributes(&attr, RowsKernel<C>));
    RPGB_CHECK(attr.numRegs == C::REGS, "kv: the rows kernel has %d registers a thread, not %d", attr.numRegs, C::REGS);
    RPGB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    grid = sms < kMaxBlocks ? sms : kMaxBlocks;
    grids[dev].store(grid, std::memory_order_release);
  }
  return grid;
}

template <typename C>
void Launch(const KvRowsParams& p, cudaStream_t s) {
  const int grid = Grid<C>();
  Maps maps{};
  if (!C::QUANT) {
    maps.k = PlaneMap(p.kv, p.kv.k, 16, 1);
    maps.v = PlaneMap(p.kv, p.kv.v, 16, 1);
    if (1 << p.kv.page_log2 >= C::KT) {
      maps.step_k = PlaneMap(p.kv, p.kv.k, C::KT, C::BOX);
      maps.step_v = PlaneMap(p.kv, p.kv.v, C::KT, C::BOX);
    }
  }
  LaunchKernelArgs(reinterpret_cast<const void*>(RowsKernel<C>), dim3(grid), dim3(C::THREADS), C::SMEM, s, true, maps, p,
                   kvd::kMagic);
  LaunchKernelArgs(reinterpret_cast<const void*>(RowsJoinKernel<C>), dim3(grid, kJoinBlocks), dim3(256), 0, s, true, p);
}

template <int D, KvType KIND>
void ByType(const KvRowsParams& p, cudaStream_t s) {
  p.type == ElemType::kF32 ? Launch<Cfg<D, KIND, true>>(p, s) : Launch<Cfg<D, KIND, false>>(p, s);
}
template <int D>
void ByKind(const KvRowsParams& p, cudaStream_t s) {
  switch (p.kv.type) {
    case KvType::kF16: return ByType<D, KvType::kF16>(p, s);
    case KvType::kQ8: return ByType<D, KvType::kQ8>(p, s);
    case KvType::kQ4: return ByType<D, KvType::kQ4>(p, s);
  }
}

}  // namespace

int64_t KvRowsWorkspace(int, int, int head_dim) { return kJobBytes + 2ll * kMaxBlocks * RecordFloats(head_dim) * 4; }

void LaunchKvRows(const KvRowsParams& p, cudaStream_t s) {
  p.kv.head_dim == 64 ? ByKind<64>(p, s) : ByKind<128>(p, s);
  RPGB_CUDA(cudaGetLastError());
  CountLaunches(2);
}

}  // namespace rpgb
