// kv.h -- host-side launchers of the paged key-value cache (k_kv.cu, k_kv_attend.cu).
//
// A cache is a pool of pages of one layer, [page][kv head][position][value]
// by default (any strides), and a page table per batch of conversations.
// Quantised caches keep one f16 scale for kKvGroup consecutive values of a
// row: q8 holds int8 codes c (value c * scale), q4 4-bit codes (value
// (c - 8) * scale, two per byte, the even value in the low half).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace rpgb {

enum class KvType : int32_t { kF16 = 0, kQ8 = 1, kQ4 = 2 };
enum class ElemType : int32_t { kF32 = 0, kF16 = 1, kBF16 = 2 };

constexpr int kKvGroup = 64;         // values that share a scale
constexpr int kKvMinPage = 16;       // a page holds whole 16-position units
constexpr int kKvMaxPage = 4096;
constexpr int kKvMaxQueries = 8;     // query heads of a KV head that one attend pass takes
constexpr int64_t kKvMaxStride = int64_t{1} << 35;  // bytes; a sixteenth of it fits 32 bits
constexpr int kKvMaxRows = 1 << 24;  // rows of one call over shared page lists
constexpr int kKvMaxBlocks = 1792;   // bound of the attend grid (sizes the workspace)
// Floats of one attend record: a vector, a maximum and a sum per query, in whole 16 bytes.
#ifdef __CUDACC__
__host__ __device__
#endif
constexpr int KvRecordFloats(int queries, int head_dim) {
  return (queries * (head_dim + 2) + 3) / 4 * 4;
}

struct KvPages {
  KvType type = KvType::kF16;
  int32_t head_dim = 0, n_kv = 0, n_pages = 0;
  int32_t page_log2 = 0;
  char *k = nullptr, *v = nullptr;  // codes
  char *k_scale = nullptr, *v_scale = nullptr;
  int64_t page_stride = 0, head_stride = 0, pos_stride = 0;  // bytes
  int64_t scale_page_stride = 0, scale_head_stride = 0;      // bytes; scales of a head's page are dense
};
// Bytes of one position's codes / scales of one head.
inline int64_t KvRowBytes(KvType t, int head_dim) {
  return t == KvType::kF16 ? 2 * head_dim : (t == KvType::kQ8 ? head_dim : head_dim / 2);
}
inline int64_t KvScaleRowBytes(int head_dim) { return 2 * (head_dim / kKvGroup); }

struct KvTable {
  const int32_t* pages = nullptr;  // [n_seq][stride]: pool page of each page-sized run of positions
  int32_t n_seq = 0, max_pages = 0;
  int64_t stride = 0;  // entries between conversations
};

struct KvAppendParams {
  KvPages kv;
  KvTable table;
  const void* qkv = nullptr;  // [n_tok] rows q | k | v
  int64_t qkv_stride = 0;     // elements
  ElemType type = ElemType::kF32;
  int32_t n_heads = 0;
  const float *q_norm = nullptr, *k_norm = nullptr;  // [head_dim]; null = no norm
  const float* rope = nullptr;  // [rope_positions][head_dim]: cos of the first half, then sin; null = no rotation
  int32_t rope_positions = 0;
  float eps = 0.f;
  const int32_t* seq = nullptr;  // null: row t belongs to conversation t
  const int32_t* pos = nullptr;
  int64_t n_tok = 0;
  void* q_out = nullptr;  // null: q is not wanted
  int64_t q_stride = 0;   // elements
};
void LaunchKvAppend(const KvAppendParams& p, cudaStream_t s);

struct KvGatherParams {
  KvPages kv;
  KvTable table;
  ElemType type = ElemType::kF32;
  const int32_t* seq = nullptr;
  const int32_t* pos = nullptr;
  int64_t n_tok = 0;
  void *k_out = nullptr, *v_out = nullptr;  // either may be null
  int64_t out_stride = 0;                   // elements
  uint32_t magic = 0;  // a constant of the kernel, filled in by LaunchKvGather
};
void LaunchKvGather(const KvGatherParams& p, cudaStream_t s);

struct KvAttendParams {
  KvPages kv;
  KvTable table;
  ElemType type = ElemType::kF32;
  const int32_t* lens = nullptr;    // [n_seq]
  const int32_t* starts = nullptr;  // [n_seq] or null (0)
  const void* q = nullptr;
  int64_t q_stride = 0;  // elements
  int32_t n_heads = 0;
  float scale = 0.f;
  void* out = nullptr;
  int64_t out_stride = 0;  // elements
  void* workspace = nullptr;
  // Positions under prefix[seq] are left out (null: none); out is of out_type;
  // lse[seq][q head] = log2 of the sum of 2^(score log2 e) (null: not wanted).
  const int32_t* prefix = nullptr;
  ElemType out_type = ElemType::kF32;
  float* lse = nullptr;
  // filled in by LaunchKvAttend: a constant of the kernel, and the strides of
  // kv in units of 16 bytes
  uint32_t magic = 0, page16 = 0, head16 = 0, pos16 = 0, spage16 = 0, shead16 = 0;
};
// Workspace bytes of LaunchKvAttend: kKvMaxBlocks counters, which start at
// zero and are zero again after every call, then two records per block.  The
// counters' place does not depend on the shape, so calls of any shapes may
// follow one another on one workspace.
int64_t KvAttendWorkspace(int n_heads, int n_kv, int head_dim);
void LaunchKvAttend(const KvAttendParams& p, cudaStream_t s);

// Attention of several rows that read one page list: the new tokens of a
// conversation (prefix null: lists are the table's rows), or the conversations
// of a group over the positions that they share (the list is that of the
// group's first; ends are the lengths).
struct KvRowsParams {
  KvPages kv;
  KvTable table;
  ElemType type = ElemType::kF32;
  const int32_t* rows = nullptr;  // [n_lists + 1]
  int32_t n_lists = 0;
  int32_t n_rows = 0;
  const int32_t *starts = nullptr, *ends = nullptr;  // [n_rows]; starts null: 0
  const int32_t* prefix = nullptr;                   // [n_rows]
  const void* q = nullptr;
  int64_t q_stride = 0;  // elements
  int32_t n_heads = 0;
  float scale = 0.f, cap = 0.f;
  const float* slopes = nullptr;
  const int32_t* pos = nullptr;
  void* out = nullptr;
  int64_t out_stride = 0;  // elements
  // the rest of a row's attention, to be added: f32 [n_rows][n_heads][head_dim]
  // and its sums [n_rows][n_heads] (KvAttendParams::lse); null: none
  const float *own = nullptr, *own_lse = nullptr;
  void* workspace = nullptr;
};
int64_t KvRowsWorkspace(int n_heads, int n_kv, int head_dim);
void LaunchKvRows(const KvRowsParams& p, cudaStream_t s);

}  // namespace rpgb
