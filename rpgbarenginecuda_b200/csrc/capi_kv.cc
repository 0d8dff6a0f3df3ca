// capi_kv.cc -- extern "C" entry points of the paged key-value cache and of the
// sampling of a batch (include/rpg_b200.h): argument checks, then the launchers
// of kv.h and sample_rows.h.
#include <climits>
#include <cmath>

#include "../../include/rpg_b200.h"
#include "common.h"
#include "kv.h"
#include "sample_rows.h"

using namespace rpgb;

namespace {

void CheckAligned(const void* p, uintptr_t a, const char* what) {
  RPGB_CHECK(reinterpret_cast<uintptr_t>(p) % a == 0, "%s is not aligned to %d bytes", what, static_cast<int>(a));
}

KvPages Pages(const rpgb_kv_pages* d) {
  RPGB_CHECK(d != nullptr, "kv: pages is NULL");
  RPGB_CHECK(d->type == RPGB_KV_F16 || d->type == RPGB_KV_Q8 || d->type == RPGB_KV_Q4, "kv: unknown cache type %d",
             d->type);
  RPGB_CHECK(d->head_dim == 64 || d->head_dim == 128, "kv: head_dim %d; the kernels are built for 64 and 128",
             d->head_dim);
  RPGB_CHECK(d->n_kv > 0 && d->n_kv <= 4096, "kv: bad KV head count %d", d->n_kv);
  RPGB_CHECK(d->n_pages > 0, "kv: bad page count %d", d->n_pages);
  RPGB_CHECK(d->page_size >= kKvMinPage && d->page_size <= kKvMaxPage && (d->page_size & (d->page_size - 1)) == 0,
             "kv: page size %d; a power of two from %d to %d is needed", d->page_size, kKvMinPage, kKvMaxPage);
  KvPages p;
  p.type = static_cast<KvType>(d->type);
  p.head_dim = d->head_dim;
  p.n_kv = d->n_kv;
  p.n_pages = d->n_pages;
  while ((1 << p.page_log2) < d->page_size) ++p.page_log2;
  p.k = static_cast<char*>(d->k);
  p.v = static_cast<char*>(d->v);
  RPGB_CHECK(p.k != nullptr && p.v != nullptr, "kv: page memory is NULL");
  CheckAligned(p.k, 16, "kv: k");
  CheckAligned(p.v, 16, "kv: v");
  const int64_t row = KvRowBytes(p.type, p.head_dim);
  p.page_stride = d->page_stride;
  p.head_stride = d->head_stride;
  p.pos_stride = d->pos_stride;
  for (const int64_t s : {p.page_stride, p.head_stride, p.pos_stride}) {
    RPGB_CHECK(s >= row && s % 16 == 0 && s <= kKvMaxStride,
               "kv: stride %lld; a multiple of 16 bytes of at least a row (%lld) is needed",
               static_cast<long long>(s), static_cast<long long>(row));
  }
  if (p.type != KvType::kF16) {
    p.k_scale = static_cast<char*>(d->k_scale);
    p.v_scale = static_cast<char*>(d->v_scale);
    RPGB_CHECK(p.k_scale != nullptr && p.v_scale != nullptr, "kv: a quantised cache needs k_scale and v_scale");
    CheckAligned(p.k_scale, 16, "kv: k_scale");
    CheckAligned(p.v_scale, 16, "kv: v_scale");
    const int64_t page = KvScaleRowBytes(p.head_dim) << p.page_log2;
    p.scale_page_stride = d->scale_page_stride;
    p.scale_head_stride = d->scale_head_stride;
    for (const int64_t s : {p.scale_page_stride, p.scale_head_stride}) {
      RPGB_CHECK(s >= page && s % 16 == 0 && s <= kKvMaxStride,
                 "kv: scale stride %lld; a multiple of 16 bytes of at least a page's scales (%lld) is needed",
                 static_cast<long long>(s), static_cast<long long>(page));
    }
  }
  return p;
}

KvTable Table(const rpgb_kv_table* d, int page_log2) {
  RPGB_CHECK(d != nullptr, "kv: table is NULL");
  RPGB_CHECK(d->n_seq >= 0 && d->n_seq <= (1 << 20), "kv: bad conversation count %d", d->n_seq);
  RPGB_CHECK(d->max_pages > 0 && d->stride >= d->max_pages, "kv: bad page table (%d pages, stride %lld)", d->max_pages,
             static_cast<long long>(d->stride));
  RPGB_CHECK(d->pages != nullptr || d->n_seq == 0, "kv: page table is NULL");
  RPGB_CHECK(d->max_pages <= (1 << 30) >> page_log2, "kv: %d pages of %d positions; at most 2^30 positions are taken",
             d->max_pages, 1 << page_log2);
  CheckAligned(d->pages, 4, "kv: page table");
  KvTable t;
  t.pages = d->pages;
  t.n_seq = d->n_seq;
  t.max_pages = d->max_pages;
  t.stride = d->stride;
  return t;
}

ElemType Type(int32_t t) {
  RPGB_CHECK(t == RPGB_F32 || t == RPGB_F16 || t == RPGB_BF16, "kv: unknown element type %d", t);
  return static_cast<ElemType>(t);
}

// A row-major activation matrix: rows of `cols` elements, 16-byte aligned.
void CheckRows(const void* p, int64_t stride, int64_t cols, ElemType t, const char* what) {
  RPGB_CHECK(p != nullptr, "kv: %s is NULL", what);
  CheckAligned(p, 16, what);
  const int64_t size = t == ElemType::kF32 ? 4 : 2;
  RPGB_CHECK(stride >= cols && stride * size % 16 == 0,
             "kv: %s rows of %lld elements with stride %lld; a multiple of 16 bytes of at least a row is needed", what,
             static_cast<long long>(cols), static_cast<long long>(stride));
}

void CheckTokens(const int32_t* pos, int64_t n_tok, const int32_t* seq, const KvTable& t) {
  RPGB_CHECK(n_tok >= 0 && n_tok <= INT_MAX, "kv: bad row count %lld", static_cast<long long>(n_tok));
  RPGB_CHECK(pos != nullptr || n_tok == 0, "kv: positions are NULL");
  RPGB_CHECK(seq != nullptr || n_tok <= t.n_seq, "kv: %lld rows without conversation ids for %d conversations",
             static_cast<long long>(n_tok), t.n_seq);
}

void CheckShape(int32_t n_heads, int32_t n_kv, int32_t head_dim) {
  RPGB_CHECK(n_kv > 0 && n_kv <= 4096 && n_heads > 0 && n_heads <= 65535 && n_heads % n_kv == 0 &&
                 (head_dim == 64 || head_dim == 128),
             "kv: bad shape (%d heads over %d KV heads of %d)", n_heads, n_kv, head_dim);
}
void CheckWorkspace(const void* p, int64_t bytes, int64_t need) {
  RPGB_CHECK(p != nullptr && bytes >= need, "kv: workspace of %lld bytes; %lld are needed",
             static_cast<long long>(p != nullptr ? bytes : 0), static_cast<long long>(need));
  CheckAligned(p, 256, "kv: workspace");
}

// Parts of the workspace of rpgb_kv_attend_shared.  The counters of the attend
// kernel, which stay zero between calls, come first whatever the batch.
struct SharedWorkspace {
  int64_t attend = 0, rows, own, own_lse, total;
};
SharedWorkspace SharedParts(int n_heads, int n_kv, int head_dim, int n_seq) {
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  SharedWorkspace w;
  w.rows = up(KvAttendWorkspace(n_heads, n_kv, head_dim));
  w.own = w.rows + up(KvRowsWorkspace(n_heads, n_kv, head_dim));
  w.own_lse = w.own + up(4ll * n_seq * n_heads * head_dim);
  w.total = w.own_lse + up(4ll * n_seq * n_heads);
  return w;
}

}  // namespace

#define RPGB_CATCH(ret)                                     \
  catch (const std::exception& e) {                         \
    SetLastError(e.what());                                 \
    return ret;                                             \
  }                                                         \
  catch (...) {                                             \
    SetLastError("unknown exception (not std::exception)"); \
    return ret;                                             \
  }

extern "C" {

int32_t rpgb_kv_append(const rpgb_kv_pages* kv, const rpgb_kv_table* table, const rpgb_kv_rotary* rotary, int32_t type,
                       const void* qkv_dev, int64_t qkv_stride, int32_t n_heads, const int32_t* seq_dev,
                       const int32_t* pos_dev, int64_t n_tok, void* q_out_dev, int64_t q_stride, void* stream) {
  try {
    SetLastError("");
    KvAppendParams p;
    p.kv = Pages(kv);
    p.table = Table(table, p.kv.page_log2);
    p.type = Type(type);
    CheckTokens(pos_dev, n_tok, seq_dev, p.table);
    RPGB_CHECK(n_heads >= 0 && n_heads <= 65535, "kv: bad head count %d", n_heads);
    if (rotary != nullptr) {
      p.q_norm = rotary->q_norm;
      p.k_norm = rotary->k_norm;
      p.rope = rotary->rope;
      p.rope_positions = rotary->rope_positions;
      p.eps = rotary->eps;
      RPGB_CHECK(p.rope == nullptr || p.rope_positions > 0, "kv: bad rotation table length %d", p.rope_positions);
      RPGB_CHECK(p.eps >= 0.f, "kv: bad norm epsilon %g", static_cast<double>(p.eps));
      CheckAligned(p.q_norm, 16, "kv: q_norm");
      CheckAligned(p.k_norm, 16, "kv: k_norm");
      CheckAligned(p.rope, 16, "kv: rope");
    }
    if (n_tok == 0) return 0;
    CheckRows(qkv_dev, qkv_stride, (n_heads + 2ll * p.kv.n_kv) * p.kv.head_dim, p.type, "qkv");
    if (q_out_dev != nullptr) {
      RPGB_CHECK(n_heads > 0, "kv: q_out without q heads");
      CheckRows(q_out_dev, q_stride, static_cast<int64_t>(n_heads) * p.kv.head_dim, p.type, "q_out");
    }
    p.qkv = qkv_dev;
    p.qkv_stride = qkv_stride;
    p.n_heads = n_heads;
    p.seq = seq_dev;
    p.pos = pos_dev;
    p.n_tok = n_tok;
    p.q_out = q_out_dev;
    p.q_stride = q_stride;
    LaunchKvAppend(p, static_cast<cudaStream_t>(stream));
    return 0;
  }
  RPGB_CATCH(-1)
}

int32_t rpgb_kv_gather(const rpgb_kv_pages* kv, const rpgb_kv_table* table, int32_t type, const int32_t* seq_dev,
                       const int32_t* pos_dev, int64_t n_tok, void* k_out_dev, void* v_out_dev, int64_t out_stride,
                       void* stream) {
  try {
    SetLastError("");
    KvGatherParams p;
    p.kv = Pages(kv);
    p.table = Table(table, p.kv.page_log2);
    p.type = Type(type);
    CheckTokens(pos_dev, n_tok, seq_dev, p.table);
    if (n_tok == 0) return 0;
    RPGB_CHECK(k_out_dev != nullptr || v_out_dev != nullptr, "kv: k_out and v_out are NULL");
    const int64_t cols = static_cast<int64_t>(p.kv.n_kv) * p.kv.head_dim;
    if (k_out_dev != nullptr) CheckRows(k_out_dev, out_stride, cols, p.type, "k_out");
    if (v_out_dev != nullptr) CheckRows(v_out_dev, out_stride, cols, p.type, "v_out");
    p.seq = seq_dev;
    p.pos = pos_dev;
    p.n_tok = n_tok;
    p.k_out = k_out_dev;
    p.v_out = v_out_dev;
    p.out_stride = out_stride;
    LaunchKvGather(p, static_cast<cudaStream_t>(stream));
    return 0;
  }
  RPGB_CATCH(-1)
}

int64_t rpgb_kv_attend_workspace(int32_t n_heads, int32_t n_kv, int32_t head_dim) {
  try {
    SetLastError("");
    CheckShape(n_heads, n_kv, head_dim);
    return KvAttendWorkspace(n_heads, n_kv, head_dim);
  }
  RPGB_CATCH(-1)
}

int32_t rpgb_kv_attend(const rpgb_kv_pages* kv, const rpgb_kv_table* table, int32_t type, const void* q_dev,
                       int64_t q_stride, int32_t n_heads, const int32_t* lens_dev, const int32_t* starts_dev,
                       float scale, void* out_dev, int64_t out_stride, void* workspace_dev, int64_t workspace_bytes,
                       void* stream) {
  try {
    SetLastError("");
    KvAttendParams p;
    p.kv = Pages(kv);
    p.table = Table(table, p.kv.page_log2);
    p.type = Type(type);
    RPGB_CHECK(n_heads > 0 && n_heads <= 65535 && n_heads % p.kv.n_kv == 0, "kv: %d q heads over %d KV heads", n_heads,
               p.kv.n_kv);
    if (p.table.n_seq == 0) return 0;
    const int64_t cols = static_cast<int64_t>(n_heads) * p.kv.head_dim;
    CheckRows(q_dev, q_stride, cols, p.type, "q");
    CheckRows(out_dev, out_stride, cols, p.type, "out");
    RPGB_CHECK(lens_dev != nullptr, "kv: lengths are NULL");
    RPGB_CHECK(std::isfinite(scale), "kv: the scale is not finite");
    CheckWorkspace(workspace_dev, workspace_bytes, KvAttendWorkspace(n_heads, p.kv.n_kv, p.kv.head_dim));
    p.lens = lens_dev;
    p.starts = starts_dev;
    p.q = q_dev;
    p.q_stride = q_stride;
    p.n_heads = n_heads;
    p.scale = scale;
    p.out = out_dev;
    p.out_type = p.type;
    p.out_stride = out_stride;
    p.workspace = workspace_dev;
    LaunchKvAttend(p, static_cast<cudaStream_t>(stream));
    return 0;
  }
  RPGB_CATCH(-1)
}

int64_t rpgb_kv_attend_rows_workspace(int32_t n_heads, int32_t n_kv, int32_t head_dim) {
  try {
    SetLastError("");
    CheckShape(n_heads, n_kv, head_dim);
    return KvRowsWorkspace(n_heads, n_kv, head_dim);
  }
  RPGB_CATCH(-1)
}

int32_t rpgb_kv_attend_rows(const rpgb_kv_pages* kv, const rpgb_kv_table* table, int32_t type, const void* q_dev,
                            int64_t q_stride, int32_t n_heads, const int32_t* rows_dev, int64_t n_rows,
                            const int32_t* ends_dev, const int32_t* starts_dev, const rpgb_kv_scores* scores,
                            void* out_dev, int64_t out_stride, void* workspace_dev, int64_t workspace_bytes,
                            void* stream) {
  try {
    SetLastError("");
    KvRowsParams p;
    p.kv = Pages(kv);
    p.table = Table(table, p.kv.page_log2);
    p.type = Type(type);
    RPGB_CHECK(n_heads > 0 && n_heads <= 65535 && n_heads % p.kv.n_kv == 0, "kv: %d q heads over %d KV heads", n_heads,
               p.kv.n_kv);
    RPGB_CHECK(n_rows >= 0 && n_rows <= kKvMaxRows, "kv: bad row count %lld", static_cast<long long>(n_rows));
    RPGB_CHECK(scores != nullptr, "kv: scores is NULL");
    RPGB_CHECK(std::isfinite(scores->scale), "kv: the scale is not finite");
    RPGB_CHECK(std::isfinite(scores->cap) && scores->cap >= 0.f, "kv: bad cap %g", static_cast<double>(scores->cap));
    RPGB_CHECK(scores->slopes == nullptr || scores->pos != nullptr, "kv: slopes need the rows' positions");
    CheckAligned(scores->slopes, 4, "kv: slopes");
    CheckAligned(scores->pos, 4, "kv: row positions");
    if (p.table.n_seq == 0 || n_rows == 0) return 0;
    const int64_t cols = static_cast<int64_t>(n_heads) * p.kv.head_dim;
    CheckRows(q_dev, q_stride, cols, p.type, "q");
    CheckRows(out_dev, out_stride, cols, p.type, "out");
    RPGB_CHECK(rows_dev != nullptr && ends_dev != nullptr, "kv: rows or ends are NULL");
    CheckAligned(rows_dev, 4, "kv: rows");
    CheckAligned(ends_dev, 4, "kv: ends");
    CheckAligned(starts_dev, 4, "kv: starts");
    CheckWorkspace(workspace_dev, workspace_bytes, KvRowsWorkspace(n_heads, p.kv.n_kv, p.kv.head_dim));
    p.rows = rows_dev;
    p.n_lists = p.table.n_seq;
    p.n_rows = static_cast<int32_t>(n_rows);
    p.starts = starts_dev;
    p.ends = ends_dev;
    p.q = q_dev;
    p.q_stride = q_stride;
    p.n_heads = n_heads;
    p.scale = scores->scale;
    p.cap = scores->cap;
    p.slopes = scores->slopes;
    p.pos = scores->pos;
    p.out = out_dev;
    p.out_stride = out_stride;
    p.workspace = workspace_dev;
    LaunchKvRows(p, static_cast<cudaStream_t>(stream));
    return 0;
  }
  RPGB_CATCH(-1)
}

int64_t rpgb_kv_attend_shared_workspace(int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t n_seq) {
  try {
    SetLastError("");
    CheckShape(n_heads, n_kv, head_dim);
    RPGB_CHECK(n_seq >= 0 && n_seq <= (1 << 20), "kv: bad conversation count %d", n_seq);
    return SharedParts(n_heads, n_kv, head_dim, n_seq).total;
  }
  RPGB_CATCH(-1)
}

int32_t rpgb_kv_attend_shared(const rpgb_kv_pages* kv, const rpgb_kv_table* table, int32_t type, const void* q_dev,
                              int64_t q_stride, int32_t n_heads, const int32_t* lens_dev, const int32_t* starts_dev,
                              const int32_t* groups_dev, int32_t n_groups, const int32_t* prefix_dev, float scale,
                              void* out_dev, int64_t out_stride, void* workspace_dev, int64_t workspace_bytes,
                              void* stream) {
  try {
    SetLastError("");
    KvRowsParams p;
    p.kv = Pages(kv);
    p.table = Table(table, p.kv.page_log2);
    p.type = Type(type);
    RPGB_CHECK(n_heads > 0 && n_heads <= 65535 && n_heads % p.kv.n_kv == 0, "kv: %d q heads over %d KV heads", n_heads,
               p.kv.n_kv);
    RPGB_CHECK(n_groups >= 0 && n_groups <= (1 << 20), "kv: bad group count %d", n_groups);
    if (p.table.n_seq == 0 || n_groups == 0) return 0;
    const int64_t cols = static_cast<int64_t>(n_heads) * p.kv.head_dim;
    CheckRows(q_dev, q_stride, cols, p.type, "q");
    CheckRows(out_dev, out_stride, cols, p.type, "out");
    RPGB_CHECK(lens_dev != nullptr && groups_dev != nullptr && prefix_dev != nullptr,
               "kv: lengths, groups or prefixes are NULL");
    CheckAligned(lens_dev, 4, "kv: lengths");
    CheckAligned(starts_dev, 4, "kv: starts");
    CheckAligned(groups_dev, 4, "kv: groups");
    CheckAligned(prefix_dev, 4, "kv: prefixes");
    RPGB_CHECK(std::isfinite(scale), "kv: the scale is not finite");
    const SharedWorkspace w = SharedParts(n_heads, p.kv.n_kv, p.kv.head_dim, p.table.n_seq);
    CheckWorkspace(workspace_dev, workspace_bytes, w.total);
    char* base = static_cast<char*>(workspace_dev);
    // first what follows the common positions, by the operator for one token of each
    KvAttendParams a;
    a.kv = p.kv;
    a.table = p.table;
    a.type = p.type;
    a.lens = lens_dev;
    a.starts = starts_dev;
    a.prefix = prefix_dev;
    a.q = q_dev;
    a.q_stride = q_stride;
    a.n_heads = n_heads;
    a.scale = scale;
    a.out = base + w.own;
    a.out_type = ElemType::kF32;
    a.out_stride = cols;
    a.lse = reinterpret_cast<float*>(base + w.own_lse);
    a.workspace = base + w.attend;
    LaunchKvAttend(a, static_cast<cudaStream_t>(stream));
    // then the common positions, for all of a group at once, and the two together
    p.rows = groups_dev;
    p.n_lists = n_groups;
    p.n_rows = p.table.n_seq;
    p.starts = starts_dev;
    p.ends = lens_dev;
    p.prefix = prefix_dev;
    p.q = q_dev;
    p.q_stride = q_stride;
    p.n_heads = n_heads;
    p.scale = scale;
    p.out = out_dev;
    p.out_stride = out_stride;
    p.own = static_cast<const float*>(a.out);
    p.own_lse = a.lse;
    p.workspace = base + w.rows;
    LaunchKvRows(p, static_cast<cudaStream_t>(stream));
    return 0;
  }
  RPGB_CATCH(-1)
}

int32_t rpgb_sample_rows(int32_t type, const void* logits_dev, int64_t stride, int32_t n_rows, int32_t vocab,
                         const rpgb_sample_rows_options* options, int32_t* tok_out_dev, float* prob_out_dev,
                         void* stream) {
  try {
    SetLastError("");
    SampleRowsParams p;
    RPGB_CHECK(type == RPGB_F32 || type == RPGB_F16 || type == RPGB_BF16, "sample_rows: unknown element type %d", type);
    p.type = static_cast<ElemType>(type);
    RPGB_CHECK(n_rows >= 0 && n_rows <= kKvMaxRows, "sample_rows: bad row count %d", n_rows);
    RPGB_CHECK(vocab > 0 && vocab <= RPGB_SAMPLE_ROWS_MAX_VOCAB, "sample_rows: vocabulary of %d; 1 to %d are taken", vocab,
               RPGB_SAMPLE_ROWS_MAX_VOCAB);
    RPGB_CHECK(stride >= vocab, "sample_rows: stride %lld under the vocabulary's %d", static_cast<long long>(stride),
               vocab);
    RPGB_CHECK(options != nullptr, "sample_rows: options is NULL");
    RPGB_CHECK(options->u != nullptr || options->temperature != nullptr,
               "sample_rows: rows that are not greedy need random numbers");
    for (const void* x : {static_cast<const void*>(options->temperature), static_cast<const void*>(options->top_k),
                          static_cast<const void*>(options->top_p), static_cast<const void*>(options->min_p),
                          static_cast<const void*>(options->u), static_cast<const void*>(tok_out_dev),
                          static_cast<const void*>(prob_out_dev)}) {
      CheckAligned(x, 4, "sample_rows: an array of options or results");
    }
    if (n_rows == 0) return 0;
    RPGB_CHECK(logits_dev != nullptr && tok_out_dev != nullptr, "sample_rows: logits or tokens are NULL");
    CheckAligned(logits_dev, type == RPGB_F32 ? 4 : 2, "sample_rows: logits");
    p.logits = logits_dev;
    p.stride = stride;
    p.n_rows = n_rows;
    p.vocab = vocab;
    p.temperature = options->temperature;
    p.top_k = options->top_k;
    p.top_p = options->top_p;
    p.min_p = options->min_p;
    p.u = options->u;
    p.tok = tok_out_dev;
    p.prob = prob_out_dev;
    LaunchSampleRows(p, static_cast<cudaStream_t>(stream));
    return 0;
  }
  RPGB_CATCH(-1)
}

}  // extern "C"
