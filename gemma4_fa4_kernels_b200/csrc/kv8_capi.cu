// C-ABI layer of the 8-bit paged KV cache (include/gemma4_b200.h): argument
// checks, workspace sizes and launches.
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "../../include/gemma4_b200.h"
#include "g4_api.h"
#include "g4_kernels.h"
#include "kv8.h"

namespace {

using namespace g4;

// Makes the call's device current while it launches, and the caller's again after.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    if (device >= 0 && cudaGetDevice(&before_) == cudaSuccess && before_ != device)
      moved_ = cudaSetDevice(device) == cudaSuccess;
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool moved_ = false;
};

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t up256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

int shift_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }
bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

int check_cache(const g4_kv8_args* a) {
  if (!a) return api_fail(G4_ERR_INVALID, "null argument block");
  if (!a->k_pages || !a->v_pages || !a->k_scale || !a->v_scale || !a->tables)
    return api_fail(G4_ERR_INVALID, "k_pages, v_pages, k_scale, v_scale and tables are required");
  if (!al16(a->k_pages) || !al16(a->v_pages))
    return api_fail(G4_ERR_INVALID, "page pools must be 16-byte aligned");
  if (a->k_pages == a->v_pages || a->k_scale == a->v_scale)
    return api_fail(G4_ERR_INVALID, "K and V must be distinct pools");
  if (a->format != G4_KV8_E4M3 && a->format != G4_KV8_INT8)
    return api_fail(G4_ERR_UNSUPPORTED, "codes must be e4m3 or int8");
  if (!page_ok(a->page_size))
    return api_fail(G4_ERR_UNSUPPORTED, "page_size must be 16, 32, 64 or 128");
  if (a->head_dim != 256 && a->head_dim != 512)
    return api_fail(G4_ERR_UNSUPPORTED, "head_dim must be 256 or 512");
  if (a->num_pages <= 0 || a->num_kv_heads <= 0 || a->num_slots <= 0 || a->pages_per_slot <= 0)
    return api_fail(G4_ERR_INVALID, "pages, heads, slots and pages_per_slot must be positive");
  if (a->num_kv_heads > 65535) return api_fail(G4_ERR_UNSUPPORTED, "too many KV heads");
  if (static_cast<int64_t>(a->pages_per_slot) * a->page_size > INT32_MAX - 65536)
    return api_fail(G4_ERR_UNSUPPORTED, "a sequence's positions must fit 31 bits");
  if (static_cast<int64_t>(a->num_pages) * a->num_kv_heads * a->page_size > INT32_MAX)
    return api_fail(G4_ERR_UNSUPPORTED, "a pool's (page, head, token) rows must fit 31 bits");
  if (!a->starts || !a->ends) return api_fail(G4_ERR_INVALID, "starts and ends are required");
  if (a->batch <= 0 || a->tokens <= 0)
    return api_fail(G4_ERR_INVALID, "batch and tokens must be positive");
  if (a->batch > kKv8MaxBatch)
    return api_fail(G4_ERR_UNSUPPORTED, "at most %d rows per call", kKv8MaxBatch);
  if (a->tokens > (1 << 24)) return api_fail(G4_ERR_UNSUPPORTED, "too many tokens per row");
  return G4_OK;
}

int check_operand(const void* p, const int64_t* st, const char* name, bool batch_stride) {
  if (!p) return api_fail(G4_ERR_INVALID, "%s is required", name);
  if (!al16(p)) return api_fail(G4_ERR_INVALID, "%s must be 16-byte aligned", name);
  for (int i = batch_stride ? 0 : 1; i < 3; ++i)
    if (st[i] <= 0 || st[i] % 8)
      return api_fail(G4_ERR_INVALID, "%s strides must be positive multiples of 8 elements", name);
  return G4_OK;
}

Kv8Cache cache_of(const g4_kv8_args* a) {
  Kv8Cache c;
  c.k = static_cast<uint8_t*>(a->k_pages);
  c.v = static_cast<uint8_t*>(a->v_pages);
  c.k_scale = a->k_scale;
  c.v_scale = a->v_scale;
  c.tables = a->tables;
  c.num_pages = a->num_pages;
  c.page = a->page_size;
  c.page_shift = shift_of(a->page_size);
  c.heads = a->num_kv_heads;
  c.num_slots = a->num_slots;
  c.pages_per_slot = a->pages_per_slot;
  return c;
}

Kv8Rows rows_of(const g4_kv8_args* a) {
  Kv8Rows r;
  r.slots = a->slots;
  r.starts = a->starts;
  r.ends = a->ends;
  r.batch = a->batch;
  r.tokens = a->tokens;
  return r;
}

int check_attn_shape(const g4_kv8_args* a) {
  if (a->num_q_heads <= 0 || a->num_q_heads % a->num_kv_heads)
    return api_fail(G4_ERR_INVALID, "query heads must be a positive multiple of KV heads");
  if (int64_t(a->num_q_heads / a->num_kv_heads) * a->tokens > (1 << 30))
    return api_fail(G4_ERR_UNSUPPORTED, "too many (token, query head) columns per KV head");
  if (a->window < 0) return api_fail(G4_ERR_INVALID, "window must be >= 0");
  if (a->max_seqlen_k <= 0 ||
      a->max_seqlen_k > static_cast<int64_t>(a->pages_per_slot) * a->page_size)
    return api_fail(G4_ERR_INVALID, "max_seqlen_k must be in [1, pages_per_slot * page_size]");
  return G4_OK;
}

// A call of at most one item per SM gives each item a CTA when that is at most this many
// tiles per run of the CTA: the tiles take longer there, but no merge follows.  Measured
// for one row (us, whole / equal runs and merge): d512 128 keys 11.1 / 17.3, 300 keys
// 16.7 / 17.1, 400 keys 20.4 / 17.0; d256 300 keys 10.4 / 15.0, 700 keys 15.4 / 15.2,
// 1100 keys 19.7 / 15.7; 32 columns d512 128 keys 13.8 / 16.3, 192 keys 17.1 / 15.4.
constexpr int kWholeTiles = 2;

// Launch shape and workspace of the attention.
struct AttnPlan {
  int64_t tiles = 0;  // upper bound of the tile list
  int cols = 0, tile = 0, col_groups = 0;
  int ctas = 0;
  bool whole = false;
  size_t part_o = 0, part_ml = 0, plan = 0, total = 0;
};

AttnPlan attn_plan(const g4_kv8_args* a) {
  AttnPlan w;
  const int64_t columns = int64_t(a->num_q_heads / a->num_kv_heads) * a->tokens;
  const Kv8AttnShape shape = kv8_attn_shape(a->head_dim, columns);
  w.cols = shape.cols;
  w.tile = shape.tile;
  w.col_groups = static_cast<int>(
      std::min<int64_t>((columns + shape.cols - 1) / shape.cols, INT32_MAX));
  int64_t keys = a->max_seqlen_k;
  if (a->window > 0) keys = std::min<int64_t>(keys, int64_t(a->window) + a->tokens - 1);
  const int64_t per_item = (keys + shape.tile - 1) / shape.tile + 1;
  // capped, so that the product below fits; the call is refused long before
  const int64_t items =
      std::min<int64_t>(int64_t(a->batch) * a->num_kv_heads * w.col_groups, int64_t(1) << 32);
  // (with what the list counts for taking up an item)
  w.tiles = items * (per_item + 2);
  // one CTA per SM; fewer when there is less than a tile per run
  w.ctas = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(api_sm_count(), (w.tiles + shape.runs - 1) / shape.runs)));
  // Few short items: a CTA each, which needs no parts and no merge.
  w.whole = items <= api_sm_count() && per_item <= kWholeTiles * shape.runs;
  if (w.whole) {
    w.ctas = static_cast<int>(items);
    w.total = 256;
    return w;
  }
  const size_t slots = size_t(w.ctas) * shape.runs * 2;
  size_t off = 0;
  w.plan = off;
  off = up256(off + sizeof(int) * (5 * size_t(a->batch) + 4));
  w.part_ml = off;
  off = up256(off + slots * shape.cols * sizeof(float4));
  w.part_o = off;
  off = up256(off + slots * size_t(shape.out_floats) * sizeof(float));
  w.total = off;
  return w;
}

// Operands of an attention launch; its shape is still to be set.
Kv8AttnParams attn_of(const g4_kv8_args* a) {
  Kv8AttnParams p;
  memset(&p, 0, sizeof(p));
  p.cache = cache_of(a);
  p.rows = rows_of(a);
  p.window = a->window;
  p.max_k = a->max_seqlen_k;
  p.group = a->num_q_heads / a->num_kv_heads;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.o = static_cast<__nv_bfloat16*>(a->o);
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = a->q_stride[i];
    p.o_stride[i] = a->o_stride[i];
  }
  p.lse = a->lse;
  p.lse_stride[0] = a->lse_stride[0];
  p.lse_stride[1] = a->lse_stride[1];
  p.status = a->status;
  return p;
}

int check_pages(const g4_pages_args* a) {
  if (!a) return api_fail(G4_ERR_INVALID, "null argument block");
  if (!a->tables || !a->lengths || !a->refcounts || !a->status)
    return api_fail(G4_ERR_INVALID, "tables, lengths, refcounts and status are required");
  if (a->num_layers <= 0 || a->num_pages <= 0 || a->num_kv_heads <= 0 || a->num_slots <= 0 ||
      a->pages_per_slot <= 0)
    return api_fail(G4_ERR_INVALID,
                    "layers, pages, heads, slots and pages_per_slot must be positive");
  if (!page_ok(a->page_size))
    return api_fail(G4_ERR_UNSUPPORTED, "page_size must be 16, 32, 64 or 128");
  if (a->head_dim != 256 && a->head_dim != 512)
    return api_fail(G4_ERR_UNSUPPORTED, "head_dim must be 256 or 512");
  if (a->num_pages > (1 << 26)) return api_fail(G4_ERR_UNSUPPORTED, "at most 2^26 pages");
  if (static_cast<int64_t>(a->pages_per_slot) * a->page_size > INT32_MAX - 65536)
    return api_fail(G4_ERR_UNSUPPORTED, "a sequence's positions must fit 31 bits");
  return G4_OK;
}

int check_pools(const g4_pages_args* a) {
  if (!a->k_pages || !a->v_pages || !a->k_scale || !a->v_scale)
    return api_fail(G4_ERR_INVALID, "k_pages, v_pages, k_scale and v_scale are required");
  if (!al16(a->k_pages) || !al16(a->v_pages))
    return api_fail(G4_ERR_INVALID, "page pools must be 16-byte aligned");
  return G4_OK;
}

int check_batch(const g4_pages_args* a, bool bounded) {
  if (a->batch <= 0) return api_fail(G4_ERR_INVALID, "batch must be positive");
  if (bounded && a->batch > kKv8MaxBatch)
    return api_fail(G4_ERR_UNSUPPORTED, "at most %d rows per call", kKv8MaxBatch);
  return G4_OK;
}

// fork: three ints per row; compact: three lists of pages
size_t pages_work(const g4_pages_args* a) {
  return up256(sizeof(int) * std::max<size_t>(3 * size_t(std::max(a->batch, 0)),
                                              2 + 3 * size_t(std::max(a->num_pages, 0))));
}

int check_work(const g4_pages_args* a, size_t need) {
  if (!a->workspace || !al16(a->workspace) || a->workspace_bytes < need)
    return api_fail(G4_ERR_WORKSPACE, "a 16-byte aligned workspace of %zu bytes is required", need);
  return G4_OK;
}

Kv8PagesParams pages_of(const g4_pages_args* a) {
  Kv8PagesParams p;
  memset(&p, 0, sizeof(p));
  p.tables = a->tables;
  p.lengths = a->lengths;
  p.refcounts = a->refcounts;
  p.status = a->status;
  p.num_pages = a->num_pages;
  p.page = a->page_size;
  p.page_shift = shift_of(a->page_size);
  p.num_slots = a->num_slots;
  p.pages_per_slot = a->pages_per_slot;
  p.k = static_cast<uint8_t*>(a->k_pages);
  p.v = static_cast<uint8_t*>(a->v_pages);
  p.k_scale = a->k_scale;
  p.v_scale = a->v_scale;
  p.layers = a->num_layers;
  p.heads = a->num_kv_heads;
  p.page_bytes = int64_t(a->num_kv_heads) * a->page_size * a->head_dim;
  p.a = a->first;
  p.b = a->second;
  p.counts = a->counts;
  p.starts = a->starts;
  p.ends = a->ends;
  p.batch = a->batch;
  p.window = a->window;
  p.work = static_cast<int*>(a->workspace);
  return p;
}

// CTAs of a copying launch: several per SM to keep loads in flight, fewer when
// there is less to do than that.
int copy_ctas(int64_t work) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(work, api_sm_count() * 8)));
}

int launched(int e, const char* what) {
  return e ? api_cuda_fail(static_cast<cudaError_t>(e), what) : static_cast<int>(G4_OK);
}

}  // namespace

extern "C" {

int g4_kv8_append(const g4_kv8_args* a, void* stream) {
  api_clear_error();
  int rc = check_cache(a);
  if (rc) return rc;
  if ((rc = check_operand(a->k, a->k_stride, "k", true))) return rc;
  if ((rc = check_operand(a->v, a->v_stride, "v", true))) return rc;
  Kv8StoreParams p;
  memset(&p, 0, sizeof(p));
  p.cache = cache_of(a);
  p.rows = rows_of(a);
  p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = a->k_stride[i];
    p.v_stride[i] = a->v_stride[i];
  }
  p.status = a->status;
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchScope ls(kKKv8Append, st);
  return launched(launch_kv8_append(a->head_dim, a->format == G4_KV8_INT8, p, st),
                  "cache append launch");
}

int g4_kv8_read(const g4_kv8_args* a, void* stream) {
  api_clear_error();
  int rc = check_cache(a);
  if (rc) return rc;
  const bool packed = a->out_rows != nullptr;
  if ((rc = check_operand(a->k, a->k_stride, "k", !packed))) return rc;
  if (!a->v || !al16(a->v) || a->k == a->v)
    return api_fail(G4_ERR_INVALID, "v must be a second 16-byte aligned output");
  for (int i = packed ? 1 : 0; i < 3; ++i)
    if (a->v_stride[i] != a->k_stride[i])
      return api_fail(G4_ERR_INVALID, "k and v outputs must have the same strides");
  Kv8StoreParams p;
  memset(&p, 0, sizeof(p));
  p.cache = cache_of(a);
  p.rows = rows_of(a);
  p.k_out = static_cast<__nv_bfloat16*>(a->k);
  p.v_out = static_cast<__nv_bfloat16*>(a->v);
  for (int i = 0; i < 3; ++i) p.out_stride[i] = a->k_stride[i];
  p.out_rows = a->out_rows;
  p.out_total = a->out_total;
  p.holes = a->holes;
  p.status = a->status;
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchScope ls(kKKv8Read, st);
  return launched(launch_kv8_read(a->head_dim, a->format == G4_KV8_INT8, p, st),
                  "cache read launch");
}

size_t g4_kv8_attn_workspace_bytes(const g4_kv8_args* a) {
  if (check_cache(a) || check_attn_shape(a)) {
    api_clear_error();
    return 0;
  }
  const OnDevice guard(a->device);
  return attn_plan(a).total;
}

int g4_kv8_attn(const g4_kv8_args* a, void* stream) {
  api_clear_error();
  int rc = check_cache(a);
  if (rc) return rc;
  if ((rc = check_attn_shape(a))) return rc;
  if ((rc = check_operand(a->q, a->q_stride, "q", true))) return rc;
  if ((rc = check_operand(a->o, a->o_stride, "o", true))) return rc;
  if (!a->lse || a->lse_stride[0] <= 0 || a->lse_stride[1] <= 0)
    return api_fail(G4_ERR_INVALID, "lse with positive strides is required");
  const OnDevice guard(a->device);
  const AttnPlan w = attn_plan(a);
  // list indices stay below 2^31
  if (w.tiles > (int64_t(1) << 30))
    return api_fail(G4_ERR_UNSUPPORTED, "too many (row, head, token, key) tiles in one call");
  if (!a->workspace || !al16(a->workspace) || a->workspace_bytes < w.total)
    return api_fail(G4_ERR_WORKSPACE, "a 16-byte aligned workspace of %zu bytes is required",
                    w.total);
  Kv8AttnParams p = attn_of(a);
  p.cols = w.cols;
  p.tile = w.tile;
  p.col_groups = w.col_groups;
  p.whole = w.whole;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.plan = reinterpret_cast<int*>(ws + w.plan);
  p.part_ml = reinterpret_cast<float4*>(ws + w.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + w.part_o);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    LaunchScope ls(kKKv8Attn, st);
    rc = launch_kv8_attn(a->head_dim, a->format == G4_KV8_INT8, p, w.ctas, st);
    if (rc) return launched(rc, "cache attention launch");
  }
  if (!w.whole) {
    LaunchScope ls(kKKv8Merge, st);
    return launched(launch_kv8_merge(a->head_dim, p, w.ctas, st), "cache attention merge launch");
  }
  return G4_OK;
}

int g4_kv8_chunk_plan(const g4_kv8_args* a, int32_t* cu_q, int32_t* cu_k, int32_t* first,
                      int32_t* last, void* stream) {
  api_clear_error();
  int rc = check_cache(a);
  if (rc) return rc;
  if ((rc = check_attn_shape(a))) return rc;
  if (!cu_q || !cu_k || !first || !last)
    return api_fail(G4_ERR_INVALID, "cu_q, cu_k, first and last are required");
  int64_t keys = a->max_seqlen_k;
  if (a->window > 0) keys = std::min<int64_t>(keys, a->window);
  if (int64_t(a->batch) * (keys - 1 + a->tokens) > INT32_MAX)
    return api_fail(G4_ERR_UNSUPPORTED, "the rows' keys must fit 31 bits");
  if (!a->holes) return api_fail(G4_ERR_INVALID, "holes is required");
  Kv8ChunkParams p;
  memset(&p, 0, sizeof(p));
  p.cache = cache_of(a);
  p.rows = rows_of(a);
  p.window = a->window;
  p.max_k = a->max_seqlen_k;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.first = first;
  p.last = last;
  p.holes = a->holes;
  p.status = a->status;
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchScope ls(kKKv8Chunk, st);
  return launched(launch_kv8_chunk_plan(p, st), "chunk plan launch");
}

int g4_kv8_pad_rows(const g4_kv8_args* a, void* stream) {
  api_clear_error();
  int rc = check_cache(a);
  if (rc) return rc;
  if ((rc = check_attn_shape(a))) return rc;
  if ((rc = check_operand(a->o, a->o_stride, "o", true))) return rc;
  if ((rc = check_operand(a->q, a->q_stride, "q", true))) return rc;
  if (!a->lse || a->lse_stride[0] <= 0 || a->lse_stride[1] <= 0)
    return api_fail(G4_ERR_INVALID, "lse with positive strides is required");
  if (!a->holes) return api_fail(G4_ERR_INVALID, "holes is required");
  const OnDevice guard(a->device);
  Kv8AttnParams p = attn_of(a);
  const int64_t columns = int64_t(p.group) * a->tokens;
  const Kv8AttnShape shape = kv8_wide_shape(a->head_dim, columns);
  p.cols = shape.cols;
  p.tile = shape.tile;
  p.col_groups = static_cast<int>((columns + shape.cols - 1) / shape.cols);
  p.only = a->holes;
  // one wave of CTAs: where no page is missing, more of them only come and go (2048 of
  // them took 18 us)
  const int64_t items = int64_t(a->num_kv_heads) * p.col_groups;
  p.per_row = static_cast<int>(
      std::min(items, std::max<int64_t>(1, api_sm_count() / a->batch)));
  // (a run's operand chunks are counted in 31 bits)
  if ((items / p.per_row + 1) * (a->max_seqlen_k / shape.tile + 2) > (int64_t(1) << 27))
    return api_fail(G4_ERR_UNSUPPORTED, "too many (head, token, key) tiles in one row");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchScope ls(kKKv8Chunk, st);
  return launched(launch_kv8_wide(a->head_dim, a->format == G4_KV8_INT8, p, a->batch * p.per_row,
                                  st),
                  "chunk completion launch");
}

size_t g4_pages_workspace_bytes(const g4_pages_args* a) { return a ? pages_work(a) : 0; }

int g4_pages_extend(const g4_pages_args* a, void* stream) {
  api_clear_error();
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_batch(a, true))) return rc;
  if (!a->first || !a->counts || !a->starts || !a->ends)
    return api_fail(G4_ERR_INVALID, "slots, counts, starts and ends are required");
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchScope ls(kKPagesPlan, st);
  return launched(launch_pages_extend(pages_of(a), st), "page reservation launch");
}

int g4_pages_fork(const g4_pages_args* a, void* stream) {
  api_clear_error();
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_pools(a))) return rc;
  if ((rc = check_batch(a, true))) return rc;
  if (!a->first || !a->second)
    return api_fail(G4_ERR_INVALID, "parents and children are required");
  if ((rc = check_work(a, up256(sizeof(int) * 3 * size_t(a->batch))))) return rc;
  const Kv8PagesParams p = pages_of(a);
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    LaunchScope ls(kKPagesPlan, st);
    rc = launch_pages_fork_plan(p, st);
    if (rc) return launched(rc, "fork plan launch");
  }
  LaunchScope ls(kKPagesApply, st);
  const int64_t units = 2 * int64_t(p.layers) * ((p.page_bytes + 16383) / 16384);
  return launched(launch_pages_fork_apply(p, copy_ctas(p.batch * (1 + units)), st), "fork launch");
}

int g4_pages_free(const g4_pages_args* a, void* stream) {
  api_clear_error();
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_batch(a, true))) return rc;
  if (!a->first) return api_fail(G4_ERR_INVALID, "slots are required");
  if (a->window < 0) return api_fail(G4_ERR_INVALID, "window must be >= 0");
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchScope ls(kKPagesPlan, st);
  return launched(launch_pages_free(pages_of(a), st), "page release launch");
}

int g4_pages_compact(const g4_pages_args* a, void* stream) {
  api_clear_error();
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_pools(a))) return rc;
  if ((rc = check_work(a, up256(sizeof(int) * (2 + 3 * size_t(a->num_pages)))))) return rc;
  const Kv8PagesParams p = pages_of(a);
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    LaunchScope ls(kKPagesPlan, st);
    rc = launch_pages_compact_plan(p, st);
    if (rc) return launched(rc, "compaction plan launch");
  }
  LaunchScope ls(kKPagesApply, st);
  return launched(launch_pages_compact_apply(p, copy_ctas(INT32_MAX), st), "compaction launch");
}

int g4_pages_copy(const g4_pages_args* a, void* stream) {
  api_clear_error();
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_pools(a))) return rc;
  if ((rc = check_batch(a, false))) return rc;
  if (!a->first || !a->second)
    return api_fail(G4_ERR_INVALID, "source and destination pages are required");
  const Kv8PagesParams p = pages_of(a);
  const OnDevice guard(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchScope ls(kKPagesApply, st);
  const int64_t units = 2 * int64_t(p.layers) * ((p.page_bytes + 16383) / 16384);
  return launched(launch_pages_copy(p, copy_ctas(p.batch * units), st), "page copy launch");
}

}  // extern "C"
