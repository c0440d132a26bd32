// The 8-bit paged KV cache shared by its kernels (kv8_attn.cu, kv8_store.cu):
// device view of one layer, rows of a call, and the codes' conversions.
//
// Keys and values of one layer live in pages of `page` tokens, each page
// [kv head][token][head_dim] codes of 8 bits (e4m3 or int8); a block is one page
// of one head and has one fp32 scale, value = code * scale.  The append writes
// scales that are powers of two: a block whose scale has to grow when later
// tokens join it then shifts its older codes exactly (up to the codes that fall
// below the smallest step), quantising is an exact multiplication and one
// rounding, and e4m3 codes lose nothing to the coarser choice (their relative
// step does not depend on the scale).
//
// A table row lists the pages of one sequence in order, -1 where there is none.
// Rows, page ids and positions that the device arrays carry are checked where
// they are used: an out-of-range page is never read or written (its keys count
// as masked), and a row whose slot or positions are out of range counts as empty and is
// reported.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace g4 {

constexpr int kKv8MaxBatch = 1024;  // rows of one call (their plan sits in shared memory)
constexpr int kKv8MaxSmem = 232448; // dynamic shared memory per CTA
constexpr int kKv8Tile = 32;        // keys per attention tile: two pieces of 16, each in one page
// Exponents of a block's scale 2^e: 2^e and 2^-e are both normal fp32 values, and every
// code * scale is finite in fp32 and bf16.  The largest bf16 value is 255 * 2^120 or
// 127.5 * 2^121: at the largest exponent codes stop at 240 (e4m3, whose next one is 256)
// and 127 (int8), off by at most 2^-4 of the value and half a step, as everywhere.
constexpr int kKv8MinExp = -100;
template <bool kInt8>
constexpr int kKv8MaxExp = kInt8 ? 121 : 120;

enum Kv8Status : int {
  kKv8PoolExhausted = 1,    // no free page left for a row
  kKv8RowFull = 2,          // a row's table is full
  kKv8BadIndex = 4,         // slot, page or count out of range, or the same one twice
  kKv8DeviceWait = 8,       // a bounded wait expired: the call's results are invalid
};

struct Kv8Cache {
  uint8_t* k;               // [page][head][token][head_dim]
  uint8_t* v;
  float* k_scale;           // [page][head]
  float* v_scale;
  const int* tables;        // [slot][pages_per_slot]
  int num_pages;
  int page;                 // tokens per page: 16, 32, 64 or 128
  int page_shift;
  int heads;
  int num_slots;
  int pages_per_slot;
};

struct Kv8Rows {
  const int* slots;         // nullable: row b uses slot b
  const int* starts;        // position of the row's first token
  const int* ends;          // one past its last
  int batch;
  int tokens;               // tokens (queries) per row in the operand; a row uses the first
                            // min(end - start, tokens), the rest is padding
};

struct Kv8Row {
  int slot;                 // -1: asks for nothing, kKv8BadRow: for what is out of range
  int start;
  int n;                    // tokens of the row, <= rows.tokens
};

constexpr int kKv8BadRow = -2;

// Checked row b: empty (n 0) when its slot or positions are out of range.
__device__ __forceinline__ Kv8Row kv8_row(const Kv8Cache& c, const Kv8Rows& r, int b, int max_end) {
  Kv8Row o;
  const int slot = r.slots ? r.slots[b] : b;
  const int start = r.starts[b], end = r.ends[b];
  const bool ok = slot >= 0 && slot < c.num_slots && start >= 0 && end > start && end <= max_end &&
                  (end - 1) >> c.page_shift < c.pages_per_slot;
  o.slot = ok ? slot : end > start ? kKv8BadRow : -1;
  o.start = ok ? start : 0;
  o.n = ok ? min(end - start, r.tokens) : 0;
  return o;
}

// Reports a row of a call (one thread of the launch).
__device__ __forceinline__ void kv8_report(int* status, int slot) {
  if (slot == kKv8BadRow && status) atomicOr(status, kKv8BadIndex);
}

// Page of a position; -1 when there is none.
__device__ __forceinline__ int kv8_page(const Kv8Cache& c, int slot, int pos) {
  const int id = c.tables[static_cast<int64_t>(slot) * c.pages_per_slot + (pos >> c.page_shift)];
  return id >= 0 && id < c.num_pages ? id : -1;
}

// Four codes (one word, byte i = element i) to fp16 pairs (0, 1) and (2, 3).  Both
// formats fit fp16 exactly (e4m3: 4 significant bits from 2^-9 to 448; int8: 7).
template <bool kInt8>
__device__ __forceinline__ void kv8_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kInt8) {
    // byte b + 128 in the low mantissa bits of 1024 gives 1024 + 128 + b
    const uint32_t x = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140);
    const uint32_t b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// ---- attention (kv8_attn.cu) ----
struct Kv8AttnParams {
  Kv8Cache cache;
  Kv8Rows rows;
  int window;               // 0: every earlier key
  int max_k;                // rows that end past it count as empty
  int group;                // query heads per KV head
  int cols;                 // (token, query head) columns of one item (Kv8AttnShape)
  int tile;                 // keys per tile of the list
  int col_groups;           // ceil(tokens * group / cols)
  bool whole;               // one CTA per item instead of equal runs: nothing to merge
  const int* only;          // nullable: the rows whose flag is set, `per_row` CTAs each; the
                            // other rows' padding is cleared
  int per_row;
  const __nv_bfloat16* q;   // (batch, token, head) strides in elements
  int64_t q_stride[3];
  __nv_bfloat16* o;
  int64_t o_stride[3];
  float* lse;               // (batch, head) strides; token stride 1
  int64_t lse_stride[2];
  // partial results (workspace): two per run, [run][head, tail]
  float* part_o;            // [slot][cols][head_dim]
  float4* part_ml;          // [slot][cols]: (shift of O, max, sum, -)
  int* status;              // nullable
  int* plan;                // (not used if whole) {runs, entries, kOver, -}, the rows' plans (int4 each), their first tiles
};
// The kernel's launch shape for a row's number of (token, query head) columns.
struct Kv8AttnShape {
  int cols;                 // columns one pass over the codes serves
  int tile;                 // keys per tile
  int runs;                 // runs per CTA
  int out_floats;           // floats of a partial O
};
Kv8AttnShape kv8_attn_shape(int d, int64_t columns);
Kv8AttnShape kv8_wide_shape(int d, int64_t columns);  // kv8_wide.cu
int launch_kv8_attn(int d, bool int8, const Kv8AttnParams& p, int ctas, cudaStream_t stream);
int launch_kv8_wide(int d, bool int8, const Kv8AttnParams& p, int ctas, cudaStream_t stream);
int launch_kv8_merge(int d, const Kv8AttnParams& p, int ctas, cudaStream_t stream);

// ---- append, read back, chunks of prompts (kv8_store.cu) ----
struct Kv8StoreParams {
  Kv8Cache cache;
  Kv8Rows rows;
  const __nv_bfloat16* k;   // append: (batch, token, head) strides in elements
  const __nv_bfloat16* v;
  int64_t k_stride[3];
  int64_t v_stride[3];
  __nv_bfloat16* k_out;     // read: same strides for both
  __nv_bfloat16* v_out;
  int64_t out_stride[3];
  const int* out_rows;      // read, nullable: rows packed, row b at [out_rows[b], out_rows[b+1])
  int out_total;            // packed: rows of the output
  int* holes;               // read, nullable: [b] = 1 where a position of row b has no page
  int* status;              // nullable
};
int launch_kv8_append(int d, bool int8, const Kv8StoreParams& p, cudaStream_t stream);
int launch_kv8_read(int d, bool int8, const Kv8StoreParams& p, cudaStream_t stream);

struct Kv8ChunkParams {
  Kv8Cache cache;
  Kv8Rows rows;
  int window;
  int max_k;
  int* cu_q;                // [batch + 1]
  int* cu_k;                // [batch + 1]
  int* first;               // [batch] first key read
  int* last;                // [batch] one past the last key read
  int* holes;               // [batch] cleared
  int* status;              // nullable
};
int launch_kv8_chunk_plan(const Kv8ChunkParams& p, cudaStream_t stream);

// ---- pages (kv8_pages.cu) ----
struct Kv8PagesParams {
  int* tables;
  int* lengths;
  int* refcounts;
  int* status;
  int num_pages, page, page_shift, num_slots, pages_per_slot;
  // the pools of all layers, as bytes
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int layers, heads;
  int64_t page_bytes;       // heads * page * head_dim
  const int* a;             // slots, parents or source pages
  const int* b;             // children or destination pages
  const int* counts;
  int* starts;
  int* ends;
  int batch;
  int window;               // free: 0 everything, > 0 only what a window no longer reaches
  int* work;                // workspace
};
int launch_pages_extend(const Kv8PagesParams& p, cudaStream_t stream);
int launch_pages_fork_plan(const Kv8PagesParams& p, cudaStream_t stream);
int launch_pages_fork_apply(const Kv8PagesParams& p, int ctas, cudaStream_t stream);
int launch_pages_free(const Kv8PagesParams& p, cudaStream_t stream);
int launch_pages_compact_plan(const Kv8PagesParams& p, cudaStream_t stream);
int launch_pages_compact_apply(const Kv8PagesParams& p, int ctas, cudaStream_t stream);
int launch_pages_copy(const Kv8PagesParams& p, int ctas, cudaStream_t stream);

}  // namespace g4
