// Pages of the 8-bit paged KV cache: reserving (extend), forking, freeing,
// compacting and copying them, with all state on the device, so that a serving
// loop needs no host round trip and can be captured in a CUDA graph.
//
// State: tables [slot][pages_per_slot] (page id or -1), lengths [slot] (tokens),
// refcounts [page] (tables that list it; 0 = free).  A page is allocated by taking
// the lowest free ids in order of the call's rows, so results never depend on
// timing.  Whole pages are shared between forks; the page a sequence still writes
// to is its own (fork copies a partly filled last page), so an append never touches
// another sequence's tokens.  A length may be lowered from outside (rejected drafts):
// the pages behind it stay the slot's; extend fills them before it takes new ones, free
// gives them back.
//
// Bound: the page copies are HBM copies; the rest is latency: one CTA scans the
// refcounts (coalesced, one scan), then every table entry is one independent load
// or atomic.  Rows that cannot be served are left as they were and raise a bit of
// the status word.
#include "g4_kernels.h"
#include "kv8.h"

namespace g4 {

namespace {

constexpr int kPlanThreads = 1024;

// Inclusive scan over the block's 1024 threads; `total` is the last value.  Sums stop at
// kMost, which is more than any pool's pages: 1024 rows may ask for 2^27 each.
constexpr int kMost = 1 << 29;
__device__ __forceinline__ int block_scan(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc = min(inc + up, kMost);
  }
  __syncthreads();  // sums may hold an earlier scan
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int s = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s = min(s + up, kMost);
    }
    sums[lane] = s;
  }
  __syncthreads();
  *total = sums[31];
  return warp > 0 ? min(inc + sums[warp - 1], kMost) : inc;
}

// Each warp owns a run of pages in order, each step of it 32 consecutive ones:
// f(page, free, free pages before it) for every page, in parallel.  Returns the
// number of free pages.  `per_warp` is a multiple of 32.
template <typename F>
__device__ __forceinline__ int for_pages(const int* refcounts, int num_pages, int* sums, F f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_warp = ((num_pages + 31) / 32 + 31) / 32 * 32;
  const int p0 = warp * per_warp, p1 = min(num_pages, p0 + per_warp);
  int count = 0;
  for (int p = p0 + lane; p < p1; p += 32) count += refcounts[p] == 0;
  int total;
  const int inc = block_scan(count, sums, &total);
  int before = __shfl_sync(0xffffffffu, inc - count, 0);
  for (int base = p0; base < p1; base += 32) {
    const int p = base + lane;
    const bool in = p < p1;
    const bool fr = in && refcounts[p] == 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, fr);
    if (in) f(p, fr, before + __popc(mask & ((1u << lane) - 1)));
    before += __popc(mask);
  }
  return total;
}

__device__ __forceinline__ int count_free(const int* refcounts, int num_pages, int* sums) {
  int count = 0;
  for (int p = threadIdx.x; p < num_pages; p += kPlanThreads) count += refcounts[p] == 0;
  int total;
  block_scan(count, sums, &total);
  return total;
}

__device__ __forceinline__ int pages_of(int tokens, int shift) {
  return (tokens + (1 << shift) - 1) >> shift;
}

constexpr int kAhead = 4;  // table entries of a thread in flight

__device__ __forceinline__ void raise(int* status, int bit) { atomicOr(status, bit); }

// One unit of a page copy: 16 KB of codes of one layer's K or V (and, in the first,
// the page's scales).  256 threads.
constexpr int kCopyUnit = 16384;

__device__ __forceinline__ void copy_unit(const Kv8PagesParams& p, int src, int dst, int sub,
                                          int64_t units) {
  const int half = static_cast<int>(sub / units);  // 2 * layer + (0 K, 1 V)
  const int64_t at = (sub - half * units) * kCopyUnit;
  const int64_t layer = half >> 1;
  uint8_t* pool = (half & 1) ? p.v : p.k;
  const uint8_t* s = pool + (layer * p.num_pages + src) * p.page_bytes + at;
  uint8_t* d = pool + (layer * p.num_pages + dst) * p.page_bytes + at;
  const int bytes = static_cast<int>(min(static_cast<int64_t>(kCopyUnit), p.page_bytes - at));
  uint4 r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int o = (static_cast<int>(threadIdx.x) + i * 256) * 16;
    if (o < bytes) r[i] = __ldcs(reinterpret_cast<const uint4*>(s + o));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int o = (static_cast<int>(threadIdx.x) + i * 256) * 16;
    if (o < bytes) __stcs(reinterpret_cast<uint4*>(d + o), r[i]);
  }
  if (at == 0) {
    float* sc = (half & 1) ? p.v_scale : p.k_scale;
    for (int h = threadIdx.x; h < p.heads; h += blockDim.x)
      sc[(layer * p.num_pages + dst) * p.heads + h] = sc[(layer * p.num_pages + src) * p.heads + h];
  }
}

__device__ __forceinline__ int64_t units_per_half(const Kv8PagesParams& p) {
  return (p.page_bytes + kCopyUnit - 1) / kCopyUnit;
}

}  // namespace

// Tables that list a page; 0 for an entry without one.
__device__ __forceinline__ int page_refs(const Kv8PagesParams& p, int page) {
  return page >= 0 && page < p.num_pages ? p.refcounts[page] : 0;
}

// Rows b in order: slot a[b] grows by counts[b] tokens.  starts/ends: the new
// tokens' positions; a row that is not served gets start = end.
__global__ void __launch_bounds__(kPlanThreads) pages_extend_kernel(const Kv8PagesParams p) {
  __shared__ int sums[32];
  __shared__ int slots[kKv8MaxBatch];
  __shared__ int first[kKv8MaxBatch + 1];  // allocations before the row
  __shared__ int have[kKv8MaxBatch];       // pages the row has; -1 not served
  pdl_enter();
  const int b = threadIdx.x;
  int slot = -1, count = 0, len = 0, need = 0, old = 0;  // old: pages the row has
  if (b < p.batch) {
    slot = p.a[b];
    count = p.counts[b];
    slots[b] = slot;
  }
  __syncthreads();
  bool ok = b < p.batch && slot >= 0 && slot < p.num_slots && count >= 0;
  if (ok)
    for (int j = 0; j < b; ++j) ok = ok && slots[j] != slot;
  const int64_t cap = static_cast<int64_t>(p.pages_per_slot) << p.page_shift;
  if (b < p.batch && slot >= 0 && slot < p.num_slots) len = p.lengths[slot];
  ok = ok && len >= 0 && len <= cap;
  if (b < p.batch && !ok) raise(p.status, kKv8BadIndex);
  if (ok) {
    if (static_cast<int64_t>(len) + count > cap) {
      ok = false;
      raise(p.status, kKv8RowFull);
    } else {
      const int* row = p.tables + static_cast<int64_t>(slot) * p.pages_per_slot;
      const int want = pages_of(len + count, p.page_shift);
      old = pages_of(len, p.page_shift);
      // The pages that the new tokens fill: the partly filled last one and, where the length
      // was lowered, those listed behind it, up to the first entry without a page.  (The
      // first step ends the search for a slot whose length was not.)
      const int begin = old;
      bool more = count > 0;
      for (int j0 = begin - ((len & (p.page - 1)) != 0); more && j0 < want; j0 += kAhead) {
        int page[kAhead], refs[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) page[i] = j0 + i < want ? row[j0 + i] : -1;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) refs[i] = page_refs(p, page[i]);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (!more) continue;
          if (refs[i] > 1) ok = false;  // another sequence's page too
          if (j0 + i >= begin) {
            more = refs[i] == 1;
            old += more;
          }
          more = more && ok;
        }
      }
      need = ok ? want - old : 0;
      if (!ok) raise(p.status, kKv8BadIndex);
    }
  }
  int total;
  int inc = block_scan(need, sums, &total);
  const int n_free = total > 0 ? count_free(p.refcounts, p.num_pages, sums) : 0;
  if (total > n_free) {  // not for all: a row that finds too few leaves them to those behind it
    if (b < p.batch) first[b] = need;
    __syncthreads();
    if (b == 0) {
      for (int j = 0, left = n_free; j < p.batch; ++j) {
        const int n = first[j];
        if (n <= left) left -= n; else first[j] = -1;
      }
    }
    __syncthreads();
    if (b < p.batch && first[b] < 0) {
      ok = false;
      need = 0;
      raise(p.status, kKv8PoolExhausted);
    }
    inc = block_scan(need, sums, &total);
  }
  if (b < p.batch) {
    first[b] = inc - need;
    have[b] = ok ? old : -1;
    if (b == p.batch - 1) first[p.batch] = total;
  }
  __syncthreads();
  if (total > 0) {
    for_pages(p.refcounts, p.num_pages, sums, [&](int page, bool fr, int rank) {
      if (!fr || rank >= total) return;
      int lo = 0, hi = p.batch;  // first[lo] <= rank < first[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= rank) lo = mid; else hi = mid;
      }
      if (have[lo] < 0) return;
      p.tables[static_cast<int64_t>(slots[lo]) * p.pages_per_slot + have[lo] + rank - first[lo]] =
          page;
      p.refcounts[page] = 1;
    });
  }
  if (b < p.batch) {
    p.starts[b] = len;
    p.ends[b] = ok ? len + count : len;
    if (ok) p.lengths[slot] = len + count;
  }
}

// Rows b: child b[b] (empty) becomes a copy of parent a[b].  work: [0, B) whole
// pages to share (-1: row not served), [B, 2B) source and [2B, 3B) destination of
// the copied last page (-1: none).
__global__ void __launch_bounds__(kPlanThreads) pages_fork_plan_kernel(const Kv8PagesParams p) {
  __shared__ int sums[32];
  __shared__ int kids[kKv8MaxBatch];
  __shared__ int row_of[kKv8MaxBatch];  // allocation -> row
  pdl_enter();
  const int b = threadIdx.x, B = p.batch;
  int parent = -1, child = -1, len = 0, old = 0;
  if (b < B) {
    parent = p.a[b];
    child = p.b[b];
    kids[b] = child;
  }
  bool ok = b < B && parent >= 0 && parent < p.num_slots && child >= 0 && child < p.num_slots;
  if (ok) {
    len = p.lengths[parent];
    old = p.lengths[child] != 0 || p.tables[static_cast<int64_t>(child) * p.pages_per_slot] >= 0;
  }
  __syncthreads();
  if (ok)
    for (int j = 0; j < b; ++j) ok = ok && kids[j] != child;
  // an occupied child would lose its pages
  ok = ok && old == 0 && len >= 0 &&
       len <= static_cast<int64_t>(p.pages_per_slot) << p.page_shift;
  if (b < B && !ok) raise(p.status, kKv8BadIndex);
  const int whole = len >> p.page_shift;
  int src = -1;
  if (ok && (len & (p.page - 1)) != 0) {
    src = p.tables[static_cast<int64_t>(parent) * p.pages_per_slot + whole];
    if (src < 0 || src >= p.num_pages) {
      ok = false;
      src = -1;
      raise(p.status, kKv8BadIndex);
    }
  }
  const int need = src >= 0;
  int total;
  const int inc = block_scan(need, sums, &total);
  const int n_free = total > 0 ? count_free(p.refcounts, p.num_pages, sums) : 0;
  if (need && inc > n_free) {
    ok = false;
    raise(p.status, kKv8PoolExhausted);
  }
  if (need) row_of[inc - 1] = b;
  if (b < B) {
    p.work[b] = ok ? whole : -1;
    p.work[B + b] = ok ? src : -1;
    p.work[2 * B + b] = -1;
    if (ok) p.lengths[child] = len;
  }
  __syncthreads();
  if (total > 0) {
    for_pages(p.refcounts, p.num_pages, sums, [&](int page, bool fr, int rank) {
      if (!fr || rank >= total) return;
      const int row = row_of[rank];
      if (p.work[row] < 0) return;
      p.work[2 * B + row] = page;
      p.refcounts[page] = 1;
      p.tables[static_cast<int64_t>(kids[row]) * p.pages_per_slot + p.work[row]] = page;
    });
  }
}

// The shared pages of every row, then the last pages' copies.
__global__ void __launch_bounds__(256) pages_fork_apply_kernel(const Kv8PagesParams p) {
  pdl_enter();
  const int B = p.batch;
  const int64_t units = units_per_half(p);
  const int64_t per_page = units * 2 * p.layers;
  const int64_t n = B * (1 + per_page);
  for (int64_t u = blockIdx.x; u < n; u += gridDim.x) {
    if (u < B) {
      const int b = static_cast<int>(u);
      const int whole = p.work[b];
      const int* from = p.tables + static_cast<int64_t>(p.a[b]) * p.pages_per_slot;
      int* to = p.tables + static_cast<int64_t>(p.b[b]) * p.pages_per_slot;
      for (int j = threadIdx.x; j < whole; j += blockDim.x) {
        const int page = from[j];
        to[j] = page;
        if (page >= 0 && page < p.num_pages) atomicAdd(&p.refcounts[page], 1);
      }
    } else {
      const int b = static_cast<int>((u - B) / per_page);
      const int dst = p.work[2 * B + b];
      if (dst >= 0)
        copy_unit(p, p.work[B + b], dst, static_cast<int>((u - B) - b * per_page), units);
    }
  }
}

// Row b: slot a[b] gives its pages back.  window 0: all that its table lists, the row is
// empty afterwards; window W: the leading pages that neither the next token at position
// `length` nor any later one sees (keys > position - W); the row keeps its length.
// An entry is taken by an atomic exchange, so a slot listed twice frees once.
constexpr int kFreeThreads = 256;
__global__ void __launch_bounds__(kFreeThreads) pages_free_kernel(const Kv8PagesParams p) {
  pdl_enter();
  const int slot = p.a[blockIdx.x];
  if (slot < 0 || slot >= p.num_slots) {
    if (threadIdx.x == 0) raise(p.status, kKv8BadIndex);
    return;
  }
  int upto = p.pages_per_slot;
  if (p.window > 0) {
    const int len = p.lengths[slot];
    upto = min(min(upto, pages_of(max(len, 0), p.page_shift)),
               max(0, len - p.window + 1) >> p.page_shift);
  }
  int* row = p.tables + static_cast<int64_t>(slot) * p.pages_per_slot;
  for (int j0 = threadIdx.x; j0 < upto; j0 += kAhead * kFreeThreads) {
    int page[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = j0 + i * kFreeThreads;
      page[i] = j < upto ? row[j] : -1;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (page[i] == -1) continue;
      page[i] = atomicExch(&row[j0 + i * kFreeThreads], -1);
      if (page[i] >= 0 && page[i] < p.num_pages) atomicSub(&p.refcounts[page[i]], 1);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && p.window == 0) p.lengths[slot] = 0;
}

// Live pages at or above n_live (their number) move into the holes below it, both
// ascending: the fewest moves, and no page is both read and written.
// work: [0] moves, [1] n_live, [2, 2 + P) sources, [2 + P, 2 + 2P) destinations,
// [2 + 2P, 2 + 3P) the new id of a moved page.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const Kv8PagesParams p) {
  __shared__ int sums[32];
  pdl_enter();
  const int P = p.num_pages;
  const int n_live = P - count_free(p.refcounts, P, sums);
  int below = 0;  // holes
  for (int i = threadIdx.x; i < n_live; i += kPlanThreads) below += p.refcounts[i] == 0;
  int holes;
  block_scan(below, sums, &holes);
  int* src = p.work + 2;
  int* dst = src + P;
  int* moved = dst + P;
  for_pages(p.refcounts, P, sums, [&](int page, bool fr, int rank) {
    if (page < n_live) {
      if (fr) dst[rank] = page;
    } else if (!fr) {
      src[(page - rank) - (n_live - holes)] = page;  // live pages before it, less those kept
    }
  });
  __syncthreads();
  for (int k = threadIdx.x; k < holes; k += kPlanThreads) {
    const int s = src[k], d = dst[k];
    moved[s] = d;
    p.refcounts[d] = p.refcounts[s];
    p.refcounts[s] = 0;
  }
  if (threadIdx.x == 0) {
    p.work[0] = holes;
    p.work[1] = n_live;
  }
}

__global__ void __launch_bounds__(256) pages_compact_apply_kernel(const Kv8PagesParams p) {
  pdl_enter();
  const int moves = p.work[0], n_live = p.work[1], P = p.num_pages;
  if (moves == 0) return;
  const int* src = p.work + 2;
  const int* dst = src + P;
  const int* moved = dst + P;
  const int64_t entries = static_cast<int64_t>(p.num_slots) * p.pages_per_slot;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < entries;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int page = p.tables[i];
    if (page >= n_live && page < P) p.tables[i] = moved[page];
  }
  const int64_t units = units_per_half(p);
  const int64_t per_page = units * 2 * p.layers;
  for (int64_t u = blockIdx.x; u < moves * per_page; u += gridDim.x) {
    const int k = static_cast<int>(u / per_page);
    copy_unit(p, src[k], dst[k], static_cast<int>(u - k * per_page), units);
  }
}

// Pair i: page a[i] to page b[i], all layers, K and V and their scales.  A pair is
// left out (status bit) when an id is out of range, when an earlier pair has the
// same destination, or when its destination is any pair's source.  Every CTA checks the
// pairs that it copies against all of them, without a workspace or a second launch: the
// checks grow with the square of the pairs.  Copies (us, with the floor of their bytes): 200
// pages of 256 KB in ten layers 173 / 160, 4096 pages of 8 KB 46 / 10, 16384 of them 475 / 41.
__global__ void __launch_bounds__(256) pages_copy_kernel(const Kv8PagesParams p) {
  pdl_enter();
  const int64_t units = units_per_half(p);
  const int64_t per_page = units * 2 * p.layers;
  int checked = -1;
  bool ok = false;
  for (int64_t u = blockIdx.x; u < p.batch * per_page; u += gridDim.x) {
    const int k = static_cast<int>(u / per_page);
    const int src = p.a[k], dst = p.b[k];
    if (k != checked) {
      int bad = src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages;
      for (int j = threadIdx.x; j < p.batch; j += blockDim.x)
        bad |= p.a[j] == dst || (j < k && p.b[j] == dst);
      ok = !__syncthreads_or(bad);
      checked = k;
      if (!ok && threadIdx.x == 0) raise(p.status, kKv8BadIndex);
    }
    if (ok) copy_unit(p, src, dst, static_cast<int>(u - k * per_page), units);
  }
}

int launch_pages_extend(const Kv8PagesParams& p, cudaStream_t st) {
  return static_cast<int>(
      launch_chained(pages_extend_kernel, dim3(1), dim3(kPlanThreads), 0, st, p));
}
int launch_pages_fork_plan(const Kv8PagesParams& p, cudaStream_t st) {
  return static_cast<int>(
      launch_chained(pages_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p));
}
int launch_pages_fork_apply(const Kv8PagesParams& p, int ctas, cudaStream_t st) {
  return static_cast<int>(
      launch_chained(pages_fork_apply_kernel, dim3(ctas), dim3(256), 0, st, p));
}
int launch_pages_free(const Kv8PagesParams& p, cudaStream_t st) {
  return static_cast<int>(
      launch_chained(pages_free_kernel, dim3(p.batch), dim3(kFreeThreads), 0, st, p));
}
int launch_pages_compact_plan(const Kv8PagesParams& p, cudaStream_t st) {
  return static_cast<int>(
      launch_chained(pages_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p));
}
int launch_pages_compact_apply(const Kv8PagesParams& p, int ctas, cudaStream_t st) {
  return static_cast<int>(
      launch_chained(pages_compact_apply_kernel, dim3(ctas), dim3(256), 0, st, p));
}
int launch_pages_copy(const Kv8PagesParams& p, int ctas, cudaStream_t st) {
  return static_cast<int>(launch_chained(pages_copy_kernel, dim3(ctas), dim3(256), 0, st, p));
}

}  // namespace g4
