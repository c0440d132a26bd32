// Attention over the 8-bit paged KV cache for several query tokens per sequence
// (drafted tokens, short chunks): more (token, query head) columns of a KV head than
// the decode kernel's 8, on the tcgen05 tensor cores.
//
//   S^T (128 keys x N columns)  = K_tile (128 x D) . Q^T (D x N)           [TMEM]
//   O^T (D x N)                += V_tile^T (D x 128) . (s_v P)^T (128 x N)  [TMEM, D/128 MMAs of M=128]
// Scales, masks and softmax as in kv8_attn.cu.  One pass over the codes serves N = 32
// or 64 columns, so drafted tokens cost little more than one.
//
// Bound: shared memory.  A code is read from HBM straight into registers, converted
// to fp16 (exact) and stored once into a 32 KB stage (128 keys x 128 dims, 128-byte
// swizzle), which the MMA reads once: 4 bytes of shared-memory traffic per code, at
// 128 bytes per clock 32 codes per clock and SM, against the SM's share of HBM of 23;
// in practice the converters' issue slots and the waits between tiles.  Five drafted
// tokens of 8 heads (40 columns) over 6 rows of 700 to 9001 int8 keys: 50 us a call with its
// merge (alone and cold 50 and 14), 95 with three blocks of 8 columns per pass of mma.sync.
//
// Warp roles: 8 softmax warps (two per 32 TMEM lanes, thread = key, half of the columns
// each), one MMA warp, three pairs of converter warps.  The pairs take turns: each keeps
// one chunk (of 128 keys x 128 dims) in flight in registers, and together they fill the
// stages in the MMAs' order K(0), K(1), V(0), K(2), V(1), ...; S(u+1) is issued before
// P V(u).  The columns' references (running maxima) lie in shared memory and are only
// renewed when a score of the tile exceeds them by more than kWideStale, which one barrier
// with a vote finds out; a 16 x 32 exchange then gives each lane its column's maximum.
//
// Work split: the list of 128-key tiles (kv8_list.cuh), one equal run per CTA; items
// that span CTAs are joined by kv8_merge_kernel.
//
// Behind a prompt chunk's packed forward the kernel serves the rows with missing pages,
// which that forward cannot mask, and clears the padding (`only`).  As a rule no page is
// missing and its CTAs leave at once: a chunk of 30 to 490 us takes 1 to 3 us longer than
// with a kernel that only clears.
#include <algorithm>

#include "g4_kernels.h"
#include "kv8_list.cuh"

namespace g4 {

namespace {

constexpr int kWideTile = 128;
constexpr int kWideOver = 2;       // entries of the tile list that stand for taking up an item
constexpr int kStageBytes = 32768;
constexpr int kSoft = 8;           // softmax warps
constexpr int kFeeds = 3;          // pairs of converter warps
constexpr int kConvWarps = 2 * kFeeds;
constexpr int kWideThreads = (kSoft + 1 + kConvWarps) * 32;
// s_v P in fp16 relative to O's reference, whose s_v counts as the power of two above
// it: a reference that may lag by 2^9 and a shift of 2^6 keep P below 2^15; its largest
// is at least 2^5, so half a step is at most 2^-11 of a weight, or 2^-30 of the largest
// for weights more than 2^19 below it.  Renewals, which cost as much as the rest of a tile,
// stay rare.  A softmax weight below 2^-126 of the largest is zero before its s_v counts.
constexpr float kWideShift = 6.f;
constexpr float kWideStale = 9.f;
constexpr float kStaleSum = 8.f;   // log2 by which the row sum's reference may lag
constexpr float kNoKey = -1e30f;   // reference before the first visible key: any score exceeds it

template <int kD, int kN, int kStages_, int kPBufs_>
struct WideShape {
  static constexpr int D = kD, N = kN, kStages = kStages_, kPBufs = kPBufs_;
  static constexpr int kOwn = N / 2;                    // columns of a softmax warp
  static constexpr int kParts = kOwn / 16;
  static constexpr int kChunks = D / 128;
  static constexpr int kQBytes = N * D * 2;
  static constexpr int kPBytes = N * kWideTile * 2;
  static constexpr int kTmem = (2 + kChunks) * N <= 128   ? 128
                               : (2 + kChunks) * N <= 256 ? 256
                                                          : 512;
  struct Misc {
    uint64_t full[kStages], empty[kStages];
    uint64_t s_full[2], s_empty[2];
    uint64_t p_full[kPBufs], p_free[kPBufs];
    uint64_t q_ready, drain;
    uint32_t tmem_base;
    int abort;
    // per column: log2(e) * 2^-e of its Q; the reference of its sum; the factor that
    // turns exp2(z - y) s_v into the P of O's reference; what z must not exceed as long
    // as log2 s_v is at most v_ref
    float4 column[N];
    float m_o[N];                   // the reference of O
    float2 scale[N];                // factors on O and the sum after a renewal
    float v_ref[2];                 // per half of the columns
    int last_key[N];                // last visible key, -1: a padded column
    float2 top[kSoft][16];          // maxima over a warp's keys
    float sum[kSoft][kOwn];
    int64_t out_at[N];              // element offset of a column's output row
    int scan[kWideThreads / 32];
  };
  static constexpr int kMisc = (sizeof(Misc) + 15) & ~15;
  static constexpr int smem(int batch) {
    return 1024 + kStages * kStageBytes + kQBytes + kPBufs * kPBytes + kMisc + 4 * (batch + 1);
  }
};

// kind::f16 with fp16 operands, fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool a_mn_major) {
  return (1u << 4) | ((a_mn_major ? 1u : 0u) << 15) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

struct MaxOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct SumOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// v[c] of every lane, reduced over the lanes: lane c (and c + 16) gets column c's
// result.  Each step halves the columns a lane keeps and exchanges the other half.
template <typename Op>
__device__ __forceinline__ float reduce_columns(const float (&v)[16], int lane, Op op) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool up = lane & 8;
    a[i] = op(up ? v[i + 8] : v[i], __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + 8], 8));
  }
#pragma unroll
  for (int w = 4; w > 0; w >>= 1) {
    const bool up = lane & w;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float send = up ? a[i] : a[i + w];
      const float keep = up ? a[i + w] : a[i];
      a[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, w));
    }
  }
  return op(a[0], __shfl_xor_sync(0xffffffffu, a[0], 16));
}

// A CTA's share of its row's padding in a chunk's output: zeros, LSE -inf.
__device__ __forceinline__ void clear_padding(const Kv8AttnParams& p, int d) {
  const int b = blockIdx.x / p.per_row;
  const int heads = p.cache.heads * p.group;
  const Kv8Row row = kv8_row(p.cache, p.rows, b, p.max_k);
  for (int t = row.n + static_cast<int>(blockIdx.x) - b * p.per_row; t < p.rows.tokens;
       t += p.per_row) {
    for (int u = threadIdx.x; u < heads * d / 8; u += blockDim.x) {
      const int h = u / (d / 8);
      *reinterpret_cast<uint4*>(p.o + b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2] +
                                (u % (d / 8)) * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
    for (int h = threadIdx.x; h < heads; h += blockDim.x)
      p.lse[b * p.lse_stride[0] + h * p.lse_stride[1] + t] = -INFINITY;
  }
}

// OR of `pred` over the 128 threads that meet on named barrier `id`.
__device__ __forceinline__ bool bar_red_or(int id, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(pred)), "r"(id)
      : "memory");
  return r != 0;
}

}  // namespace

template <typename Cfg, bool kInt8>
__global__ void __launch_bounds__(kWideThreads, 1) kv8_wide_kernel(const Kv8AttnParams p) {
  constexpr int D = Cfg::D, N = Cfg::N, kChunks = Cfg::kChunks, kStages = Cfg::kStages;
  constexpr int kPBufs = Cfg::kPBufs, kParts = Cfg::kParts, kOwn = Cfg::kOwn;
  using Misc = typename Cfg::Misc;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem;
  uint8_t* q_s = ring + kStages * kStageBytes;
  uint8_t* p_s = q_s + Cfg::kQBytes;
  Misc* misc = reinterpret_cast<Misc*>(p_s + kPBufs * Cfg::kPBytes);
  int* prefix = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(misc) + Cfg::kMisc);

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // provably warp-uniform
  const int lane = tid & 31;
  if (p.only) {
    pdl_enter();
    if (!p.only[blockIdx.x / p.per_row]) {
      clear_padding(p, D);
      return;
    }
  }
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&misc->full[s], 2);
      mbar_init(&misc->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&misc->s_full[b], 1);
      mbar_init(&misc->s_empty[b], kSoft);
    }
    for (int b = 0; b < kPBufs; ++b) {
      mbar_init(&misc->p_full[b], kSoft);
      mbar_init(&misc->p_free[b], 1);
    }
    mbar_init(&misc->q_ready, kSoft);
    mbar_init(&misc->drain, 1);
    misc->abort = 0;
    fence_mbar_init();
  }
  if (warp == kSoft) {
    tmem_alloc(&misc->tmem_base, Cfg::kTmem);
    tmem_relinquish();
  }
  pdl_enter();
  const int heads = p.cache.heads;
  const auto row_at = [&](int b) { return row_plan(p, b); };
  const TileList<kWideTile, N, kWideOver, decltype(row_at)> list{p, row_at, prefix};
  tc_fence_before();
  const int W = blockIdx.x;
  Place pl = {0, 0, 0, 0};
  int todo = 0;
  if (p.whole) {
    const int items = heads * p.col_groups, b = W / items;
    if (W == b * items && tid == 0) kv8_report(p.status, row_at(b).slot);
    __syncthreads();
    pl = list.item_place(b, W - b * items);
    todo = pl.left;
  } else if (p.only) {  // an equal share of the row's items, whole ones
    const int items = heads * p.col_groups, b = W / p.per_row, j = W - b * p.per_row;
    const int first = run_begin(j, p.per_row, items), last = run_begin(j + 1, p.per_row, items);
    const RowPlan r = row_at(b);
    const int act = list.active_items(r);
    __syncthreads();
    pl = list.item_place(b, first);
    todo = (min(last, act) - min(first, act)) * row_tiles(r, kWideTile) +
           (max(last, act) - max(first, act));
  } else {
    plan_rows<kWideThreads>(p, list, prefix, misc->scan, [](int, const RowPlan&) {});
    const int total = prefix[p.rows.batch];
    const int runs = min(total, static_cast<int>(gridDim.x));
    if (W == 0 && tid == 0) *reinterpret_cast<int4*>(p.plan) = make_int4(runs, total, kWideOver, 0);
    if (W < runs) {
      int t0, t1;
      list.locate(run_begin(W + 1, runs, total), t1);
      pl = list.locate(run_begin(W, runs, total), t0);
      todo = t1 - t0;
    }
  }
  tc_fence_after();
  const uint32_t tmem = misc->tmem_base;
  const CtaAbort ab{&misc->abort, nullptr};
  bool ok = true;

  if (warp > kSoft) {
    // ============================ converters ============================
    // thread: rows r0, r0 + 16, ... of the tile, 16 dims `piece` of both 64-dim halves:
    // a quarter-warp stores to two rows whose swizzles differ in the lowest bit, and so
    // hits all banks
    const int feed = (warp - kSoft - 1) >> 1;
    const int ct = (tid - (kSoft + 1) * 32) & 63;
    const int r0 = ct >> 2, piece = ct & 3;
    const uint32_t at0 = r0 * 128 + (((2 * piece) ^ (r0 & 7)) << 4);
    const uint32_t at1 = r0 * 128 + (((2 * piece + 1) ^ (r0 & 7)) << 4);
    // the feed: operands of the run's items in order; this pair takes every third chunk
    int f_todo = todo, f_n = 0, f_k = 0, f_v = 0, f_c = feed + kChunks, f_tile = 0, f_head = 0;
    bool f_is_v = false;
    RowPlan row;
    int f_hi = 0;
    // pool row (page, head, token) of the thread's rows r0 + 16 j in the next chunk's
    // operand; its table entries are requested a chunk earlier.  Rows that no column sees
    // are zeros, whatever the pool holds: they load row 0, and `live` leaves them out.
    int from[8], entry[8];
    uint32_t live = 0, live_next = 0;   // bit j: row r0 + 16 j
    auto next_operand = [&]() {
      if (f_v == f_n) {  // the next item
        if (f_n > 0) {
          pl.tile += f_n;
          pl.left -= f_n;
          if (pl.left == 0) list.next_item(pl);
        }
        f_n = min(pl.left, f_todo);
        f_todo -= f_n;
        f_k = f_v = 0;
        row = row_at(pl.b);
        int cg;
        list.item_head(pl.b, pl.item, f_head, cg);
        f_hi = pl.item < list.active_items(row) ? row.start + row.n : 0;
      }
      f_is_v = !(f_k < f_n && f_k <= f_v + 1);
      f_tile = pl.tile + (f_is_v ? f_v++ : f_k++);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = f_tile * kWideTile + r0 + 16 * j;
        entry[j] = -1;
        if (key < f_hi && key >= row.lo)
          entry[j] = p.cache.tables[static_cast<int64_t>(row.slot) * p.cache.pages_per_slot +
                                    (key >> p.cache.page_shift)];
      }
    };
    uint4 raw[16];
    const uint8_t *pool = nullptr, *pool_next = nullptr;
    int d_head = 0, d_tile = 0;
    auto look_ahead = [&]() {  // the feed's next chunk: its pool and table entries
      for (; f_c >= kChunks; f_c -= kChunks) next_operand();
      pool_next = (f_is_v ? p.cache.v : p.cache.k) + f_c * 128 + piece * 16;
      d_head = f_head;
      d_tile = f_tile;
      f_c += kFeeds;
    };
    auto next_chunk = [&]() {  // from the entries to rows
      pool = pool_next;
      live_next = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = d_tile * kWideTile + r0 + 16 * j;
        const bool ok_page = entry[j] >= 0 && entry[j] < p.cache.num_pages;
        from[j] = ok_page ? (entry[j] * heads + d_head) * p.cache.page + (key & (p.cache.page - 1))
                          : 0;
        live_next |= ok_page ? 1u << j : 0u;
      }
    };
    auto fetch = [&](int j) {  // row block j / 2, half j % 2
      return __ldcs(reinterpret_cast<const uint4*>(
          pool + static_cast<int64_t>(from[j >> 1]) * D + (j & 1) * 64));
    };
    const int chunks = todo * 2 * kChunks;  // of the run; this pair's are feed, feed + 3, ...
    uint32_t stage = feed % kStages, phase = 0;
    if (feed < chunks) {
      look_ahead();
      next_chunk();
      if (feed + kFeeds < chunks) look_ahead();
#pragma unroll
      for (int j = 0; j < 16; ++j) raw[j] = fetch(j);
    }
#pragma unroll 1
    for (int q = feed; q < chunks && ok; q += kFeeds) {
      live = live_next;
      if (q + kFeeds < chunks) next_chunk();  // else the last chunk's rows once more, unused
      if (__any_sync(0xffffffffu, live != 255u)) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (!(live >> (j >> 1) & 1u)) raw[j] = make_uint4(0u, 0u, 0u, 0u);
      }
      if (q + 2 * kFeeds < chunks) look_ahead();
      ok = mbar_wait(&misc->empty[stage], phase ^ 1, ab, kDevTimeoutMma);
      uint8_t* st = ring + stage * kStageBytes;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint4 x = raw[j];
        uint32_t h[8];
        kv8_to_half<kInt8>(x.x, h[0], h[1]);
        kv8_to_half<kInt8>(x.y, h[2], h[3]);
        kv8_to_half<kInt8>(x.z, h[4], h[5]);
        kv8_to_half<kInt8>(x.w, h[6], h[7]);
        uint8_t* dst = st + (j >> 1) * 2048 + (j & 1) * 16384;
        *reinterpret_cast<uint4*>(dst + at0) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + at1) = make_uint4(h[4], h[5], h[6], h[7]);
        raw[j] = fetch(j);  // the pair's next chunk, a chunk's time ahead
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&misc->full[stage]);
      stage += kFeeds;
      if (stage >= kStages) {
        stage -= kStages;
        phase ^= 1;
      }
    }
  } else if (warp == kSoft) {
    // ============================ MMA issuer ============================
    constexpr uint32_t kIdS = idesc_f16(128, N, false);
    constexpr uint32_t kIdO = idesc_f16(128, N, true);
    const uint32_t ring_b = smem_addr(ring), q_b = smem_addr(q_s), p_b = smem_addr(p_s);
    uint32_t stage = 0, phase = 0, tile = 0, seg = 0;  // tile: S issued in the run so far
    uint32_t done = 0;                                 // P V issued in the run so far
    auto take = [&]() {
      ok = ok && mbar_wait(&misc->full[stage], phase, ab, kDevTimeoutPeer);
      tc_fence_after();
      return ok;
    };
    auto release = [&]() {
      umma_commit_w(&misc->empty[stage]);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    };
    auto issue_s = [&]() {
      const uint32_t b = tile & 1;
      ok = ok && mbar_wait(&misc->s_empty[b], ((tile >> 1) & 1) ^ 1, ab, kDevTimeoutPeer);
      tc_fence_after();
      for (int c = 0; c < kChunks && ok; ++c) {
        if (!take()) break;
        const uint32_t kb = ring_b + stage * kStageBytes;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_ss_w(tmem + b * N, sdesc_sw128(kb + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                    sdesc_sw128(q_b + (2 * c + (kk >> 2)) * (N * 128) + (kk & 3) * 32, 16, 1024),
                    kIdS, (c | kk) != 0);
        release();
      }
      umma_commit_w(&misc->s_full[b]);
      ++tile;
    };
    auto issue_o = [&](bool accumulate) {
      const uint32_t b = kPBufs == 2 ? done & 1 : 0;
      const uint32_t par = kPBufs == 2 ? (done >> 1) & 1 : done & 1;
      ok = ok && mbar_wait(&misc->p_full[b], par, ab, kDevTimeoutPeer);
      tc_fence_after();
      for (int c = 0; c < kChunks && ok; ++c) {
        if (!take()) break;
        const uint32_t vb = ring_b + stage * kStageBytes;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_ss_w(tmem + 2 * N + c * N, sdesc_sw128(vb + kk * 2048, 16384, 1024),
                    sdesc_sw128(p_b + b * Cfg::kPBytes + (kk >> 2) * (N * 128) + (kk & 3) * 32, 16,
                                1024),
                    kIdO, accumulate || kk != 0);
        release();
      }
      umma_commit_w(&misc->p_free[b]);
      ++done;
    };
    while (todo > 0 && ok) {
      const int n = min(pl.left, todo);
      ok = mbar_wait(&misc->q_ready, seg & 1, ab, kDevTimeoutPeer);
      tc_fence_after();
      if (ok) issue_s();
      for (int u = 0; u < n && ok; ++u) {
        if (u + 1 < n) issue_s();
        if (ok) issue_o(u > 0);
      }
      todo -= n;
      pl.tile += n;
      pl.left -= n;
      if (pl.left == 0) list.next_item(pl);
      ++seg;
    }
    // every MMA this warp issued has completed before TMEM is freed
    umma_commit_w(&misc->drain);
    mbar_wait(&misc->drain, 0, ab, kDevTimeoutMma);
    __syncwarp();
  } else {
    // ============================ softmax ============================
    // tcgen05.ld/st are .sync.aligned, and warps meet on named barriers: control flow
    // stays uniform, an expired wait only skips the later ones.
    const int quarter = warp & 3, half = warp >> 2;  // TMEM lanes; columns kOwn * half ..
    const int own = half * kOwn;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + own;
    uint32_t tile = 0;  // of the run
    bool from_start = todo > 0 && list.at_start(pl);
    const auto meet = [&]() {  // the four warps of these columns
      asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
    };
    const auto meet_all = [&]() {
      asm volatile("bar.sync 3, %0;" ::"n"(kSoft * 32) : "memory");
    };
    while (todo > 0) {
      const int n = min(pl.left, todo);
      const RowPlan r = row_at(pl.b);
      int head, cg;
      list.item_head(pl.b, pl.item, head, cg);
      {  // ---- Q^T, kPer threads per column ----
        constexpr int kPer = kSoft * 32 / N, kLoads = D / 8 / kPer;
        const int c = tid / kPer, sub = tid % kPer;
        const int col = cg * N + c;
        const int tok = col / p.group, gh = col - tok * p.group;
        const bool have = tok < r.n;
        const uint4* src = reinterpret_cast<const uint4*>(
            p.q + static_cast<int64_t>(pl.b) * p.q_stride[0] +
            static_cast<int64_t>(have ? tok : 0) * p.q_stride[1] +
            static_cast<int64_t>(head * p.group + (have ? gh : 0)) * p.q_stride[2]);
        uint4 x[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          x[i] = have ? src[kPer * i + sub] : make_uint4(0u, 0u, 0u, 0u);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          top = __vmaxu2(__vmaxu2(top, x[i].x & 0x7fff7fffu), x[i].y & 0x7fff7fffu);
          top = __vmaxu2(__vmaxu2(top, x[i].z & 0x7fff7fffu), x[i].w & 0x7fff7fffu);
        }
        top = max(top >> 16, top & 0xffffu);
#pragma unroll
        for (int o = 1; o < kPer; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e = q_exponent(__uint_as_float(top << 16));
        const float f1 = __uint_as_float(static_cast<uint32_t>(127 + e / 2) << 23);
        const float f2 = __uint_as_float(static_cast<uint32_t>(127 + e - e / 2) << 23);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int ch = kPer * i + sub;  // 8 dims
          const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          uint32_t h[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const __half2 v = __floats2half2_rn(__uint_as_float(w[y] << 16) * f1 * f2,
                                                __uint_as_float(w[y] & 0xffff0000u) * f1 * f2);
            h[y] = *reinterpret_cast<const uint32_t*>(&v);
          }
          *reinterpret_cast<uint4*>(q_s + (ch >> 3) * (N * 128) + c * 128 +
                                    (((ch & 7) ^ (c & 7)) << 4)) =
              make_uint4(h[0], h[1], h[2], h[3]);
        }
        if (sub == 0) {
          misc->last_key[c] = have ? r.start + tok : -1;
          misc->column[c] =
              make_float4(kLog2e * __uint_as_float(static_cast<uint32_t>(127 - e) << 23), kNoKey,
                          0.f, kNoKey);
          misc->m_o[c] = kNoKey;
          if (c < 2) misc->v_ref[c] = -200.f;
          misc->out_at[c] = static_cast<int64_t>(pl.b) * p.o_stride[0] +
                            static_cast<int64_t>(tok) * p.o_stride[1] +
                            static_cast<int64_t>(head * p.group + gh) * p.o_stride[2];
        }
        fence_proxy_async_smem();
        meet_all();
        if (lane == 0) mbar_arrive(&misc->q_ready);
      }
      // tiles all of whose keys the group's first to last query see (the padding's columns
      // may see anything: their results are left out at the end)
      const int q0 = r.start + cg * N / p.group, t1 = min(r.n - 1, (cg * N + N - 1) / p.group);
      const int full_lo =
          p.window > 0 ? (max(0, r.start + t1 - p.window + 1) + kWideTile - 1) / kWideTile : 0;
      const int full_hi = (q0 + 1) / kWideTile;
      const int hi = pl.item < list.active_items(r) ? r.start + r.n : 0;
      const int cols = min(N, p.rows.tokens * p.group - cg * N) - own;  // that are written
      // this thread's key of the next tile: its page's scales, requested a tile ahead
      float ks_next = 0.f, vs_next = 0.f;
      bool key_next = false;
      const auto look = [&](int t) {
        const int key = t * kWideTile + quarter * 32 + lane;
        const int page = key < hi && key >= r.lo ? kv8_page(p.cache, r.slot, key) : -1;
        key_next = page >= 0;
        const int64_t block = static_cast<int64_t>(max(page, 0)) * heads + head;
        ks_next = key_next ? p.cache.k_scale[block] : 0.f;
        vs_next = key_next ? p.cache.v_scale[block] : 0.f;
      };
      look(pl.tile);
      float l[kParts][16];
#pragma unroll
      for (int h = 0; h < kParts; ++h)
#pragma unroll
        for (int c = 0; c < 16; ++c) l[h][c] = 0.f;
      for (int u = 0; u < n; ++u, ++tile) {
        const uint32_t b = tile & 1;
        const float ks = ks_next, vs = vs_next;
        const bool key_ok = key_next;
        if (u + 1 < n) look(pl.tile + u + 1);
        const int key = (pl.tile + u) * kWideTile + quarter * 32 + lane;
        const bool full = pl.tile + u >= full_lo && pl.tile + u < full_hi &&
                          __all_sync(0xffffffffu, key_ok);
        const float v_exp =
            static_cast<float>(static_cast<int>((__float_as_uint(vs) >> 23) & 255u) - 126);
        const float vs_up = vs * 64.f;  // 2^kWideShift
        if (ok) ok = mbar_wait(&misc->s_full[b], (tile >> 1) & 1, ab, kDevTimeoutMma);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        float z[kParts][16];
        bool over = key_ok && v_exp > misc->v_ref[half];
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          uint32_t sr[16];
          tmem_ld16(lane_base + b * N + h * 16, sr);
          tmem_wait_ld();
          reg_fence16(sr);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float4 k = misc->column[own + h * 16 + c];
            z[h][c] = __uint_as_float(sr[c]) * (ks * k.x);
            if (full) over |= z[h][c] > k.w;
          }
          if (!full) {
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const int last = misc->last_key[own + h * 16 + c];
              if (!key_ok || key > last || (p.window > 0 && key <= last - p.window))
                z[h][c] = -INFINITY;
              over |= z[h][c] > misc->column[own + h * 16 + c].w;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&misc->s_empty[b]);
        bool any_o = false;
        if (bar_red_or(1 + half, over)) {  // renew the columns' references
          const bool one_exp = __all_sync(0xffffffffu, v_exp == __shfl_sync(0xffffffffu, v_exp, 0));
          float v_ref = key_ok ? v_exp : -200.f;  // the tile's, all lanes and warps
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) v_ref = fmaxf(v_ref, __shfl_xor_sync(0xffffffffu, v_ref, o));
          if (lane == 0) misc->sum[warp][0] = v_ref;
#pragma unroll 1
          for (int h = 0; h < kParts; ++h) {
            float y[16], yv[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              y[c] = kParts == 1 || h == 0 ? z[0][c] : z[kParts - 1][c];
              yv[c] = y[c] + v_exp;
            }
            const float top = reduce_columns(y, lane, MaxOp());
            const float top_v = one_exp ? top + v_exp : reduce_columns(yv, lane, MaxOp());
            if (lane < 16) misc->top[warp][lane] = make_float2(top, top_v);
            meet();
            const int col = own + h * 16 + (lane & 15);
            float2 tm = misc->top[half * 4][lane & 15];
            v_ref = misc->v_ref[half];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float2 x = misc->top[half * 4 + w][lane & 15];
              tm.x = fmaxf(tm.x, x.x);
              tm.y = fmaxf(tm.y, x.y);
              v_ref = fmaxf(v_ref, misc->sum[half * 4 + w][0]);
            }
            const float4 k = misc->column[col];
            const float m_old = misc->m_o[col];
            const float m_l = fmaxf(k.y, tm.x);
            const float m_o = tm.y > m_old + kWideStale ? tm.y : m_old;
            any_o |= __any_sync(0xffffffffu, m_o != m_old);
            meet();
            if (quarter == 0 && lane < 16) {
              misc->column[col] = make_float4(k.x, m_l, m_o == kNoKey ? 0.f : ex2(m_l - m_o),
                                              fminf(m_o + kWideStale - v_ref, m_l + kStaleSum));
              misc->m_o[col] = m_o;
              misc->scale[col] = make_float2(ex2(m_old - m_o), ex2(k.y - m_l));
            }
          }
          if (quarter == 0 && lane == 0) misc->v_ref[half] = v_ref;
          meet();
#pragma unroll
          for (int h = 0; h < kParts; ++h)
#pragma unroll
            for (int c = 0; c < 16; ++c) l[h][c] *= misc->scale[own + h * 16 + c].y;
        }
        // P^T's buffer once the earlier P V that read it is done
        const uint32_t pb = kPBufs == 2 ? b : 0;
        const uint32_t par = kPBufs == 2 ? (tile >> 1) & 1 : tile & 1;
        if (ok) ok = mbar_wait(&misc->p_free[pb], par ^ 1, ab, kDevTimeoutMma);
        ok = __all_sync(0xffffffffu, ok);
        {
          uint8_t* dst = p_s + pb * Cfg::kPBytes + (quarter >> 1) * (N * 128) + own * 128;
          const int kc = ((quarter & 1) * 32 + lane) >> 3, ke = (lane & 7) * 2;
#pragma unroll
          for (int h = 0; h < kParts; ++h)
#pragma unroll
            for (int c0 = 0; c0 < 16; c0 += 8) {  // in batches: the stores hold back later loads
              __half x[8];
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const float4 k = misc->column[own + h * 16 + c0 + c];
                const float t = ex2(z[h][c0 + c] - k.y);
                l[h][c0 + c] += t;
                x[c] = __float2half_rn(t * k.z * vs_up);
              }
#pragma unroll
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<__half*>(dst + (h * 16 + c0 + c) * 128 + ((kc ^ c) << 4) + ke) =
                    x[c];
            }
        }
        if (any_o && u > 0) {  // O^T holds every earlier tile before it is scaled in place
          if (kPBufs == 2) {
            if (ok) ok = mbar_wait(&misc->p_free[b ^ 1], ((tile - 1) >> 1) & 1, ab, kDevTimeoutMma);
            ok = __all_sync(0xffffffffu, ok);
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < kChunks * kParts; ++c) {
            const int at = (c % kParts) * 16;
            uint32_t o[16];
            tmem_ld16(lane_base + 2 * N + (c / kParts) * N + at, o);
            tmem_wait_ld();
            reg_fence16(o);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              o[j] = __float_as_uint(__uint_as_float(o[j]) * misc->scale[own + at + j].x);
            tmem_st16(lane_base + 2 * N + (c / kParts) * N + at, o);
          }
          tmem_wait_st();
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&misc->p_full[pb]);
      }
      // ---- the item's end in this run ----
      {
        const uint32_t last = tile - 1;
        const uint32_t pb = kPBufs == 2 ? last & 1 : 0;
        if (ok) ok = mbar_wait(&misc->p_free[pb], kPBufs == 2 ? (last >> 1) & 1 : last & 1, ab,
                               kDevTimeoutMma);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const float x = reduce_columns(l[h], lane, SumOp());
        if (lane < 16) misc->sum[warp][h * 16 + lane] = x;
      }
      meet();
      todo -= n;
      pl.tile += n;
      pl.left -= n;
      const bool whole = from_start && pl.left == 0;
      const int64_t slot = 2 * static_cast<int64_t>(W) + (pl.left == 0 && todo > 0 ? 0 : 1);
      if (quarter == 0 && lane < kOwn) {
        float sum = (misc->sum[half * 4][lane] + misc->sum[half * 4 + 1][lane]) +
                    (misc->sum[half * 4 + 2][lane] + misc->sum[half * 4 + 3][lane]);
        // without a visible key: references as kv8_merge_kernel expects them
        float m_l = misc->column[own + lane].y, m_o = misc->m_o[own + lane];
        const bool have = misc->last_key[own + lane] >= 0;
        if (!have) sum = 0.f;
        if (!have || m_l == kNoKey) m_l = -INFINITY;
        if (!have || m_o == kNoKey) m_o = -INFINITY;
        m_o += kShiftUp - kWideShift;  // the shift that out_factor and the merge know
        misc->scale[own + lane].x = whole ? out_factor(m_o, m_l, sum) : 1.f;
        if (lane < cols) {
          if (whole) put_lse(p, pl.b, head, cg * N + own + lane, m_l, sum);
          else p.part_ml[slot * N + own + lane] = make_float4(m_o, m_l, sum, 0.f);
        }
      }
      meet();
      const int at_dim = quarter * 32 + lane;
      float* po = p.part_o + (slot * N + own) * D + at_dim;
#pragma unroll 1
      for (int c = 0; c < kChunks * kParts; ++c) {
        const int c0 = (c % kParts) * 16, dim = (c / kParts) * 128;
        if (c0 >= cols) continue;
        uint32_t o[16];
        tmem_ld16(lane_base + 2 * N + (c / kParts) * N + c0, o);
        tmem_wait_ld();
        reg_fence16(o);
        if (whole) {
          __nv_bfloat16* out = p.o + dim + at_dim;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < cols)
              out[misc->out_at[own + c0 + j]] =
                  __float2bfloat16_rn(__uint_as_float(o[j]) * misc->scale[own + c0 + j].x);
        } else {
          float* at = po + c0 * D + dim;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < cols) at[j * D] = __uint_as_float(o[j]);
        }
      }
      tc_fence_before();
      meet_all();  // the columns' data above is rewritten by the next item
      if (pl.left == 0) list.next_item(pl);
      from_start = true;
    }
    if (!ok && lane == 0 && p.status) atomicOr(p.status, kKv8DeviceWait);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kSoft) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kTmem);
  }
}

namespace {

// 32 columns where they suffice: half the Q and P in shared memory, five stages.  At
// 64 columns Q and P leave four, and at head dim 512 (64 KB of Q) one P buffer.
template <int D>
using Wide32 = WideShape<D, 32, 5, 2>;
template <int D>
using Wide64 = WideShape<D, 64, 4, D == 512 ? 1 : 2>;

template <typename Cfg, bool kInt8>
int launch_wide(const Kv8AttnParams& p, int ctas, cudaStream_t stream) {
  static_assert(Cfg::smem(kKv8MaxBatch) <= kKv8MaxSmem, "shared memory of the largest batch");
  const int smem = Cfg::smem(p.rows.batch);
  // a property of the kernel and not of the call: the same from every host thread
  cudaError_t e = cudaFuncSetAttribute(kv8_wide_kernel<Cfg, kInt8>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg::smem(kKv8MaxBatch));
  if (e == cudaSuccess)
    e = launch_chained(kv8_wide_kernel<Cfg, kInt8>, dim3(ctas), dim3(kWideThreads), smem, stream,
                       p);
  return static_cast<int>(e);
}

}  // namespace

Kv8AttnShape kv8_wide_shape(int d, int64_t columns) {
  const int n = columns <= 32 ? 32 : 64;
  return {n, kWideTile, 1, n * d};
}

int launch_kv8_wide(int d, bool int8, const Kv8AttnParams& p, int ctas, cudaStream_t stream) {
  if (p.cols == 32) {
    if (d == 512) return int8 ? launch_wide<Wide32<512>, true>(p, ctas, stream)
                              : launch_wide<Wide32<512>, false>(p, ctas, stream);
    return int8 ? launch_wide<Wide32<256>, true>(p, ctas, stream)
                : launch_wide<Wide32<256>, false>(p, ctas, stream);
  }
  if (d == 512) return int8 ? launch_wide<Wide64<512>, true>(p, ctas, stream)
                            : launch_wide<Wide64<512>, false>(p, ctas, stream);
  return int8 ? launch_wide<Wide64<256>, true>(p, ctas, stream)
              : launch_wide<Wide64<256>, false>(p, ctas, stream);
}

}  // namespace g4
