// Attention over the 8-bit paged KV cache for sm_100a: up to 8 (query token, query
// head) columns per KV head and sequence (decode), any batch of ragged lengths.  More
// columns: kv8_wide.cu.
//
//   S = Q K^T,  P = softmax(S masked),  O = P V,  K = s_k * k8,  V = s_v * v8
// with s_k, s_v one scale per (page, KV head).  The scales stay outside the
// products: S = s_k (Q k8^T), and P V = sum over tiles of (s_v P) v8.
//
// Bound: the cache bytes (2 D per key and KV head).  What the SM has to do per
// byte is converting codes to fp16 and feeding them to the tensor core, so each
// code is loaded into registers once for all the query heads that share it:
//   S^T (16 keys x 8 columns)  = K_tile (16 x D) . Q^T (D x 8)
//   O^T (D x 8 columns)       += V_tile^T (D x 16) . P^T (16 x 8)
// with mma.sync m16n8k16 (fp16 in, fp32 out).  A column is one (token, query
// head) of the KV head's group.  The warp-level MMA takes its A operand from
// registers, where the conversion leaves it; the fp16 codes never go back to
// shared memory, which a tcgen05 operand would need (3 times the shared-memory
// traffic per byte read for 8 of at least 16 useful columns).
//
// Work split: every (sequence, KV head, column group) is an item of n 32-key
// tiles; all items' tiles form one list, cut into equal runs, one per team, so
// ragged batches load every SM alike whatever the lengths are.  A team is kTeam
// warps that hold kDims = D / kTeam dims each, of Q, K, V and O: their partial S
// meet in shared memory (one named barrier per tile), everything else of a warp is
// its own: it streams its dims of the run's K and V through its own ring of padded
// shared-memory buffers (cp.async, 16 keys each).  An item that lies in one run is
// written at once; the ends of the CTA's runs that belong to one item are summed
// in shared memory; what then still spans CTAs goes to the workspace and
// kv8_merge_kernel adds it up (in a fixed order: results do not depend on timing).
//
// Fragments: the dims of a K chunk and the dims and keys of a V chunk may be dealt
// to the MMA's indices in any order as long as both operands agree.  K: thread
// (g, t) = (lane / 4, lane % 4) takes 16-byte chunks of key rows g and g + 8; each
// word of a chunk is two k-pairs of one MMA.  V: it takes the same 16-byte chunk of
// keys t, t + 4, t + 8, t + 12; a byte permute pairs two keys' codes of one dim
// before the conversion.  Rows are padded by 16 bytes, and the chunk orders below
// make every quarter-warp of 16-byte loads hit 32 different banks.
//
// Numerics: S, both running maxima, sums and O are fp32.  Q is multiplied by a
// power of two per column so that its largest element lies in [2^13, 2^14), then
// held in fp16: exact down to elements 2^27 below the largest.  s_v P is held in
// fp16 relative to its running maximum, which may lag by 2^3, and shifted up by
// 2^11: below 2^15, rounded by at most 2^-11 of itself, or, for weights more than
// 2^25 below the largest, by 2^-36 of the largest.  The output's rounding to bf16
// is at most 2^-8 of it.
#include <algorithm>

#include "g4_kernels.h"
#include "kv8_list.cuh"

namespace g4 {

namespace {

constexpr int kOver = 1;  // entries of the tile list that stand for taking up an item

// A launch shape: kTeam warps share a run; one pass over the codes serves 8 columns.
template <int kD, int kTeam_, int kWarps_, int kBufs_>
struct AttnShape {
  static constexpr int D = kD, kTeam = kTeam_, kWarps = kWarps_;
  static constexpr int kTeams = kWarps / kTeam;        // runs per CTA
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCols = 8;
  static constexpr int kDims = D / kTeam;              // dims per warp
  static constexpr int kRow = kDims + 16;              // bytes per key row in a buffer
  static constexpr int kBuf = 16 * kRow;
  static constexpr int kBufs = kBufs_;                 // 16-key K or V pieces in flight per warp
  static constexpr int kRing = kBufs * kBuf;
  static constexpr int kChunks = kDims / 64;           // K chunks per thread and row
  static constexpr int kSteps = kDims / 128;           // V chunks per thread and key
  static constexpr int kTilesM = kDims / 16;           // MMAs over a warp's dims
  static constexpr int kOut = D * kCols;               // floats of a partial O
  static constexpr int kOutRow = D + 4;                // and of its columns in shared memory
  static constexpr int kRingBytes = kWarps * kRing;
  static constexpr int kSwaps = kTeam > 1 ? 2 : 1;     // copies of the S buffers
  static constexpr int kExchange = kWarps * kSwaps * 1024;
  static constexpr int kStats = kTeams * kCols * 16;
  static constexpr int kTails = kTeams * 4 * 4;
  static_assert(kRingBytes >= kTeams * kCols * kOutRow * 4, "the runs' ends are summed in the ring's place");
  static constexpr int smem(int batch) {
    return kRingBytes + kExchange + kStats + ((kTails + 15) & ~15) + 16 * batch + 4 * (batch + 1) +
           4 * kWarps;
  }
};

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 (4) bytes global -> shared; the _z form writes zeros where `bytes` is 0.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_z(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp4_z(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

// 16-byte chunk of a V row (of the warp's dims) that thread row g takes in step i.
__device__ __forceinline__ int v_chunk(int g, int i) { return (g & 1) * 4 + (g >> 1) + 8 * i; }

}  // namespace

template <typename Cfg, bool kInt8>
__global__ void __launch_bounds__(Cfg::kThreads, 1) kv8_attn_kernel(const Kv8AttnParams p) {
  constexpr int D = Cfg::D, kTeam = Cfg::kTeam, kCols = Cfg::kCols;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int team = warp / kTeam, part = warp % kTeam;  // part: which dims
  uint8_t* ring = smem + warp * Cfg::kRing;
  float* exchange = reinterpret_cast<float*>(smem + Cfg::kRingBytes);
  float4* stats = reinterpret_cast<float4*>(smem + Cfg::kRingBytes + Cfg::kExchange);  // [team][col]
  int* tails = reinterpret_cast<int*>(stats + Cfg::kTeams * kCols);  // [4][team]
  RowPlan* rows = reinterpret_cast<RowPlan*>(reinterpret_cast<uint8_t*>(tails) +
                                             ((Cfg::kTails + 15) & ~15));
  int* prefix = reinterpret_cast<int*>(rows + p.rows.batch);
  int* scan = prefix + p.rows.batch + 1;

  pdl_enter();
  const int B = p.rows.batch, heads = p.cache.heads;
  const auto row_at = [&](int b) { return rows[b]; };
  const TileList<kKv8Tile, kCols, kOver, decltype(row_at)> list{p, row_at, prefix};
  const int W = blockIdx.x * Cfg::kTeams + team;
  Place first = {0, 0, 0, 0};
  int todo = 0;
  if (p.whole) {  // the CTA's item, cut into a run per team
    const int items = heads * p.col_groups, b = blockIdx.x / items;
    if (tid == 0) {
      rows[b] = row_plan(p, b);
      if (blockIdx.x == b * items) kv8_report(p.status, rows[b].slot);
    }
    __syncthreads();
    first = list.item_place(b, blockIdx.x - b * items);
    const int runs = min(first.left, Cfg::kTeams);
    if (team < runs) {
      const int at = run_begin(team, runs, first.left);
      todo = run_begin(team + 1, runs, first.left) - at;
      first.tile += at;
      first.left -= at;
    }
  } else {
    plan_rows<Cfg::kThreads>(p, list, prefix, scan, [&](int b, const RowPlan& r) { rows[b] = r; });
    const int total = prefix[B];
    const int runs = min(total, static_cast<int>(gridDim.x) * Cfg::kTeams);
    if (blockIdx.x == 0 && tid == 0)
      *reinterpret_cast<int4*>(p.plan) = make_int4(runs, total, kOver, 0);
    if (W < runs) {
      int t0, t1;
      list.locate(run_begin(W + 1, runs, total), t1);
      first = list.locate(run_begin(W, runs, total), t0);
      todo = t1 - t0;
    }
  }

  // ---- the loading side: 16-key pieces in order K0a K0b V0a V0b K1a ... ----
  Place ld = first;
  int ld_todo = todo;        // tiles not yet requested
  uint32_t ld_buf = 0;       // ring offset of the next request
  int ld_phase = 0;          // 0, 1: K halves; 2, 3: V halves
  int ld_page[2], ld_next[2];
  int ld_head = 0, ld_lo = 0, ld_hi = 0, ld_slot = -1;
  // Page of the 16 keys at `pos`; -1 when no column of the row sees any of them.
  auto lookup = [&](int pos) {
    return pos < ld_hi && pos + 16 > ld_lo ? kv8_page(p.cache, ld_slot, pos) : -1;
  };
  auto set_item = [&]() {
    int cg;
    list.item_head(ld.b, ld.item, ld_head, cg);
    const RowPlan r = rows[ld.b];
    const bool act = ld.item < list.active_items(r);
    ld_slot = r.slot;
    ld_lo = r.lo;
    ld_hi = act ? r.start + r.n : 0;
    ld_page[0] = lookup(ld.tile * kKv8Tile);
    ld_page[1] = lookup(ld.tile * kKv8Tile + 16);
  };
  if (todo > 0) set_item();
  // lane's place in a piece: kDims / 16 lanes per row
  constexpr int kLanesRow = Cfg::kDims / 16, kRowsStep = 32 / kLanesRow;
  const uint32_t ring_s = smem_addr(ring);
  const uint32_t ld_dst = (lane / kLanesRow) * Cfg::kRow + (lane % kLanesRow) * 16;
  const int ld_src = (lane / kLanesRow) * D + part * Cfg::kDims + (lane % kLanesRow) * 16;
  auto request = [&]() {
    if (ld_todo > 0) {
      const int half = ld_phase & 1;
      const bool is_v = ld_phase >= 2;
      const int pos = ld.tile * kKv8Tile + half * 16;
      const int page = ld_page[half];
      const int64_t block = static_cast<int64_t>(max(page, 0)) * heads + ld_head;
      const uint8_t* src = (is_v ? p.cache.v : p.cache.k) + ld_src +
                           (block * p.cache.page + (pos & (p.cache.page - 1))) * D;
      const uint32_t dst = ring_s + ld_buf + ld_dst;
      const int rows_ok = page >= 0 ? ld_hi - pos : 0;
      if (rows_ok >= 16) {
#pragma unroll
        for (int j = 0; j < 16 / kRowsStep; ++j)
          cp16(dst + j * kRowsStep * Cfg::kRow, src + j * kRowsStep * D);
      } else {  // zeros in rows past the end, or everywhere
#pragma unroll
        for (int j = 0; j < 16 / kRowsStep; ++j)
          cp16_z(dst + j * kRowsStep * Cfg::kRow, src + j * kRowsStep * D,
                 j * kRowsStep + lane / kLanesRow < rows_ok ? 16 : 0);
      }
      if (lane == 0 && ld_phase != 3) {
        // a piece's scale and page id ride in its first row's padding; V's second
        // scale comes with the first half, since P needs both
        cp4_z(ring_s + ld_buf + Cfg::kDims,
              (is_v ? p.cache.v_scale : p.cache.k_scale) + block, page >= 0 ? 4 : 0);
        *reinterpret_cast<int*>(ring + ld_buf + Cfg::kDims + 4) = page;
        if (is_v) {
          const int page1 = ld_page[1];
          cp4_z(ring_s + ld_buf + Cfg::kDims + 8,
                p.cache.v_scale + static_cast<int64_t>(max(page1, 0)) * heads + ld_head,
                page1 >= 0 ? 4 : 0);
        }
      }
      if (ld_phase == 0) {  // look the next tile's pages up one tile ahead
        const int np = pos + kKv8Tile;
        ld_next[0] = ld.left > 1 ? lookup(np) : -1;
        ld_next[1] = ld.left > 1 ? lookup(np + 16) : -1;
      }
      if (ld_phase == 3) {
        --ld_todo;
        ++ld.tile;
        if (--ld.left == 0) {
          list.next_item(ld);
          if (ld_todo > 0) set_item();
        } else {
          ld_page[0] = ld_next[0];
          ld_page[1] = ld_next[1];
        }
      }
      ld_phase = (ld_phase + 1) & 3;
      ld_buf = ld_buf + Cfg::kBuf == Cfg::kRing ? 0 : ld_buf + Cfg::kBuf;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < Cfg::kBufs; ++i) request();

  // ---- the computing side ----
  uint32_t qf[Cfg::kChunks][8];
  float acc[Cfg::kTilesM][4];
  float m_o[2], m_s[2], l_s[2];           // columns 2t, 2t + 1: shift of O; max and sum of P
  float q_back[2];               // log2(e) * 2^-e of the column's Q
  int last_key[2];               // last visible key, -1: a padded column
  Place pl = first;
  uint32_t use = 0;                       // ring offset of the next piece
  int head = 0, cg = 0, swap = 0;

  auto begin_item = [&]() {
    list.item_head(pl.b, pl.item, head, cg);
    const RowPlan r = rows[pl.b];
    // this thread's Q fragments: column g, dims of chunk c(t, i)
    const int col = cg * kCols + g;
    const int tok = col / p.group;
    const bool have = tok < r.n;
    const __nv_bfloat16* qp =
        p.q + static_cast<int64_t>(pl.b) * p.q_stride[0] +
        static_cast<int64_t>(have ? tok : 0) * p.q_stride[1] +
        static_cast<int64_t>(head * p.group + (have ? col - tok * p.group : 0)) * p.q_stride[2];
    // its raw values, and the column's largest magnitude over all D dims (the other
    // warps' dims too, so that every warp of the team finds the same one)
    uint4 raw[Cfg::kChunks][2];
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < kTeam; ++w) {
#pragma unroll
      for (int i = 0; i < Cfg::kChunks; ++i) {
        const uint4* s = reinterpret_cast<const uint4*>(
            qp + (part ^ (kTeam - 1 - w)) * Cfg::kDims + (2 * t + (i & 1) + 8 * (i >> 1)) * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          raw[i][h] = have ? s[h] : make_uint4(0u, 0u, 0u, 0u);
          const uint4 x = raw[i][h];
          top = __vmaxu2(__vmaxu2(top, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu);
          top = __vmaxu2(__vmaxu2(top, x.z & 0x7fff7fffu), x.w & 0x7fff7fffu);
        }
      }
    }
    top = max(top >> 16, top & 0xffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = q_exponent(__uint_as_float(top << 16));
    // two factors: 2^e alone may leave the fp32 range for the smallest inputs
    const float f1 = __uint_as_float(static_cast<uint32_t>(127 + e / 2) << 23);
    const float f2 = __uint_as_float(static_cast<uint32_t>(127 + e - e / 2) << 23);
#pragma unroll
    for (int i = 0; i < Cfg::kChunks; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w[4] = {raw[i][h].x, raw[i][h].y, raw[i][h].z, raw[i][h].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float lo = __uint_as_float(w[x] << 16) * f1 * f2;
          const float hi = __uint_as_float(w[x] & 0xffff0000u) * f1 * f2;
          const __half2 v = __floats2half2_rn(lo, hi);
          qf[i][4 * h + x] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int ce = __shfl_sync(0xffffffffu, e, (2 * t + x) * 4);  // column 2t + x
      q_back[x] = kLog2e * __uint_as_float(static_cast<uint32_t>(127 - ce) << 23);
      const int ct = (cg * kCols + 2 * t + x) / p.group;
      last_key[x] = ct < r.n ? r.start + ct : -1;
      m_o[x] = m_s[x] = -INFINITY;
      l_s[x] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < Cfg::kTilesM; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[i][x] = 0.f;
  };
  auto column_sums = [&]() {  // over the warp's key rows
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1)
        l_s[x] += __shfl_xor_sync(0xffffffffu, l_s[x], o);
  };
  // A partial O is [column][dim]; padded columns are left out.  (In shared memory the
  // column stride and the order of the four stores keep a quarter-warp's banks apart.)
  auto store_part = [&](float* po, int stride, float4* ml, int cols) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int col = 2 * t + x;
      if (col < cols) {
#pragma unroll
        for (int i = 0; i < Cfg::kSteps; ++i) {
          float4* dst = reinterpret_cast<float4*>(po + col * stride + part * Cfg::kDims +
                                                  v_chunk(g, i) * 16);
          const auto quad = [&](int y) {
            return make_float4(acc[i * 8 + 2 * y][x], acc[i * 8 + 2 * y][2 + x],
                               acc[i * 8 + 2 * y + 1][x],
                               acc[i * 8 + 2 * y + 1][2 + x]);
          };
#pragma unroll
          for (int y = 0; y < 4; ++y) dst[y ^ (g & 1)] = (g & 1) ? quad(y ^ 1) : quad(y);
        }
        if (g == 0 && part == 0)
          ml[col] = make_float4(m_o[x], m_s[x], l_s[x], 0.f);
      }
    }
  };
  auto finish = [&]() {  // the whole item lies in this run
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int col = cg * kCols + 2 * t + x;
      const float f = out_factor(m_o[x], m_s[x], l_s[x]);
#pragma unroll
      for (int i = 0; i < Cfg::kSteps; ++i) {
        float v[16];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          v[2 * y] = acc[i * 8 + y][x];
          v[2 * y + 1] = acc[i * 8 + y][2 + x];
        }
        put_out(p, pl.b, head, col, part * Cfg::kDims + v_chunk(g, i) * 16, v, f);
      }
      if (g == 0 && part == 0) put_lse(p, pl.b, head, col, m_s[x], l_s[x]);
    }
  };

  bool open = false;           // an item is in progress
  bool from_start = false;     // its first tile lies in this run
  if (todo > 0) from_start = list.at_start(pl);
#pragma unroll 1
  while (todo > 0) {
    if (!open) {
      begin_item();
      open = true;
    }
    // ---- S^T of the tile, through shared memory: rows g and g + 8 of both halves ----
    float k_scale[2];
    bool page_ok[2];
    float* mine = exchange + (swap * Cfg::kWarps + warp) * 256 + lane;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Cfg::kBufs - 1) : "memory");
      __syncwarp();
      const uint8_t* kb = ring + use;
      const float sc = *reinterpret_cast<const float*>(kb + Cfg::kDims);
      const bool ok = *reinterpret_cast<const int*>(kb + Cfg::kDims + 4) >= 0;
      k_scale[0] = half == 0 ? sc : k_scale[0];
      page_ok[0] = half == 0 ? ok : page_ok[0];
      k_scale[1] = sc;
      page_ok[1] = ok;
      float c[2][4];
#pragma unroll
      for (int x = 0; x < 4; ++x) c[0][x] = c[1][x] = 0.f;
      const uint8_t* r0 = kb + g * Cfg::kRow + 32 * t;
#pragma unroll
      for (int i = 0; i < Cfg::kChunks; ++i) {
        const int off = (i & 1) * 16 + (i >> 1) * 128;
        const uint4 x = *reinterpret_cast<const uint4*>(r0 + off);
        const uint4 y = *reinterpret_cast<const uint4*>(r0 + 8 * Cfg::kRow + off);
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[4];
          kv8_to_half<kInt8>(xw[j], a[0], a[2]);
          kv8_to_half<kInt8>(yw[j], a[1], a[3]);
          mma_16816(c[j & 1], a, qf[i][2 * j], qf[i][2 * j + 1]);
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        mine[(half * 4 + x) * 32] =
            c[0][x] + c[1][x];
      __syncwarp();
      request();
      use = use + Cfg::kBuf == Cfg::kRing ? 0 : use + Cfg::kBuf;
    }
    if constexpr (kTeam > 1)
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * kTeam) : "memory");
    float s[2][4];
    {  // the team's partial sums, added in the same order by all
      const float* all = exchange + (swap * Cfg::kWarps + team * kTeam) * 256 + lane;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int at = (half * 4 + x) * 32;
          float sum = all[at];
#pragma unroll
          for (int w = 1; w < kTeam; ++w) sum += all[w * 256 + at];
          s[half][x] = sum;
        }
      if constexpr (kTeam > 1) swap ^= 1;
    }

    // ---- mask, running maxima, P ----
    asm volatile("cp.async.wait_group %0;" ::"n"(Cfg::kBufs - 1) : "memory");
    __syncwarp();
    float v_exp[2], v_mant[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t bits =
          *reinterpret_cast<const uint32_t*>(ring + use + Cfg::kDims + 8 * half);
      const int e = static_cast<int>((bits >> 23) & 255u) - 127;
      v_exp[half] = static_cast<float>(e);
      v_mant[half] = e == -127 ? 0.f : __uint_as_float((bits & 0x807fffffu) | 0x3f800000u);
    }
    uint32_t pf[2][2];  // P^T as B operands: column g, keys t, t + 4, t + 8, t + 12
    bool rescale = false;
    float alpha[2];
    const int k_first = pl.tile * kKv8Tile + g;
    uint32_t pk[2][2];         // [half][rows g, g + 8], columns 2t and 2t + 1
    float pv[2][2][2];         // [column][half][row]
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int hi = last_key[x];
      const int lo = p.window > 0 ? hi - p.window : -1;    // keys > lo are visible
      float z[2][2];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int k = k_first + half * 16 + y * 8;
          z[half][y] = page_ok[half] && k <= hi && k > lo
                           ? s[half][2 * y + x] * (k_scale[half] * q_back[x])
                           : -INFINITY;
        }
      float top = fmaxf(z[0][0], z[0][1]), top1 = fmaxf(z[1][0], z[1][1]);
      float top_v = fmaxf(top + v_exp[0], top1 + v_exp[1]);
      top = fmaxf(top, top1);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
      }
      const float m_new = fmaxf(m_s[x], top);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      l_s[x] = l_s[x] * ex2(m_s[x] - m_use) +
                   ((ex2(z[0][0] - m_use) + ex2(z[0][1] - m_use)) +
                    (ex2(z[1][0] - m_use) + ex2(z[1][1] - m_use)));
      m_s[x] = m_new;
      alpha[x] = 1.f;
      if (top_v > m_o[x] + kStale) {  // also the first visible key
        alpha[x] = m_o[x] == -INFINITY ? 0.f : ex2(m_o[x] - top_v);
        m_o[x] = top_v;
        rescale = true;
      }
      const float m_sub = (m_o[x] == -INFINITY ? 0.f : m_o[x]) - kShiftUp;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          pv[x][half][y] = ex2(z[half][y] + v_exp[half] - m_sub) * v_mant[half];
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const __half2 v = __floats2half2_rn(pv[0][half][y], pv[1][half][y]);
        pk[half][y] = *reinterpret_cast<const uint32_t*>(&v);
      }
      const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t x0 = __shfl_sync(0xffffffffu, pk[half][y], t * 4 + (g >> 1));
        const uint32_t x1 = __shfl_sync(0xffffffffu, pk[half][y], (t + 4) * 4 + (g >> 1));
        pf[half][y] = __byte_perm(x0, x1, sel);
      }
    }
    if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
      for (int i = 0; i < Cfg::kTilesM; ++i) {
        acc[i][0] *= alpha[0];
        acc[i][1] *= alpha[1];
        acc[i][2] *= alpha[0];
        acc[i][3] *= alpha[1];
      }
    }
    // ---- O^T += V^T P^T ----
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      uint32_t pb[2];
      pb[0] = half == 0 ? pf[0][0] : pf[1][0];
      pb[1] = half == 0 ? pf[0][1] : pf[1][1];
      const uint8_t* r0 = ring + use + t * Cfg::kRow;
#pragma unroll
      for (int i = 0; i < Cfg::kSteps; ++i) {
        const int off = v_chunk(g, i) * 16;
        uint4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = *reinterpret_cast<const uint4*>(r0 + 4 * j * Cfg::kRow + off);
        const uint32_t w[4][4] = {{x[0].x, x[0].y, x[0].z, x[0].w},
                                  {x[1].x, x[1].y, x[1].z, x[1].w},
                                  {x[2].x, x[2].y, x[2].z, x[2].w},
                                  {x[3].x, x[3].y, x[3].z, x[3].w}};
#pragma unroll
        for (int y = 0; y < 4; ++y) {  // dims 4y .. 4y + 3 of the chunk: two MMAs
          uint32_t a[4], c[4];
          kv8_to_half<kInt8>(__byte_perm(w[0][y], w[1][y], 0x5140), a[0], a[1]);
          kv8_to_half<kInt8>(__byte_perm(w[2][y], w[3][y], 0x5140), a[2], a[3]);
          kv8_to_half<kInt8>(__byte_perm(w[0][y], w[1][y], 0x7362), c[0], c[1]);
          kv8_to_half<kInt8>(__byte_perm(w[2][y], w[3][y], 0x7362), c[2], c[3]);
          mma_16816(acc[i * 8 + 2 * y], a, pb[0], pb[1]);
          mma_16816(acc[i * 8 + 2 * y + 1], c, pb[0], pb[1]);
        }
      }
      __syncwarp();
      request();
      use = use + Cfg::kBuf == Cfg::kRing ? 0 : use + Cfg::kBuf;
      // the second half's codes (after it, the next tile's, which it waits for anyway)
      asm volatile("cp.async.wait_group %0;" ::"n"(Cfg::kBufs - 1) : "memory");
      __syncwarp();
    }

    --todo;
    ++pl.tile;
    if (--pl.left == 0) {
      if (from_start) {  // complete
        column_sums();
        finish();
        open = false;
      } else if (todo > 0) {
        column_sums();
        const int64_t sl = 2 * static_cast<int64_t>(W);
        store_part(p.part_o + sl * Cfg::kOut, D, p.part_ml + sl * kCols,
                   p.rows.tokens * p.group - cg * kCols);
        open = false;
      }
      if (!open) {
        from_start = true;
        list.next_item(pl);
      }
    }
  }

  // ---- the runs' ends: sum what belongs to one item over the CTA's teams ----
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // every warp's ring is free
  if (open) column_sums();
  // tails, one per team each: item key (-1 none), starts in the run, ends in it, row
  if (lane == 0 && part == 0) {
    tails[team] = open ? pl.b * (heads * p.col_groups) + pl.item : -1;
    tails[Cfg::kTeams + team] = from_start;
    tails[2 * Cfg::kTeams + team] = pl.left == 0;
    tails[3 * Cfg::kTeams + team] = pl.b;
  }
  __syncthreads();
  float* osh = reinterpret_cast<float*>(smem);  // [team][column] partial O
  if (open) {
    const int key = tails[team];
    const bool alone = (team == 0 || tails[team - 1] != key) &&
                       (team == Cfg::kTeams - 1 || tails[team + 1] != key);
    if (alone) {  // nothing to add in this CTA
      const int64_t sl = 2 * static_cast<int64_t>(W) + 1;
      store_part(p.part_o + sl * Cfg::kOut, D, p.part_ml + sl * kCols,
                 p.rows.tokens * p.group - cg * kCols);
    } else {
      store_part(osh + team * kCols * Cfg::kOutRow, Cfg::kOutRow, stats + team * kCols, kCols);
    }
  }
  __syncthreads();
  for (int w0 = 0; w0 < Cfg::kTeams;) {
    const int key = tails[w0];
    if (key < 0) {
      ++w0;
      continue;
    }
    int w1 = w0 + 1;
    while (w1 < Cfg::kTeams && tails[w1] == key) ++w1;
    if (w1 == w0 + 1) {
      w0 = w1;
      continue;
    }
    const bool whole = tails[Cfg::kTeams + w0] && tails[2 * Cfg::kTeams + w1 - 1];
    const int b = tails[3 * Cfg::kTeams + w0];
    int h, grp;
    list.item_head(b, key - b * (heads * p.col_groups), h, grp);
    const int cols = min(kCols, p.rows.tokens * p.group - grp * kCols);
    const int64_t sl = 2 * (static_cast<int64_t>(blockIdx.x) * Cfg::kTeams + w0) + 1;
    for (int u = tid; u < cols * (D / 4); u += blockDim.x) {  // four dims of a column
      const int col = u / (D / 4), dim = (u % (D / 4)) * 4;
      float m_shift = -INFINITY, m = -INFINITY, l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = w0; w < w1; ++w) {
        const float2 f = join(m_shift, m, l, stats[w * kCols + col]);
        axpby(v, f, *reinterpret_cast<const float4*>(osh + (w * kCols + col) * Cfg::kOutRow + dim));
      }
      if (whole) {
        put_dims(p, b, h, grp * kCols + col, dim, v, out_factor(m_shift, m, l));
        if (dim == 0) put_lse(p, b, h, grp * kCols + col, m, l);
      } else {
        *reinterpret_cast<float4*>(p.part_o + sl * Cfg::kOut + col * D + dim) = v;
        if (dim == 0) p.part_ml[sl * kCols + col] = make_float4(m_shift, m, l, 0.f);
      }
    }
    w0 = w1;
  }
}

// Items that span CTAs: the sum of their parts.  A part is the tail of the first run
// of the item in each CTA, and, where the item ends inside a run, that run's head.
// A CTA takes kThreads / kSub units (four dims of a column) of one item; kSub groups
// of threads take every kSub-th part each, kAhead of them in flight, and shared memory
// joins them in order.  kSub = 8 when an item has many parts (few long sequences: the
// parts are read by many threads at once), 1 when most have two or three.
template <int kSub, int kThreads, int kAhead>
__global__ void __launch_bounds__(kThreads) kv8_merge_kernel(const Kv8AttnParams p, const int d,
                                                             const int teams) {
  constexpr int kUnits = kThreads / kSub;
  __shared__ float4 sh_o[kSub][kUnits];
  __shared__ float4 sh_ml[kSub][kUnits];
  pdl_enter();
  const int B = p.rows.batch, items = p.cache.heads * p.col_groups;
  const int b = blockIdx.x / items, rest = blockIdx.x % items;
  const int h = rest / p.col_groups, grp = rest % p.col_groups;
  const int4 head4 = *reinterpret_cast<const int4*>(p.plan);
  const int4 row4 = reinterpret_cast<const int4*>(p.plan)[1 + b];
  const int row_first = p.plan[4 + 4 * B + b];
  const int runs = head4.x, total = head4.y, over = head4.z;
  const RowPlan r = {row4.x, row4.y, row4.z, row4.w};
  const int act = (r.n * p.group + p.cols - 1) / p.cols;
  if (grp >= act) return;  // padding: written by the run that met it
  const int nt = row_tiles(r, p.tile);
  const int i0 = row_first + (h * act + grp) * (nt + over), i1 = i0 + nt;
  const int w0 = run_of(i0, runs, total), w1 = run_of(i1 - 1, runs, total);
  if (w0 == w1) return;                                           // one run had it all
  const bool has_head = i1 + over < run_begin(w1 + 1, runs, total);  // run w1 goes on behind it
  if (!has_head && w0 / teams == w1 / teams) return;          // one CTA had it all
  // CTAs that hold a tail of it
  const int c0 = w0 / teams, c1 = (has_head ? w1 - 1 : w1) / teams;
  const int parts = c1 - c0 + 1 + (has_head ? 1 : 0);
  const int sub = threadIdx.x / kUnits, u = threadIdx.x % kUnits;
  const int unit = blockIdx.y * kUnits + u, quads = d / 4;
  const int col = unit / quads, dim = (unit % quads) * 4;
  const bool ok = col < min(p.cols, p.rows.tokens * p.group - grp * p.cols);
  const int64_t out = static_cast<int64_t>(p.cols) * d;
  float m_shift = -INFINITY, m = -INFINITY, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (ok) {
    for (int k0 = sub; k0 < parts; k0 += kAhead * kSub) {
      float4 o[kAhead], st[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int k = k0 + j * kSub;
        if (k < parts) {
          const int c = c0 + k;
          const int64_t sl = c <= c1 ? 2 * static_cast<int64_t>(max(w0, c * teams)) + 1
                                     : 2 * static_cast<int64_t>(w1);
          st[j] = p.part_ml[sl * p.cols + col];
          o[j] = *reinterpret_cast<const float4*>(p.part_o + sl * out + col * d + dim);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (k0 + j * kSub < parts) axpby(v, join(m_shift, m, l, st[j]), o[j]);
    }
  }
  if constexpr (kSub > 1) {
    sh_o[sub][u] = v;
    sh_ml[sub][u] = make_float4(m_shift, m, l, 0.f);
    __syncthreads();
    if (sub > 0) return;
    for (int k = 1; k < kSub; ++k) axpby(v, join(m_shift, m, l, sh_ml[k][u]), sh_o[k][u]);
  }
  if (!ok) return;
  put_dims(p, b, h, grp * p.cols + col, dim, v, out_factor(m_shift, m, l));
  if (dim == 0) put_lse(p, b, h, grp * p.cols + col, m, l);
}

namespace {

// 256 dims per warp (at head dim 512 two warps share a run), 12 warps (170 registers),
// three 16-key pieces in flight per warp: 153 KB per SM.  One row of 131072 keys, 4 KV
// heads, D = 512, e4m3: 99 us against 82 us for its bytes alone.  Measured and slower: 8 or
// 10 warps, 16 warps of 128 registers, four pieces, pieces brought by TMA.
template <int D>
using Decode = AttnShape<D, D / 256, 12, 3>;
template <typename Cfg, bool kInt8>
int launch_attn(const Kv8AttnParams& p, int ctas, cudaStream_t stream) {
  static_assert(Cfg::smem(kKv8MaxBatch) <= kKv8MaxSmem, "shared memory of the largest batch");
  const int smem = Cfg::smem(p.rows.batch);
  // a property of the kernel and not of the call: the same from every host thread
  cudaError_t e = cudaFuncSetAttribute(kv8_attn_kernel<Cfg, kInt8>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg::smem(kKv8MaxBatch));
  if (e == cudaSuccess)
    e = launch_chained(kv8_attn_kernel<Cfg, kInt8>, dim3(ctas), dim3(Cfg::kThreads), smem, stream,
                       p);
  return static_cast<int>(e);
}
template <typename Cfg>
Kv8AttnShape shape_of() {
  return {Cfg::kCols, kKv8Tile, Cfg::kTeams, Cfg::kOut};
}

}  // namespace

Kv8AttnShape kv8_attn_shape(int d, int64_t columns) {
  if (columns > 8) return kv8_wide_shape(d, columns);
  return d == 512 ? shape_of<Decode<512>>() : shape_of<Decode<256>>();
}

int launch_kv8_attn(int d, bool int8, const Kv8AttnParams& p, int ctas, cudaStream_t stream) {
  if (p.cols > 8) return launch_kv8_wide(d, int8, p, ctas, stream);
  if (d == 512) return int8 ? launch_attn<Decode<512>, true>(p, ctas, stream)
                            : launch_attn<Decode<512>, false>(p, ctas, stream);
  return int8 ? launch_attn<Decode<256>, true>(p, ctas, stream)
              : launch_attn<Decode<256>, false>(p, ctas, stream);
}

int launch_kv8_merge(int d, const Kv8AttnParams& p, int ctas, cudaStream_t stream) {
  const int teams = kv8_attn_shape(d, p.cols).runs;
  const int items = p.rows.batch * p.cache.heads * p.col_groups;
  const int columns = std::min(p.cols, p.rows.tokens * p.group);
  const int units = columns * (d / 4);
  // Parts per item: about one per CTA that it spans.  Eight threads per unit pay off as
  // long as they make no more CTAs than the GPU holds at once (16 items of 64
  // columns: a call of 71 us with their 4096 CTAs, of 38 us with one thread per unit).
  if (ctas >= 8 * items && int64_t(items) * units <= 128 * ctas)
    return static_cast<int>(launch_chained(kv8_merge_kernel<8, 256, 8>,
                                           dim3(items, (units + 31) / 32), dim3(256), 0, stream, p,
                                           d, teams));
  return static_cast<int>(launch_chained(kv8_merge_kernel<1, 128, 2>,
                                         dim3(items, (units + 127) / 128), dim3(128), 0, stream, p,
                                         d, teams));
}

}  // namespace g4
