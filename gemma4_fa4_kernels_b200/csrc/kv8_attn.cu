// Attention over the 8-bit paged KV cache for sm_100a: one to a few query tokens
// per sequence (decode, drafted tokens), any batch of ragged lengths.
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
// Work split: every (sequence, KV head, column block) is an item of n 16-key
// tiles; all items' tiles form one list, cut into equal runs, one per warp, so
// ragged batches load every SM alike whatever the lengths are.  A warp streams its
// run's K and V tiles through its own ring of padded shared-memory buffers
// (cp.async), with no barrier against other warps.  An item that lies in one run
// is written at once; the ends of the CTA's runs that belong to one item are
// summed in shared memory; what then still spans CTAs goes to the workspace and
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
// 2^11: below 2^15, rounded by at most 2^-12 of itself, or, for weights more than
// 2^25 below the largest, by 2^-36 of the largest.  The output's rounding to bf16
// is 2^-9 of it.
#include "g4_kernels.h"
#include "g4_sm100.cuh"
#include "kv8.h"

namespace g4 {

namespace {

constexpr float kShiftUp = 11.f;    // log2 of the factor on P
constexpr float kStale = 3.f;       // log2 by which O's maximum may lag before a rescale

template <int D>
struct AttnCfg {
  static constexpr int kRow = D + 16;                  // bytes per key row in a buffer
  static constexpr int kBuf = kKv8Tile * kRow;
  static constexpr int kBufs = D == 512 ? 3 : 6;       // K and V tiles in flight per warp
  static constexpr int kRing = kBufs * kBuf;
  static constexpr int kChunks = D / 64;               // K chunks per thread and row
  static constexpr int kSteps = D / 128;               // V chunks per thread and key
  static constexpr int kAcc = D / 4;                   // O registers per thread
  static constexpr int kRingBytes = kKv8Warps * kRing;
  static constexpr int kStatBytes = kKv8Warps * kKv8Cols * 16 + kKv8Warps * 4 * 4;
  static constexpr int smem(int batch) {
    return kRingBytes + kStatBytes + 16 * batch + 4 * (batch + 1) + 64;
  }
};

// A tile range's place: row, item within the row, tile.
struct Place {
  int b;
  int item;     // active items (queries present) first, then the padded column blocks
  int tile;     // absolute tile index (16 keys)
  int left;     // tiles left in the item
};

struct RowPlan {  // shared memory, one per row
  int slot;
  int start;
  int n;
  int lo;       // first visible key of the row
};

__device__ __forceinline__ int active_blocks(const RowPlan& r, int group) {
  return (r.n * group + kKv8Cols - 1) / kKv8Cols;
}
__device__ __forceinline__ int row_tiles(const RowPlan& r) {
  return r.n > 0 ? (r.start + r.n + kKv8Tile - 1) / kKv8Tile - r.lo / kKv8Tile : 1;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes global -> shared, zeros where `bytes` is 0.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

// 2^(e) * value scaled exactly: the factor of a column's Q and its exponent.
__device__ __forceinline__ int q_exponent(float amax) {
  // amax in [2^(x-1), 2^x): bring it to [2^13, 2^14); zeros and non-finite values stay
  const int bits = static_cast<int>(__float_as_uint(amax) >> 23);
  if (bits == 0 || bits == 255) return 0;
  return min(13 - (bits - 127), 100);
}

// The 16 output dims of V chunk step i in thread row g: one 16-byte chunk.
__device__ __forceinline__ int v_chunk(int g, int i) { return (g & 1) * 4 + (g >> 1) + 8 * i; }

}  // namespace

template <int D, bool kInt8>
__global__ void __launch_bounds__(kKv8Warps * 32, 1) kv8_attn_kernel(const Kv8AttnParams p) {
  using Cfg = AttnCfg<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * Cfg::kRing;
  float4* stats = reinterpret_cast<float4*>(smem + Cfg::kRingBytes);          // [warp][col]
  int* tails = reinterpret_cast<int*>(smem + Cfg::kRingBytes + kKv8Warps * kKv8Cols * 16);
  RowPlan* rows = reinterpret_cast<RowPlan*>(smem + Cfg::kRingBytes + Cfg::kStatBytes);
  int* prefix = reinterpret_cast<int*>(rows + p.rows.batch);
  int* scan = prefix + p.rows.batch + 1;  // 8 warp sums (+ total)

  pdl_enter();
  // ---- plan: checked rows, their tiles, the prefix sum over rows ----
  const int B = p.rows.batch, heads = p.cache.heads;
  {
    const int per = (B + 255) / 256;  // rows per thread, consecutive
    int mine = 0;
    for (int j = 0; j < per; ++j) {
      const int b = tid * per + j;
      if (b >= B) break;
      const Kv8Row r = kv8_row(p.cache, p.rows, b, p.max_k);
      RowPlan rp;
      rp.slot = r.slot;
      rp.start = r.start;
      rp.n = r.n;
      rp.lo = p.window > 0 ? max(0, r.start - p.window + 1) : 0;
      rows[b] = rp;
      const int act = active_blocks(rp, p.group);
      mine += heads * (act * row_tiles(rp) + p.col_blocks - act);
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += scan[w];
    int at = before + inc - mine;
    for (int j = 0; j < per; ++j) {
      const int b = tid * per + j;
      if (b >= B) break;
      prefix[b] = at;
      const RowPlan rp = rows[b];
      const int act = active_blocks(rp, p.group);
      at += heads * (act * row_tiles(rp) + p.col_blocks - act);
      if (b == B - 1) prefix[B] = at;
    }
    __syncthreads();
  }
  const int total = prefix[B];
  const int n_warps = gridDim.x * kKv8Warps;
  const int per = (total + n_warps - 1) / n_warps;
  if (blockIdx.x == 0) {
    if (tid == 0) p.plan[0] = per;
    for (int b = tid; b <= B; b += blockDim.x) p.plan[1 + b] = prefix[b];
  }
  const int W = blockIdx.x * kKv8Warps + warp;
  const int w_begin = min(total, W * per), w_end = min(total, w_begin + per);
  int todo = w_end - w_begin;

  // place of a list index
  auto locate = [&](int x) {
    int lo = 0, hi = B;  // prefix[lo] <= x < prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= x) lo = mid; else hi = mid;
    }
    Place pl;
    pl.b = lo;
    const RowPlan r = rows[lo];
    const int nt = row_tiles(r);
    const int act = heads * active_blocks(r, p.group);
    const int rel = x - prefix[lo];
    if (rel < act * nt) {
      pl.item = rel / nt;
      const int at = rel - pl.item * nt;
      pl.tile = r.lo / kKv8Tile + at;
      pl.left = nt - at;
    } else {
      pl.item = act + rel - act * nt;
      pl.tile = 0;
      pl.left = 1;
    }
    return pl;
  };
  auto next_item = [&](Place& pl) {
    const RowPlan r = rows[pl.b];
    ++pl.item;
    if (pl.item >= heads * p.col_blocks) {
      ++pl.b;
      pl.item = 0;
      if (pl.b >= B) {
        pl.left = 0;
        return;
      }
    }
    const RowPlan q = pl.item == 0 ? rows[pl.b] : r;
    const bool act = pl.item < heads * active_blocks(q, p.group);
    pl.tile = act ? q.lo / kKv8Tile : 0;
    pl.left = act ? row_tiles(q) : 1;
  };
  // KV head and column block of an item
  auto item_head = [&](const Place& pl, int& head, int& cb) {
    const int a = active_blocks(rows[pl.b], p.group);
    if (pl.item < heads * a) {
      head = pl.item / a;
      cb = pl.item - head * a;
    } else {
      const int rest = p.col_blocks - a;
      const int j = pl.item - heads * a;
      head = j / rest;
      cb = a + j - head * rest;
    }
  };

  // ---- the loading side: K and V tiles in order K0 V0 K1 V1 ... ----
  Place ld = locate(todo > 0 ? w_begin : 0);
  int ld_todo = todo;        // tiles not yet requested
  int ld_slot = 0;           // ring buffer of the next request
  bool ld_v = false;
  int ld_page = -1, ld_next = -1;
  int ld_head = 0;
  int ld_hi = 0;             // one past the last key of the item's row
  auto lookup = [&](const Place& pl) {
    const RowPlan r = rows[pl.b];
    return r.n > 0 && pl.left > 0 ? kv8_page(p.cache, r.slot, pl.tile * kKv8Tile) : -1;
  };
  auto set_item = [&]() {
    int cb;
    item_head(ld, ld_head, cb);
    ld_hi = rows[ld.b].n > 0 ? rows[ld.b].start + rows[ld.b].n : 0;
  };
  if (todo > 0) {
    set_item();
    ld_page = lookup(ld);
  }
  auto request = [&]() {
    if (ld_todo > 0) {
      const int pos = ld.tile * kKv8Tile;
      uint8_t* buf = ring + ld_slot * Cfg::kBuf;
      const uint32_t dst = smem_addr(buf);
      const int page = ld_page;
      const int64_t block = static_cast<int64_t>(max(page, 0)) * heads + ld_head;
      const uint8_t* src = (ld_v ? p.cache.v : p.cache.k) +
                           (block * p.cache.page + (pos & (p.cache.page - 1))) * D;
      const int rows_ok = page >= 0 ? min(kKv8Tile, ld_hi - pos) : 0;
      if constexpr (D == 512) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          cp16(dst + j * Cfg::kRow + lane * 16, src + j * 512 + lane * 16, j < rows_ok ? 16 : 0);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int row = 2 * j + (lane >> 4);
          cp16(dst + row * Cfg::kRow + (lane & 15) * 16, src + j * 512 + lane * 16,
               row < rows_ok ? 16 : 0);
        }
      }
      if (lane == 0) {  // the block's scale and the page id ride in the first row's padding
        cp4(dst + D, (ld_v ? p.cache.v_scale : p.cache.k_scale) + block, page >= 0 ? 4 : 0);
        *reinterpret_cast<int*>(buf + D + 4) = page;
      }
      if (ld_v) {
        --ld_todo;
        ++ld.tile;
        if (--ld.left == 0) {
          next_item(ld);
          if (ld_todo > 0) {
            set_item();
            ld_page = lookup(ld);
          }
        } else {
          ld_page = ld_next;
        }
      } else {  // look the next tile's page up one tile ahead
        Place nx = ld;
        ++nx.tile;
        --nx.left;
        ld_next = ld_todo > 1 ? lookup(nx) : -1;
      }
      ld_v = !ld_v;
      ld_slot = ld_slot + 1 == Cfg::kBufs ? 0 : ld_slot + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < Cfg::kBufs; ++i) request();

  // ---- the computing side ----
  uint32_t qf[Cfg::kChunks][8];
  float acc[Cfg::kAcc / 4][4];
  float m_o[2], m_s[2], l_s[2];  // per column 2t, 2t + 1: shift of O; max and partial sum of P
  float q_back[2];               // log2(e) * 2^-e of the column's Q
  Place pl = locate(todo > 0 ? w_begin : 0);
  int use_slot = 0;
  int head = 0, cb = 0;

  auto begin_item = [&]() {
    item_head(pl, head, cb);
    const RowPlan r = rows[pl.b];
    // this thread's Q fragments: column g, dims of chunk c(t, i)
    const int col = cb * kKv8Cols + g;
    const int tok = col / p.group;
    const bool have = tok < r.n;
    const __nv_bfloat16* qp =
        p.q + static_cast<int64_t>(pl.b) * p.q_stride[0] +
        static_cast<int64_t>(have ? tok : 0) * p.q_stride[1] +
        static_cast<int64_t>(head * p.group + (have ? col - tok * p.group : 0)) * p.q_stride[2];
    uint4 raw[Cfg::kChunks][2];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < Cfg::kChunks; ++i) {
      const int c = 2 * t + (i & 1) + 8 * (i >> 1);
      const uint4* s = reinterpret_cast<const uint4*>(qp + c * 16);
      raw[i][0] = have ? s[0] : make_uint4(0u, 0u, 0u, 0u);
      raw[i][1] = have ? s[1] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < Cfg::kChunks; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w[4] = {raw[i][h].x, raw[i][h].y, raw[i][h].z, raw[i][h].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          amax = fmaxf(amax, fabsf(__uint_as_float(w[x] << 16)));
          amax = fmaxf(amax, fabsf(__uint_as_float(w[x] & 0xffff0000u)));
        }
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = q_exponent(amax);
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
      m_o[x] = m_s[x] = -INFINITY;
      l_s[x] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < Cfg::kAcc / 4; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[i][x] = 0.f;
  };

  // Sum over the warp's rows of a column's partial sums.
  auto column_sums = [&]() {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l_s[x] += __shfl_xor_sync(0xffffffffu, l_s[x], o);
    }
  };
  auto slot_store = [&](int which) {  // raw partial of this warp (0 head, 1 tail)
    const int64_t s = 2 * static_cast<int64_t>(W) + which;
    float* po = p.part_o + s * (D * kKv8Cols);
    const int cols = p.rows.tokens * p.group - cb * kKv8Cols;
    if (2 * t < cols) {
#pragma unroll
      for (int i = 0; i < Cfg::kAcc / 4; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) po[(i * 4 + x) * 32 + lane] = acc[i][x];
    }
    if (g == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
        p.part_ml[s * kKv8Cols + 2 * t + x] = make_float4(m_o[x], m_s[x], l_s[x], 0.f);
    }
  };
  // 16 consecutive dims of one column
  auto put = [&](int b, int h, int block, int col8, int step, int gg, const float (&v)[16],
                 float f) {
    const int col = block * kKv8Cols + col8;
    const int tok = col / p.group;
    if (tok >= p.rows.tokens) return;
    uint32_t w[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) w[x] = pack_bf16x2(v[2 * x] * f, v[2 * x + 1] * f);
    uint4* dst = reinterpret_cast<uint4*>(
        p.o + static_cast<int64_t>(b) * p.o_stride[0] + static_cast<int64_t>(tok) * p.o_stride[1] +
        static_cast<int64_t>(h * p.group + col - tok * p.group) * p.o_stride[2] +
        v_chunk(gg, step) * 16);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  };
  auto put_lse = [&](int b, int h, int block, int col8, float m, float l) {
    const int col = block * kKv8Cols + col8;
    const int tok = col / p.group;
    if (tok >= p.rows.tokens) return;
    p.lse[static_cast<int64_t>(b) * p.lse_stride[0] +
          static_cast<int64_t>(h * p.group + col - tok * p.group) * p.lse_stride[1] + tok] =
        l > 0.f ? (m + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
  };
  auto out_factor = [&](float m_shift, float m, float l) {
    // O is held as sum * 2^(kShiftUp - m_shift); without a visible key it is zero
    return l == 0.f || m_shift == -INFINITY ? 0.f : ex2(m_shift - kShiftUp - m) / l;
  };
  auto finish = [&]() {  // the whole item lies in this warp's run
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float f = out_factor(m_o[x], m_s[x], l_s[x]);
#pragma unroll
      for (int i = 0; i < Cfg::kSteps; ++i) {
        float v[16];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          v[2 * y] = acc[i * 8 + y][x];
          v[2 * y + 1] = acc[i * 8 + y][2 + x];
        }
        put(pl.b, head, cb, 2 * t + x, i, g, v, f);
      }
      if (g == 0) put_lse(pl.b, head, cb, 2 * t + x, m_s[x], l_s[x]);
    }
  };

  bool open = false;           // an item is in progress
  bool from_start = false;     // its first tile lies in this run
  if (todo > 0) {
    from_start = pl.left == (pl.item < heads * active_blocks(rows[pl.b], p.group)
                                 ? row_tiles(rows[pl.b]) : 1);
  }
#pragma unroll 1
  while (todo > 0) {
    if (!open) {
      begin_item();
      open = true;
    }
    const RowPlan r = rows[pl.b];
    // ---- S^T of the tile ----
    asm volatile("cp.async.wait_group %0;" ::"n"(Cfg::kBufs - 1) : "memory");
    __syncwarp();
    float s[2][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) s[0][x] = s[1][x] = 0.f;
    const uint8_t* kb = ring + use_slot * Cfg::kBuf;
    const float k_scale = *reinterpret_cast<const float*>(kb + D);
    const int page = *reinterpret_cast<const int*>(kb + D + 4);
    {
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
          mma_16816(s[j & 1], a, qf[i][2 * j], qf[i][2 * j + 1]);
        }
      }
    }
    __syncwarp();
    request();
    use_slot = use_slot + 1 == Cfg::kBufs ? 0 : use_slot + 1;

    // ---- mask, running maxima, P ----
    asm volatile("cp.async.wait_group %0;" ::"n"(Cfg::kBufs - 1) : "memory");
    __syncwarp();
    const uint8_t* vb = ring + use_slot * Cfg::kBuf;
    const float v_scale = *reinterpret_cast<const float*>(vb + D);
    const int v_exp = static_cast<int>((__float_as_uint(v_scale) >> 23) & 255u) - 127;
    const float v_mant = v_exp == -127 ? 0.f
                                       : __uint_as_float((__float_as_uint(v_scale) & 0x807fffffu) |
                                                         0x3f800000u);
    uint32_t pk[2];  // P of keys g and g + 8, columns 2t and 2t + 1
    bool rescale = false;
    float alpha[2];
    {
      float pv[2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int tok = (cb * kKv8Cols + 2 * t + x) / p.group;
        const int q_pos = r.start + tok;
        float z[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int k_pos = pl.tile * kKv8Tile + g + 8 * y;
          const bool seen = page >= 0 && tok < r.n && k_pos <= q_pos &&
                            (p.window == 0 || k_pos > q_pos - p.window);
          z[y] = seen ? (s[0][2 * y + x] + s[1][2 * y + x]) * (k_scale * q_back[x]) : -INFINITY;
        }
        float top = fmaxf(z[0], z[1]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m_s[x], top);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        l_s[x] = l_s[x] * ex2(m_s[x] - m_use) + ex2(z[0] - m_use) + ex2(z[1] - m_use);
        m_s[x] = m_new;
        alpha[x] = 1.f;
        const float top_v = top + static_cast<float>(v_exp);
        if (top_v > m_o[x] + kStale) {  // also the first visible key
          alpha[x] = m_o[x] == -INFINITY ? 0.f : ex2(m_o[x] - top_v);
          m_o[x] = top_v;
          rescale = true;
        }
        const float m_sub = (m_o[x] == -INFINITY ? 0.f : m_o[x]) - static_cast<float>(v_exp) -
                            kShiftUp;
        pv[x][0] = ex2(z[0] - m_sub) * v_mant;
        pv[x][1] = ex2(z[1] - m_sub) * v_mant;
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const __half2 v = __floats2half2_rn(pv[0][y], pv[1][y]);
        pk[y] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
      for (int i = 0; i < Cfg::kAcc / 4; ++i) {
        acc[i][0] *= alpha[0];
        acc[i][1] *= alpha[1];
        acc[i][2] *= alpha[0];
        acc[i][3] *= alpha[1];
      }
    }
    // P^T as the B operand: column g, keys t, t + 4, t + 8, t + 12
    uint32_t b0, b1;
    {
      const uint32_t x0 = __shfl_sync(0xffffffffu, pk[0], t * 4 + (g >> 1));
      const uint32_t x1 = __shfl_sync(0xffffffffu, pk[0], (t + 4) * 4 + (g >> 1));
      const uint32_t x2 = __shfl_sync(0xffffffffu, pk[1], t * 4 + (g >> 1));
      const uint32_t x3 = __shfl_sync(0xffffffffu, pk[1], (t + 4) * 4 + (g >> 1));
      const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
      b0 = __byte_perm(x0, x1, sel);
      b1 = __byte_perm(x2, x3, sel);
    }
    // ---- O^T += V^T P^T ----
    {
      const uint8_t* r0 = vb + t * Cfg::kRow;
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
          mma_16816(acc[i * 8 + 2 * y], a, b0, b1);
          mma_16816(acc[i * 8 + 2 * y + 1], c, b0, b1);
        }
      }
    }
    __syncwarp();
    request();
    use_slot = use_slot + 1 == Cfg::kBufs ? 0 : use_slot + 1;

    --todo;
    ++pl.tile;
    if (--pl.left == 0) {
      if (from_start) {  // complete
        column_sums();
        finish();
        open = false;
      } else if (todo > 0) {  // began in an earlier run, ends inside this one
        column_sums();
        slot_store(0);
        open = false;
      }
      if (!open) {
        from_start = true;
        next_item(pl);
      }
    }
  }

  // ---- the runs' ends: sum what belongs to one item over the CTA's warps ----
  // tails, one per warp each: item key (-1 none), starts in the run, ends in it, row
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // every warp's ring is free
  if (open) column_sums();
  if (lane == 0) {
    tails[warp] = open ? pl.b * (heads * p.col_blocks) + pl.item : -1;
    tails[8 + warp] = from_start;
    tails[16 + warp] = pl.left == 0;
    tails[24 + warp] = pl.b;
  }
  float* osh = reinterpret_cast<float*>(smem);  // [warp][register][lane]
  if (open) {
#pragma unroll
    for (int i = 0; i < Cfg::kAcc / 4; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        osh[warp * (D * kKv8Cols) + (i * 4 + x) * 32 + lane] = acc[i][x];
    if (g == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
        stats[warp * kKv8Cols + 2 * t + x] = make_float4(m_o[x], m_s[x], l_s[x], 0.f);
    }
  }
  __syncthreads();
  for (int w0 = 0; w0 < kKv8Warps;) {
    const int key = tails[w0];
    if (key < 0) {
      ++w0;
      continue;
    }
    int w1 = w0 + 1;
    while (w1 < kKv8Warps && tails[w1] == key) ++w1;
    const bool whole = tails[8 + w0] && tails[16 + w1 - 1];
    Place it;
    it.b = tails[24 + w0];
    it.item = key - it.b * (heads * p.col_blocks);
    int h, block;
    item_head(it, h, block);
    // thread: step, column of a lane's pair, lane
    for (int u = tid; u < Cfg::kSteps * 64; u += blockDim.x) {
      const int ln = u & 31, x = (u >> 5) & 1, i = u >> 6;
      const int col8 = 2 * (ln & 3) + x;
      float m_shift = -INFINITY, m = -INFINITY, l = 0.f;
      for (int w = w0; w < w1; ++w) {
        const float4 st = stats[w * kKv8Cols + col8];
        m_shift = fmaxf(m_shift, st.x);
        m = fmaxf(m, st.y);
      }
      float v[16];
#pragma unroll
      for (int y = 0; y < 16; ++y) v[y] = 0.f;
      for (int w = w0; w < w1; ++w) {
        const float4 st = stats[w * kKv8Cols + col8];
        const float fo = st.x == -INFINITY ? 0.f : ex2(st.x - m_shift);
        l += st.y == -INFINITY ? st.z : st.z * ex2(st.y - m);
        const float* src = osh + w * (D * kKv8Cols) + i * 32 * 32 + ln;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          v[2 * y] += fo * src[(y * 4 + x) * 32];
          v[2 * y + 1] += fo * src[(y * 4 + 2 + x) * 32];
        }
      }
      if (whole) {
        put(it.b, h, block, col8, i, ln >> 2, v, out_factor(m_shift, m, l));
        if (i == 0 && (ln >> 2) == 0) put_lse(it.b, h, block, col8, m, l);
      } else {
        const int64_t sl = 2 * (static_cast<int64_t>(blockIdx.x) * kKv8Warps + w0) + 1;
        float* po = p.part_o + sl * (D * kKv8Cols) + i * 32 * 32 + ln;
        if (block * kKv8Cols + col8 < p.rows.tokens * p.group) {
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            po[(y * 4 + x) * 32] = v[2 * y];
            po[(y * 4 + 2 + x) * 32] = v[2 * y + 1];
          }
        }
        if (i == 0 && (ln >> 2) == 0)
          p.part_ml[sl * kKv8Cols + col8] = make_float4(m_shift, m, l, 0.f);
      }
    }
    w0 = w1;
  }
}

// Items that span CTAs: the sum of their parts, one CTA per (item, 128 dims).  A
// part is the tail of the first warp of the item in each CTA, and, where the item
// ends inside a warp's run, the head of that warp.  Four groups of threads take
// every fourth part each; shared memory joins them in order.
template <int D>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const Kv8AttnParams p) {
  __shared__ float sh_o[3][64][16];
  __shared__ float4 sh_ml[3][64];
  pdl_enter();
  const int items = p.cache.heads * p.col_blocks;
  const int b = blockIdx.x / items, rest = blockIdx.x % items;
  const int h = rest / p.col_blocks, block = rest % p.col_blocks;
  const Kv8Row row = kv8_row(p.cache, p.rows, b, p.max_k);
  RowPlan r;
  r.slot = row.slot;
  r.start = row.start;
  r.n = row.n;
  r.lo = p.window > 0 ? max(0, row.start - p.window + 1) : 0;
  const int act = active_blocks(r, p.group);
  if (block >= act) return;  // padding: written by the warp that met it
  const int per = p.plan[0];
  const int nt = row_tiles(r);
  const int i0 = p.plan[1 + b] + (h * act + block) * nt, i1 = i0 + nt;
  const int w0 = i0 / per, w1 = (i1 - 1) / per;
  if (w0 == w1) return;  // one warp had it all
  const int total = p.plan[1 + p.rows.batch];
  const bool has_head = i1 < min(total, (w1 + 1) * per);      // ends inside warp w1's run
  if (!has_head && w0 / kKv8Warps == w1 / kKv8Warps) return;  // one CTA had it all
  // CTAs that hold a tail of it
  const int c0 = w0 / kKv8Warps, c1 = (has_head ? w1 - 1 : w1) / kKv8Warps;
  const int parts = c1 - c0 + 1 + (has_head ? 1 : 0);
  const int tid = threadIdx.x, sub = tid >> 6, u = tid & 63;
  const int ln = u & 31, x = u >> 5, i = blockIdx.y;
  const int col8 = 2 * (ln & 3) + x;
  const bool col_ok = block * kKv8Cols + col8 < p.rows.tokens * p.group;
  float m_shift = -INFINITY, m = -INFINITY, l = 0.f, v[16];
#pragma unroll
  for (int y = 0; y < 16; ++y) v[y] = 0.f;
  if (col_ok) {
    for (int k = sub; k < parts; k += 4) {
      const int c = c0 + k;
      const int64_t sl = c <= c1 ? 2 * static_cast<int64_t>(max(w0, c * kKv8Warps)) + 1
                                 : 2 * static_cast<int64_t>(w1);
      const float4 st = p.part_ml[sl * kKv8Cols + col8];
      const float* po = p.part_o + sl * (D * kKv8Cols) + i * 32 * 32 + ln;
      float o[16];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        o[2 * y] = po[(y * 4 + x) * 32];
        o[2 * y + 1] = po[(y * 4 + 2 + x) * 32];
      }
      const float ms = fmaxf(m_shift, st.x), mn = fmaxf(m, st.y);
      const float fa = m_shift == -INFINITY ? 0.f : ex2(m_shift - ms);
      const float fb = st.x == -INFINITY ? 0.f : ex2(st.x - ms);
      l = (m == -INFINITY ? l : l * ex2(m - mn)) + (st.y == -INFINITY ? st.z : st.z * ex2(st.y - mn));
#pragma unroll
      for (int y = 0; y < 16; ++y) v[y] = v[y] * fa + o[y] * fb;
      m_shift = ms;
      m = mn;
    }
  }
  if (sub > 0) {
#pragma unroll
    for (int y = 0; y < 16; ++y) sh_o[sub - 1][u][y] = v[y];
    sh_ml[sub - 1][u] = make_float4(m_shift, m, l, 0.f);
  }
  __syncthreads();
  if (sub > 0 || !col_ok) return;
#pragma unroll 1
  for (int k = 0; k < 3; ++k) {
    const float4 st = sh_ml[k][u];
    const float ms = fmaxf(m_shift, st.x), mn = fmaxf(m, st.y);
    const float fa = m_shift == -INFINITY ? 0.f : ex2(m_shift - ms);
    const float fb = st.x == -INFINITY ? 0.f : ex2(st.x - ms);
    l = (m == -INFINITY ? l : l * ex2(m - mn)) + (st.y == -INFINITY ? st.z : st.z * ex2(st.y - mn));
#pragma unroll
    for (int y = 0; y < 16; ++y) v[y] = v[y] * fa + sh_o[k][u][y] * fb;
    m_shift = ms;
    m = mn;
  }
  const float f = l == 0.f || m_shift == -INFINITY ? 0.f : ex2(m_shift - kShiftUp - m) / l;
  const int col = block * kKv8Cols + col8;
  const int tok = col / p.group, qh = h * p.group + col - tok * p.group;
  uint32_t w[8];
#pragma unroll
  for (int y = 0; y < 8; ++y) w[y] = pack_bf16x2(v[2 * y] * f, v[2 * y + 1] * f);
  uint4* dst = reinterpret_cast<uint4*>(p.o + static_cast<int64_t>(b) * p.o_stride[0] +
                                        static_cast<int64_t>(tok) * p.o_stride[1] +
                                        static_cast<int64_t>(qh) * p.o_stride[2] +
                                        v_chunk(ln >> 2, i) * 16);
  dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
  dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  if (i == 0 && (ln >> 2) == 0)
    p.lse[static_cast<int64_t>(b) * p.lse_stride[0] + static_cast<int64_t>(qh) * p.lse_stride[1] +
          tok] = l > 0.f ? (m + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
}

namespace {
template <int D, bool kInt8>
int launch_attn(const Kv8AttnParams& p, int ctas, cudaStream_t stream) {
  const int smem = AttnCfg<D>::smem(p.rows.batch);
  cudaError_t e = cudaFuncSetAttribute(kv8_attn_kernel<D, kInt8>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess)
    e = launch_chained(kv8_attn_kernel<D, kInt8>, dim3(ctas), dim3(kKv8Warps * 32), smem, stream,
                       p);
  return static_cast<int>(e);
}
}  // namespace

int launch_kv8_attn(int d, bool int8, const Kv8AttnParams& p, int ctas, cudaStream_t stream) {
  if (d == 512) return int8 ? launch_attn<512, true>(p, ctas, stream)
                            : launch_attn<512, false>(p, ctas, stream);
  return int8 ? launch_attn<256, true>(p, ctas, stream) : launch_attn<256, false>(p, ctas, stream);
}

int launch_kv8_merge(int d, const Kv8AttnParams& p, cudaStream_t stream) {
  const dim3 grid(p.rows.batch * p.cache.heads * p.col_blocks, d / 128);
  return static_cast<int>(
      d == 512 ? launch_chained(kv8_merge_kernel<512>, grid, dim3(256), 0, stream, p)
               : launch_chained(kv8_merge_kernel<256>, grid, dim3(256), 0, stream, p));
}

}  // namespace g4
