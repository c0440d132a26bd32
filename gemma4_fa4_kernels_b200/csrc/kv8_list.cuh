// What the kernels of the attention over the 8-bit paged KV cache share: the tile
// list that their work is cut from, the column bounds of an item, and the parts'
// joining and writing (kv8_attn.cu, kv8_wide.cu).
#pragma once

#include "g4_sm100.cuh"
#include "kv8.h"

namespace g4 {

// s_v P is held in fp16 as 2^kShiftUp times its value relative to the running
// maximum, which may lag by 2^kStale before O is rescaled: below 2^15, and normal
// down to 2^-25 of the largest.
constexpr float kShiftUp = 11.f;
constexpr float kStale = 3.f;

// A tile's place: row, item within the row, tile.
struct Place {
  int b;
  int item;     // active items (queries present) first, then the padded column groups
  int tile;     // absolute tile index
  int left;     // tiles left in the item
};

struct RowPlan {
  int slot;
  int start;
  int n;
  int lo;       // first visible key of the row
};

__device__ __forceinline__ RowPlan row_plan(const Kv8AttnParams& p, int b) {
  const Kv8Row r = kv8_row(p.cache, p.rows, b, p.max_k);
  RowPlan rp;
  rp.slot = r.slot;
  rp.start = r.start;
  rp.n = r.n;
  rp.lo = p.window > 0 ? max(0, r.start - p.window + 1) : 0;
  return rp;
}
__device__ __forceinline__ int row_tiles(const RowPlan& r, int tile) {
  return r.n > 0 ? (r.start + r.n + tile - 1) / tile - r.lo / tile : 1;
}

// Run i of n over `total` tiles begins at floor(i * total / n); n <= total.
__device__ __forceinline__ int run_begin(int i, int n, int total) {
  return static_cast<int>(static_cast<int64_t>(i) * total / n);
}
__device__ __forceinline__ int run_of(int tile, int n, int total) {
  return static_cast<int>((static_cast<int64_t>(tile + 1) * n - 1) / total);
}

// The list of a call's tiles: rows in order, each row's active items (KV head major),
// then one tile for every padded column group.  Every item ends with kOver entries more
// that stand for no tile: taking up an item costs a run the time of about one tile (wide
// kernel: two), and with these entries runs of many short items are as long as the others.
// us, without / with one / two: decode, 24 rows of 90 to 32768 keys 129 / 121 / 120, a
// window over 96 rows 123 / 117 / 119; five drafted tokens, 6 rows 60 / 53.7 / 50.6.
// `rows(b)` gives row b's plan, prefix[b] its first list index.
template <int kTile, int kCols, int kOver, typename Rows>
struct TileList {
  const Kv8AttnParams& p;
  const Rows& rows;
  const int* prefix;

  __device__ __forceinline__ int groups(const RowPlan& r) const {
    return (r.n * p.group + kCols - 1) / kCols;
  }
  __device__ __forceinline__ int active_items(const RowPlan& r) const {
    return p.cache.heads * groups(r);
  }
  __device__ __forceinline__ int row_weight(const RowPlan& r) const {
    const int a = groups(r);
    return p.cache.heads * (a * (row_tiles(r, kTile) + kOver) + (p.col_groups - a) * (1 + kOver));
  }
  __device__ __forceinline__ bool at_start(const Place& pl) const {
    const RowPlan r = rows(pl.b);
    return pl.left == (pl.item < active_items(r) ? row_tiles(r, kTile) : 1);
  }
  // Entry x's place, the next item's start if it stands for no tile; `before`: the tiles
  // before it.
  __device__ __forceinline__ Place locate(int x, int& before) const {
    const int per_row = p.cache.heads * p.col_groups;
    if (x >= prefix[p.rows.batch]) {
      before = x - kOver * p.rows.batch * per_row;
      return {p.rows.batch, 0, 0, 0};
    }
    int lo = 0, hi = p.rows.batch;  // prefix[lo] <= x < prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= x) lo = mid; else hi = mid;
    }
    Place pl;
    pl.b = lo;
    const RowPlan r = rows(lo);
    const int nt = row_tiles(r, kTile);
    const int act = active_items(r);
    const int rel = x - prefix[lo];
    int left;
    if (rel < act * (nt + kOver)) {
      pl.item = rel / (nt + kOver);
      const int at = rel - pl.item * (nt + kOver);
      pl.tile = r.lo / kTile + at;
      left = nt - at;
    } else {
      const int at = rel - act * (nt + kOver);
      pl.item = act + at / (1 + kOver);
      pl.tile = 0;
      left = 1 - at % (1 + kOver);
    }
    pl.left = max(left, 0);
    before = x - kOver * (lo * per_row + pl.item) + min(left, 0);
    if (left <= 0) next_item(pl);
    return pl;
  }
  // The first tile of an item.
  __device__ __forceinline__ Place item_place(int b, int item) const {
    const RowPlan r = rows(b);
    const bool act = item < active_items(r);
    return {b, item, act ? r.lo / kTile : 0, act ? row_tiles(r, kTile) : 1};
  }
  __device__ __forceinline__ void next_item(Place& pl) const {
    ++pl.item;
    if (pl.item >= p.cache.heads * p.col_groups) {
      ++pl.b;
      pl.item = 0;
      if (pl.b >= p.rows.batch) {
        pl.left = 0;
        return;
      }
    }
    pl = item_place(pl.b, pl.item);
  }
  // KV head and column group of an item
  __device__ __forceinline__ void item_head(int b, int item, int& head, int& cg) const {
    const int a = groups(rows(b));
    if (item < p.cache.heads * a) {
      head = item / a;
      cg = item - head * a;
    } else {
      const int rest = p.col_groups - a;
      const int j = item - p.cache.heads * a;
      head = j / rest;
      cg = a + j - head * rest;
    }
  }
};

// The whole CTA: prefix sums of the rows' weights, and the plan that the merge reads
// (written by CTA 0, which also reports the rows).  `keep(b, row)` sees every row once, before `rows(b)` is used.
template <int kThreads, typename List, typename Keep>
__device__ __forceinline__ void plan_rows(const Kv8AttnParams& p, const List& list, int* prefix,
                                          int* scan, const Keep& keep) {
  const int B = p.rows.batch, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (B + kThreads - 1) / kThreads;  // rows per thread, consecutive
  int mine = 0;
  for (int j = 0; j < per; ++j) {
    const int b = tid * per + j;
    if (b >= B) break;
    const RowPlan r = row_plan(p, b);
    keep(b, r);
    if (blockIdx.x == 0) {
      reinterpret_cast<int4*>(p.plan)[1 + b] = make_int4(r.slot, r.start, r.n, r.lo);
      kv8_report(p.status, r.slot);
    }
    mine += list.row_weight(r);
  }
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) scan[warp] = inc;
  __syncthreads();
  int at = inc - mine;
  for (int w = 0; w < warp; ++w) at += scan[w];
  for (int j = 0; j < per; ++j) {
    const int b = tid * per + j;
    if (b >= B) break;
    prefix[b] = at;
    if (blockIdx.x == 0) p.plan[4 + 4 * B + b] = at;
    at += list.row_weight(row_plan(p, b));
    if (b == B - 1) prefix[B] = at;
  }
  __syncthreads();
}

// Exponent of the power of two that brings a column's Q to [2^13, 2^14); zeros and
// non-finite values stay.
__device__ __forceinline__ int q_exponent(float amax) {
  const int bits = static_cast<int>(__float_as_uint(amax) >> 23);
  if (bits == 0 || bits == 255) return 0;
  return min(13 - (bits - 127), 100);
}

// Factor from a held O (sum * 2^(kShiftUp - m_shift)) to the output; 0 without a key.
__device__ __forceinline__ float out_factor(float m_shift, float m, float l) {
  return l == 0.f || m_shift == -INFINITY ? 0.f : ex2(m_shift - kShiftUp - m) / l;
}

// Where column `col` of KV head `h` in row b goes: 16 consecutive dims, and its LSE.
__device__ __forceinline__ void put_out(const Kv8AttnParams& p, int b, int h, int col, int dim,
                                        const float (&v)[16], float f) {
  const int tok = col / p.group;
  if (tok >= p.rows.tokens) return;
  uint32_t w[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) w[x] = pack_bf16x2(v[2 * x] * f, v[2 * x + 1] * f);
  uint4* dst = reinterpret_cast<uint4*>(
      p.o + static_cast<int64_t>(b) * p.o_stride[0] + static_cast<int64_t>(tok) * p.o_stride[1] +
      static_cast<int64_t>(h * p.group + col - tok * p.group) * p.o_stride[2] + dim);
  dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
  dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
// The same for four dims.
__device__ __forceinline__ void put_dims(const Kv8AttnParams& p, int b, int h, int col, int dim,
                                         const float4& v, float f) {
  const int tok = col / p.group;
  *reinterpret_cast<uint2*>(
      p.o + static_cast<int64_t>(b) * p.o_stride[0] + static_cast<int64_t>(tok) * p.o_stride[1] +
      static_cast<int64_t>(h * p.group + col - tok * p.group) * p.o_stride[2] + dim) =
      make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
}
__device__ __forceinline__ void put_lse(const Kv8AttnParams& p, int b, int h, int col, float m,
                                        float l) {
  const int tok = col / p.group;
  if (tok >= p.rows.tokens) return;
  p.lse[static_cast<int64_t>(b) * p.lse_stride[0] +
        static_cast<int64_t>(h * p.group + col - tok * p.group) * p.lse_stride[1] + tok] =
      l > 0.f ? (m + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
}

// Running (shift of O, max, sum) <- with another part's; returns the factors on both Os.
__device__ __forceinline__ float2 join(float& m_shift, float& m, float& l, const float4 st) {
  const float ms = fmaxf(m_shift, st.x), mn = fmaxf(m, st.y);
  const float fa = m_shift == -INFINITY ? 0.f : ex2(m_shift - ms);
  const float fb = st.x == -INFINITY ? 0.f : ex2(st.x - ms);
  l = (m == -INFINITY ? l : l * ex2(m - mn)) + (st.y == -INFINITY ? st.z : st.z * ex2(st.y - mn));
  m_shift = ms;
  m = mn;
  return make_float2(fa, fb);
}

__device__ __forceinline__ void axpby(float4& v, const float2 f, const float4& o) {
  v.x = v.x * f.x + o.x * f.y;
  v.y = v.y * f.x + o.y * f.y;
  v.z = v.z * f.x + o.z * f.y;
  v.w = v.w * f.x + o.w * f.y;
}

}  // namespace g4
