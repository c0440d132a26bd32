// Writing to and reading from the 8-bit paged KV cache: append (quantise), read
// back (dequantise), and the plan of a prompt chunk's attention.
//
// Append.  A block (page, KV head) has the scale 2^e with the least e such that
// its largest finite magnitude is at most `top` * 2^e (448 for e4m3, 127 for
// int8), e in [kKv8MinExp, kKv8MaxExp]:
//   code = round_to_nearest_even(x * 2^-e), at the largest e at most 240 (e4m3).
// When tokens join a page that holds earlier ones, e only grows; the older codes
// are then requantised from their own values.  x * 2^-e is exact (a power of
// two), so the one rounding is the format's.  Codes are always finite: infinities
// saturate to the largest magnitude, NaN becomes 0, and neither enters e.
//
// Bound: HBM, 2 bytes read and 1 written per element (a decode step: latency).
// One CTA takes one page of one row, one head, K or V: the page's new tokens are
// read once and stay in registers between the maximum and the rounding.
#include "g4_kernels.h"
#include "kv8.h"

namespace g4 {

namespace {

constexpr int kChunk = 8;          // elements per thread and step: 16 bytes of bf16, 8 of codes

// Largest magnitude (bf16 bits, non-finite ignored) of two packed values, kept per half.
__device__ __forceinline__ uint32_t max_finite2(uint32_t m, uint32_t x) {
  const uint32_t a = x & 0x7fff7fffu;
  const uint32_t bad = __vcmpgeu2(a, 0x7f807f80u);
  return __vmaxu2(m, a & ~bad);
}

template <bool kInt8>
__device__ __forceinline__ int block_exponent(uint32_t bits) {  // bits: bf16 magnitude
  // magnitude 1.f * 2^(x - 127); top = 1.75 * 2^8 (e4m3) or 1.984375 * 2^6 (int8)
  const int x = static_cast<int>(bits >> 7), f = static_cast<int>(bits & 127u);
  const int e = kInt8 ? x - 127 - 6 + (f > 126) : x - 127 - 8 + (f > 96);
  return bits == 0 ? kKv8MinExp : min(max(e, kKv8MinExp), kKv8MaxExp<kInt8>);
}

__device__ __forceinline__ float pow2f(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Codes of four finite values that the block's scale covers (below the largest scale).
template <bool kInt8>
__device__ __forceinline__ uint32_t pack4_fast(float a, float b, float c, float d, float back) {
  if constexpr (kInt8) {
    // 1.5 * 2^23 + y rounds y to an integer (ties to even); its low byte is the code
    const float magic = 12582912.f;
    const uint32_t ab = __byte_perm(__float_as_uint(fmaf(a, back, magic)),
                                    __float_as_uint(fmaf(b, back, magic)), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(fmaf(c, back, magic)),
                                    __float_as_uint(fmaf(d, back, magic)), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
  } else {
    uint16_t lo, hi;  // the first source is the upper byte
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b * back), "f"(a * back));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d * back), "f"(c * back));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  }
}

// The same for any values: what lies beyond `top` saturates, NaN becomes 0.
template <bool kInt8>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float top) {
  if constexpr (kInt8) {
    const auto code = [&](float x) {
      const float y = x == x ? fminf(fmaxf(x, -top), top) : 0.f;
      return static_cast<uint32_t>(__float2int_rn(y)) & 255u;
    };
    return code(a) | (code(b) << 8) | (code(c) << 16) | (code(d) << 24);
  } else {
    const auto fin = [&](float x) { return x == x ? fminf(fmaxf(x, -top), top) : 0.f; };
    uint16_t lo, hi;  // the first source is the upper byte
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(fin(b)), "f"(fin(a)));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(fin(d)), "f"(fin(c)));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  }
}

__device__ __forceinline__ float2 half2_floats(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace

// kSteps: chunks a thread holds (1 for single tokens, else 8; 16 for the largest pages).
template <int D, bool kInt8, int kSteps>
__global__ void __launch_bounds__(512) kv8_append_kernel(const Kv8StoreParams p) {
  __shared__ uint32_t red[16];
  pdl_enter();
  const int b = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  const int head = blockIdx.y;
  const Kv8Cache& c = p.cache;
  const Kv8Row row = kv8_row(c, p.rows, b, INT32_MAX);
  if (row.n <= 0) {
    if (blockIdx.x == 0 && head == 0 && !is_v && threadIdx.x == 0) kv8_report(p.status, row.slot);
    return;
  }
  const int first = row.start >> c.page_shift;
  const int page_pos = (first + static_cast<int>(blockIdx.x)) << c.page_shift;
  const int a = max(row.start, page_pos);
  const int n = min(row.start + row.n, page_pos + c.page) - a;  // new tokens of this page
  if (n <= 0) return;
  constexpr int kPerRow = D / kChunk;
  const int64_t* xs = is_v ? p.v_stride : p.k_stride;
  const __nv_bfloat16* x = (is_v ? p.v : p.k) + static_cast<int64_t>(b) * xs[0] +
                           static_cast<int64_t>(a - row.start) * xs[1] +
                           static_cast<int64_t>(head) * xs[2];
  // the values first: the page's lookup below runs while they are on their way
  uint4 in[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int u = threadIdx.x + s * blockDim.x;
    in[s] = make_uint4(0u, 0u, 0u, 0u);
    if (u < n * kPerRow)
      in[s] = *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(u / kPerRow) * xs[1] +
                                              (u % kPerRow) * kChunk);
  }
  const int page = kv8_page(c, row.slot, page_pos);
  // a slot that two rows write to: the first one does, later ones are left out (two
  // CTAs would race on the page's scale)
  if (p.rows.slots) {
    int dup = 0;
    for (int j = threadIdx.x; j < b; j += blockDim.x)
      dup |= p.rows.slots[j] == row.slot && p.rows.ends[j] > p.rows.starts[j];
    if (__syncthreads_or(dup)) {
      if (threadIdx.x == 0 && p.status) atomicOr(p.status, kKv8BadIndex);
      return;
    }
  }
  if (page < 0) {
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, kKv8BadIndex);
    return;
  }
  const int64_t block = static_cast<int64_t>(page) * c.heads + head;
  uint8_t* codes = (is_v ? c.v : c.k) + block * c.page * D;
  float* scale = (is_v ? c.v_scale : c.k_scale) + block;
  const int held = a - page_pos;  // earlier tokens of the page
  const float old_scale = held > 0 ? *scale : 0.f;
  uint32_t m = 0;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    m = __vmaxu2(__vmaxu2(m, in[s].x & 0x7fff7fffu), in[s].y & 0x7fff7fffu);
    m = __vmaxu2(__vmaxu2(m, in[s].z & 0x7fff7fffu), in[s].w & 0x7fff7fffu);
  }
  const bool odd = (m >> 16) >= 0x7f80u || (m & 0xffffu) >= 0x7f80u;  // an infinity or NaN
  if (odd) {
    m = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      m = max_finite2(max_finite2(max_finite2(max_finite2(m, in[s].x), in[s].y), in[s].z), in[s].w);
  }
  m = max(m >> 16, m & 0xffffu);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) m = max(m, red[w]);
  int e = block_exponent<kInt8>(m);
  const auto top_code = [](int exp) {
    return kInt8 ? 127.f : exp == kKv8MaxExp<kInt8> ? 240.f : 448.f;
  };
  if (held > 0) {
    // least power of two not below the stored scale (which is one itself when the
    // append wrote it)
    const uint32_t ob = __float_as_uint(old_scale);
    const int oe = static_cast<int>((ob >> 23) & 255u) - 127 + ((ob & 0x7fffffu) != 0);
    e = max(e, min(max(oe, kKv8MinExp), kKv8MaxExp<kInt8>));
    const float back = pow2f(-e), top = top_code(e);
    if (old_scale * back != 1.f) {
      for (int u = threadIdx.x; u < held * kPerRow; u += blockDim.x) {
        uint2* at = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(u) * kChunk);
        const uint2 old = *at;
        uint32_t w[2] = {old.x, old.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t lo, hi;
          kv8_to_half<kInt8>(w[i], lo, hi);
          const float2 l2 = half2_floats(lo), h2 = half2_floats(hi);
          w[i] = pack4<kInt8>(l2.x * old_scale * back, l2.y * old_scale * back,
                              h2.x * old_scale * back, h2.y * old_scale * back, top);
        }
        *at = make_uint2(w[0], w[1]);
      }
    }
  }
  const float back = pow2f(-e), top = top_code(e);
  const bool any = odd || e == kKv8MaxExp<kInt8>;  // values beyond the codes
  codes += static_cast<int64_t>(held) * D;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int u = threadIdx.x + s * blockDim.x;
    if (u < n * kPerRow) {
      const uint32_t r[4] = {in[s].x, in[s].y, in[s].z, in[s].w};
      uint32_t w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
      {
        const float v[4] = {__uint_as_float(r[2 * i] << 16),
                            __uint_as_float(r[2 * i] & 0xffff0000u),
                            __uint_as_float(r[2 * i + 1] << 16),
                            __uint_as_float(r[2 * i + 1] & 0xffff0000u)};
        w[i] = any ? pack4<kInt8>(v[0] * back, v[1] * back, v[2] * back, v[3] * back, top)
                   : pack4_fast<kInt8>(v[0], v[1], v[2], v[3], back);
      }
      *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(u) * kChunk) = make_uint2(w[0], w[1]);
    }
  }
  if (threadIdx.x == 0) *scale = pow2f(e);
}

// Read back: K and V of the rows' positions as bf16 (code * scale rounded once;
// exact for scales that are powers of two), zeros where the row or the page has
// nothing.  Bound: HBM, 1 byte read and 2 written per element.
// Packed output: so are the rows behind the last segment that a 128-key tile of the
// forward may load (masked there, but 0 * NaN would not be 0).
constexpr int kReadTokens = 16;  // tokens per CTA, K and V
constexpr int kReadTail = 128;
template <int D, bool kInt8>
__global__ void __launch_bounds__(128) kv8_read_kernel(const Kv8StoreParams p) {
  pdl_enter();
  const int b = blockIdx.z;
  const int head = blockIdx.y;
  const Kv8Cache& c = p.cache;
  const Kv8Row row = kv8_row(c, p.rows, b, INT32_MAX);
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) kv8_report(p.status, row.slot);
  const int base = p.out_rows ? p.out_rows[b] : 0;
  int len = p.out_rows ? p.out_rows[b + 1] - base : p.rows.tokens;
  if (p.out_rows && b == p.rows.batch - 1) len += min(kReadTail, p.out_total - base - len);
  const int64_t out_at = (p.out_rows ? static_cast<int64_t>(base) * p.out_stride[1]
                                     : static_cast<int64_t>(b) * p.out_stride[0]) +
                         static_cast<int64_t>(head) * p.out_stride[2];
  constexpr int kPerRow = D / kChunk;
  constexpr int kRows = 128 / kPerRow;  // tokens per step
  constexpr int kSteps = kReadTokens / kRows;
  const int t0 = blockIdx.x * kReadTokens;
  if (t0 >= len) return;
  const int at = threadIdx.x / kPerRow, chunk = (threadIdx.x % kPerRow) * kChunk;
  int page[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int t = t0 + i * kRows + at;
    page[i] = t < min(len, row.n) ? kv8_page(c, row.slot, row.start + t) : -1;
  }
  uint2 w[2][kSteps];
  float s[2][kSteps];
  bool hole = false;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int pos = row.start + t0 + i * kRows + at;
    const int64_t block = static_cast<int64_t>(max(page[i], 0)) * c.heads + head;
    const int64_t from = (block * c.page + (pos & (c.page - 1))) * D + chunk;
    w[0][i] = w[1][i] = make_uint2(0u, 0u);
    s[0][i] = s[1][i] = 0.f;  // a hole reads as exact zeros: its codes and scales are zero here
    if (page[i] >= 0) {
      w[0][i] = __ldcs(reinterpret_cast<const uint2*>(c.k + from));
      w[1][i] = __ldcs(reinterpret_cast<const uint2*>(c.v + from));
      s[0][i] = c.k_scale[block];
      s[1][i] = c.v_scale[block];
    } else {
      hole |= t0 + i * kRows + at < min(len, row.n);
    }
  }
  if (hole && p.holes) p.holes[b] = 1;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int t = t0 + i * kRows + at;
    if (t >= len) break;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint32_t r[2] = {w[kv][i].x, w[kv][i].y};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t lo, hi;
        kv8_to_half<kInt8>(r[j], lo, hi);
        const float2 l2 = half2_floats(lo), h2 = half2_floats(hi);
        o[2 * j] = bf16_pair(l2.x * s[kv][i], l2.y * s[kv][i]);
        o[2 * j + 1] = bf16_pair(h2.x * s[kv][i], h2.y * s[kv][i]);
      }
      *reinterpret_cast<uint4*>((kv ? p.v_out : p.k_out) + out_at +
                                static_cast<int64_t>(t) * p.out_stride[1] + chunk) =
          make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// A prompt chunk's attention runs on the bf16 kernels over a copy of the keys it
// sees, packed: row b's queries are `tokens` rows, its keys the positions
// [first, start + tokens), so that the queries are the keys' last rows (padding
// included; a padded key is later than every real query).  Empty rows get
// `tokens` zero keys.  The bf16 kernels mask by position only: a key of a missing page
// would count with the score of its zeros, so the read marks such rows.  The wide kernel
// then computes the marked rows from the codes and clears the others' padding.
__global__ void __launch_bounds__(1024) kv8_chunk_plan_kernel(const Kv8ChunkParams p) {
  __shared__ int sums[32];
  pdl_enter();
  const int b = threadIdx.x, lane = b & 31, warp = b >> 5;
  int keys = 0, first = 0, last = 0;
  if (b < p.rows.batch) {
    const Kv8Row r = kv8_row(p.cache, p.rows, b, p.max_k);
    kv8_report(p.status, r.slot);
    first = p.window > 0 ? max(0, r.start - p.window + 1) : 0;
    keys = r.start + p.rows.tokens - first;
    last = r.start + r.n;
  }
  int inc = keys;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  for (int w = 0; w < warp; ++w) inc += sums[w];
  if (b < p.rows.batch) {
    p.cu_k[b + 1] = inc;
    p.cu_q[b + 1] = (b + 1) * p.rows.tokens;
    p.first[b] = first;
    p.last[b] = last;
    p.holes[b] = 0;
  }
  if (b == 0) p.cu_q[0] = p.cu_k[0] = 0;
}

namespace {
template <int D, bool kInt8>
int append(const Kv8StoreParams& p, cudaStream_t stream) {
  const int page = p.cache.page, tokens = p.rows.tokens;
  const int pages = tokens > 1 ? (tokens - 2) / page + 2 : 1;  // most that `tokens` can touch
  const int chunks = (tokens < page ? tokens : page) * (D / kChunk);
  const dim3 grid(pages, p.cache.heads, 2 * p.rows.batch);
  const auto threads = [&](int steps) { return dim3((chunks / steps + 31) / 32 * 32); };
  cudaError_t e;
  if (chunks <= 512)
    e = launch_chained(kv8_append_kernel<D, kInt8, 1>, grid, threads(1), 0, stream, p);
  else if (chunks <= 4096)
    e = launch_chained(kv8_append_kernel<D, kInt8, 8>, grid, threads(8), 0, stream, p);
  else
    e = launch_chained(kv8_append_kernel<D, kInt8, 16>, grid, threads(16), 0, stream, p);
  return static_cast<int>(e);
}
template <int D, bool kInt8>
int read(const Kv8StoreParams& p, cudaStream_t stream) {
  const int most = p.rows.tokens + (p.out_rows ? kReadTail : 0);
  return static_cast<int>(launch_chained(
      kv8_read_kernel<D, kInt8>,
      dim3((most + kReadTokens - 1) / kReadTokens, p.cache.heads, p.rows.batch),
      dim3(128), 0, stream, p));
}
}  // namespace

int launch_kv8_append(int d, bool int8, const Kv8StoreParams& p, cudaStream_t stream) {
  if (d == 512) return int8 ? append<512, true>(p, stream) : append<512, false>(p, stream);
  return int8 ? append<256, true>(p, stream) : append<256, false>(p, stream);
}

int launch_kv8_read(int d, bool int8, const Kv8StoreParams& p, cudaStream_t stream) {
  if (d == 512) return int8 ? read<512, true>(p, stream) : read<512, false>(p, stream);
  return int8 ? read<256, true>(p, stream) : read<256, false>(p, stream);
}

int launch_kv8_chunk_plan(const Kv8ChunkParams& p, cudaStream_t stream) {
  return static_cast<int>(
      launch_chained(kv8_chunk_plan_kernel, dim3(1), dim3(1024), 0, stream, p));
}

}  // namespace g4
