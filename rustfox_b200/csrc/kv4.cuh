// A paged K/V cache held in 4 bits: its format, the kernels that write rows
// into it and read them back, and the norms and rotation of the queries and
// keys on their way there (sm_100a). Upstream keeps an fp32 cache per context
// (src/forward.c:91-92) and has no counterpart.
//
// Format. The cache is [page][kv_head][K block | V block]; a page holds
// KV_PAGE = 64 positions. A block holds the 64 x hd codes (0..15), then for
// each position and group of 64 dimensions the fp16 pair (d, m) of
//   x = m + d * code:   36 * hd bytes, 4.5 bits a value.
// m is the largest fp16 not above the group's minimum and d the smallest fp16
// with m + 15 d not below its maximum, so every value of the group lies
// between the first and the last level and is at most d / 2 from its own. The
// code is the nearest level (ties to even), decided without rounding. Values
// beyond fp16's range are taken as its largest; a group that holds a NaN
// reads back as NaN.
//
// The codes lie where the attention's matrix instructions want them
// (kv4_attn.cuh), so a lane's fragment is a vector load and two masks:
// - K: a position's codes are words of 8 dimensions (nibble i = dimension i),
//   in the order (slab of 128 dimensions; position; t; group; w) for
//   dimension = slab * 128 + group * 64 + t * 16 + w * 8 + i.
// - V: a word holds 4 dimensions of a pair of positions, the even one in the
//   low half: order (slab; step; half; t; g; b) for position =
//   step * 16 + half * 8 + t * 2 + parity and dimension = slab * 128 + b * 32
//   + g * 4 + i. A position owns whole 16-bit halves, so no two rows write
//   to one of them.
#pragma once

#include "common.cuh"
#include "host.cuh"

namespace fox {

constexpr int KV4_GROUP = 64;
__host__ __device__ constexpr int kv4_block_bytes(int hd) { return KV_PAGE * (hd / 2 + 4 * (hd / KV4_GROUP)); }
__host__ __device__ constexpr int kv4_codes_bytes(int hd) { return KV_PAGE * hd / 2; }

// Byte of the 16 bits that hold dimensions d..d+3 (d a multiple of 4) of
// position p in a block.
template <int HD>
FOX_DEV int kv4_k_at(int p, int d) {
  constexpr int SLAB = HD < 128 ? HD : 128, G = SLAB / 64;
  const int r = d % SLAB;
  return (d / SLAB) * (KV_PAGE * SLAB / 2) + p * (SLAB / 2) +
         4 * ((r % 64 / 16) * 2 * G + 2 * (r / 64) + (r % 16) / 8) + (r % 8) / 2;
}
template <int HD>
FOX_DEV int kv4_v_at(int p, int d) {
  constexpr int SLAB = HD < 128 ? HD : 128, NB = SLAB / 32;
  const int r = d % SLAB;
  const int at = ((((d / SLAB) * 4 + p / 16) * 2 + (p / 8) % 2) * 4 + (p % 8) / 2) * 8 + (r % 32) / 4;
  return 4 * (at * NB + r / 32) + 2 * (p % 2);
}

// Rows of sequences: sequence s has the rows row_start[s] ..
// row_start[s+1]-1, standing at the last of its kv_len[s] cached positions.
struct Kv4Rows {
  uint8_t* cache;
  const int* table;      // [n_seq][table_stride] pages
  const int* row_start;  // [n_seq + 1]
  const int* kv_len;     // [n_seq]
  int n_pages, n_kv, n_seq, table_stride, n_rows;
  int* err;
};

// The sequence of a row (all lanes of a warp ask for the same row): the
// number of sequences that end at or before it. One round of loads for every
// 32 sequences. n_seq for a padding row.
FOX_DEV int kv4_seq_of(const Kv4Rows& c, int row) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int s = 0; s < c.n_seq; s += 32) {
    const bool past = s + lane < c.n_seq && __ldg(c.row_start + s + lane + 1) <= row;
    n += __popc(__ballot_sync(0xffffffffu, past));
  }
  return n;
}

// Cached positions of sequence s, held to its block table (an overrun is
// reported once per call of this).
FOX_DEV int kv4_len(const Kv4Rows& c, int s) {
  const int L = __ldg(c.kv_len + s), most = c.table_stride * KV_PAGE;
  if (L > most && c.err) atomicExch(c.err, KERR_PAGES);
  return min(max(L, 0), most);
}

// The page of sequence s that holds position p (inside the table), or -1
// (reported) when the table names none of the cache's pages.
FOX_DEV int kv4_page(const Kv4Rows& c, int s, int p) {
  const int page = __ldg(c.table + (size_t)s * c.table_stride + p / KV_PAGE);
  if ((unsigned)page < (unsigned)c.n_pages) return page;
  if (c.err) atomicExch(c.err, KERR_PAGES);
  return -1;
}

// The row's page and position in it; false for rows that have none.
FOX_DEV bool kv4_place(const Kv4Rows& c, int row, int* page, int* at) {
  const int s = kv4_seq_of(c, row);
  if (s >= c.n_seq) return false;
  const int pos = kv4_len(c, s) - (__ldg(c.row_start + s + 1) - row);
  if (pos < 0) return false;
  *page = kv4_page(c, s, pos);
  *at = pos % KV_PAGE;
  return *page >= 0;
}

FOX_DEV uint8_t* kv4_block(const Kv4Rows& c, int page, int head, int side, int block_bytes) {
  return c.cache + (((size_t)page * c.n_kv + head) * 2 + side) * block_bytes;
}

// 4 values from 16-byte aligned floats or 8-byte aligned halves.
FOX_DEV float4 kv4_load4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
FOX_DEV float4 kv4_load4(const __half* p) {
  const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
FOX_DEV void kv4_store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
FOX_DEV void kv4_store4(__half* p, float4 v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// The code of x: the k that is nearest to (x - m) / d, ties to even. x - m is
// rounded to s (its error e exact, by Knuth's two-sum), but a code near s / d
// leaves r = s - k d without rounding (both lie within d of each other), so
// |r| against d / 2 decides, and e where they are equal.
FOX_DEV uint32_t kv4_code(float x, float m, float d, float inv) {
  const float s = __fsub_rn(x, m);
  float k = rintf(s * inv);
  const float r = __fmaf_rn(-k, d, s), half = 0.5f * d;
  if (fabsf(r) >= half) {
    if (fabsf(r) > half) {
      k += r > 0.0f ? 1.0f : -1.0f;
    } else {
      const float b = __fsub_rn(x, s), e = __fadd_rn(__fsub_rn(x, __fadd_rn(s, b)), __fsub_rn(b, m));
      const float off = r > 0.0f ? e : -e;  // beyond the border (> 0), short of it, or on it
      if (off > 0.0f || (off == 0.0f && ((int)k & 1))) k += r > 0.0f ? 1.0f : -1.0f;
    }
  }
  return (uint32_t)(int)fminf(fmaxf(k, 0.0f), 15.0f);
}

// The group's parameters from its least and largest value. Directed
// roundings nest: rounding up to fp32 and then to fp16 is rounding up to fp16.
FOX_DEV __half2 kv4_pair(float lo, float hi, bool nan) {
  if (nan) return __half2half2(__ushort_as_half(0x7fff));
  const __half m = __float2half_rd(lo);
  const __half d = __float2half_ru(__fdiv_ru(__fsub_ru(hi, __half2float(m)), 15.0f));
  return __halves2half2(d, m);
}

// A group's 64 values over 16 lanes (4 each): its parameters, and this lane's
// 4 codes as 16 bits.
FOX_DEV uint32_t kv4_quantise(float4 x, __half2* pair) {
  constexpr float kMax = 65504.0f;
  bool nan = x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w;
  x = make_float4(fminf(fmaxf(x.x, -kMax), kMax), fminf(fmaxf(x.y, -kMax), kMax), fminf(fmaxf(x.z, -kMax), kMax),
                  fminf(fmaxf(x.w, -kMax), kMax));
  float lo = fminf(fminf(x.x, x.y), fminf(x.z, x.w)), hi = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const uint32_t any = __ballot_sync(0xffffffffu, nan);
  nan = (any >> (threadIdx.x & 16)) & 0xffffu;
  *pair = kv4_pair(lo, hi, nan);
  const float d = __low2float(*pair), m = __high2float(*pair);
  if (!(d > 0.0f)) return 0;  // one value (or a NaN): every code is 0
  const float inv = __fdiv_rn(1.0f, d);
  return kv4_code(x.x, m, d, inv) | kv4_code(x.y, m, d, inv) << 4 | kv4_code(x.z, m, d, inv) << 8 |
         kv4_code(x.w, m, d, inv) << 12;
}

struct Kv4WriteParams {
  Kv4Rows c;
  const void *k, *v;
  size_t k_stride, v_stride;  // elements between rows
};

// One warp quantises a row's K and V of one head: 16 lanes a group.
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4WriteParams p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int G = HD / KV4_GROUP, BB = kv4_block_bytes(HD);
  const int lane = threadIdx.x & 31;
  const size_t unit = blockIdx.x * (size_t)(blockDim.x / 32) + threadIdx.x / 32;
  if (unit >= (size_t)p.c.n_rows * p.c.n_kv) return;
  const int row = (int)(unit / p.c.n_kv), head = (int)(unit - (size_t)row * p.c.n_kv);
  int page, at;
  if (!kv4_place(p.c, row, &page, &at)) return;
  const T* src[2] = {static_cast<const T*>(p.k) + row * p.k_stride + head * HD,
                     static_cast<const T*>(p.v) + row * p.v_stride + head * HD};
  uint8_t* block = kv4_block(p.c, page, head, 0, BB);
  // 2 G groups of 64 dimensions: K's, then V's; each half warp takes one
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int u = 2 * i + (lane >> 4), side = u / G, g = u % G, d = g * KV4_GROUP + 4 * (lane & 15);
    __half2 pair;
    const uint32_t code = kv4_quantise(kv4_load4(src[side] + d), &pair);
    uint8_t* b = block + side * BB;
    *reinterpret_cast<uint16_t*>(b + (side ? kv4_v_at<HD>(at, d) : kv4_k_at<HD>(at, d))) = (uint16_t)code;
    if ((lane & 15) == 0) *reinterpret_cast<__half2*>(b + kv4_codes_bytes(HD) + 4 * (at * G + g)) = pair;
  }
}

struct Kv4ReadParams {
  Kv4Rows c;
  void *k, *v;
};

FOX_DEV float4 kv4_decode(uint32_t code, __half2 pair) {
  const float d = __low2float(pair), m = __high2float(pair);
  return make_float4(__fmaf_rn(d, (float)(code & 15), m), __fmaf_rn(d, (float)(code >> 4 & 15), m),
                     __fmaf_rn(d, (float)(code >> 8 & 15), m), __fmaf_rn(d, (float)(code >> 12 & 15), m));
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int G = HD / KV4_GROUP, BB = kv4_block_bytes(HD);
  const int lane = threadIdx.x & 31;
  const size_t unit = blockIdx.x * (size_t)(blockDim.x / 32) + threadIdx.x / 32;
  if (unit >= (size_t)p.c.n_rows * p.c.n_kv) return;
  const int row = (int)(unit / p.c.n_kv), head = (int)(unit - (size_t)row * p.c.n_kv);
  int page, at;
  if (!kv4_place(p.c, row, &page, &at)) return;
  const uint8_t* block = kv4_block(p.c, page, head, 0, BB);
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int u = 2 * i + (lane >> 4), side = u / G, g = u % G, d = g * KV4_GROUP + 4 * (lane & 15);
    const uint8_t* b = block + side * BB;
    const uint32_t code = *reinterpret_cast<const uint16_t*>(b + (side ? kv4_v_at<HD>(at, d) : kv4_k_at<HD>(at, d)));
    const __half2 pair = *reinterpret_cast<const __half2*>(b + kv4_codes_bytes(HD) + 4 * (at * G + g));
    T* out = static_cast<T*>(side ? p.v : p.k) + unit * HD + d;
    kv4_store4(out, kv4_decode(code, pair));
  }
}

struct RopeParams {
  const void* x;  // rows of n_head query heads, then n_kv key heads
  const int* pos;
  const float *q_norm, *k_norm;  // [hd], or null: no norm
  const float *cos, *sin;        // [n_pos][hd / 2]
  void *q, *k;
  size_t x_stride, q_stride, k_stride;
  int n_rows, n_head, n_kv, n_pos, halves;
  float eps;
  int* err;
};

// RMSNorm of every query and key head and the rotation of its position:
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w
//   (a, b) -> (a cos - b sin, a sin + b cos) for the pairs (2i, 2i+1), or
//   (i, i + hd/2) when halves is set.
// One warp a head: a lane holds HD/32 neighbouring dimensions, so the pairs
// lie in a lane and the halves 16 lanes apart. Without norms the result is
// that of the decode step's rotation, bit for bit.
template <typename T, int HD>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const RopeParams p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31, heads = p.n_head + p.n_kv;
  const size_t unit = blockIdx.x * (size_t)(blockDim.x / 32) + threadIdx.x / 32;
  if (unit >= (size_t)p.n_rows * heads) return;
  const int row = (int)(unit / heads), h = (int)(unit - (size_t)row * heads);
  const int pos = __ldg(p.pos + row);
  if (pos < 0) return;
  if (pos >= p.n_pos) {
    if (lane == 0 && p.err) atomicExch(p.err, KERR_PAGES);
    return;
  }
  const bool is_q = h < p.n_head;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + (size_t)h * HD + lane * E;
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = (float)x[i];
  const float* w = is_q ? p.q_norm : p.k_norm;
  if (w) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) ss = fmaf(v[i], v[i], ss);
    const float scale = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(warp_sum(ss), (float)HD), p.eps)));
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], scale), __ldg(w + lane * E + i));
  }
  const float* cs = p.cos + (size_t)pos * (HD / 2);
  const float* sn = p.sin + (size_t)pos * (HD / 2);
  float o[E];
  if (p.halves) {
    const int i0 = (lane & 15) * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, v[i], 16);
      const float c = __ldg(cs + i0 + i), s = __ldg(sn + i0 + i);
      o[i] = lane < 16 ? __fsub_rn(__fmul_rn(v[i], c), __fmul_rn(other, s))
                       : __fadd_rn(__fmul_rn(other, s), __fmul_rn(v[i], c));
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float c = __ldg(cs + (lane * E + i) / 2), s = __ldg(sn + (lane * E + i) / 2);
      o[i] = __fsub_rn(__fmul_rn(v[i], c), __fmul_rn(v[i + 1], s));
      o[i + 1] = __fadd_rn(__fmul_rn(v[i], s), __fmul_rn(v[i + 1], c));
    }
  }
  T* out = is_q ? static_cast<T*>(p.q) + row * p.q_stride + (size_t)h * HD
                : static_cast<T*>(p.k) + row * p.k_stride + (size_t)(h - p.n_head) * HD;
#pragma unroll
  for (int i = 0; i < E; ++i) out[lane * E + i] = (T)o[i];
}

}  // namespace fox
