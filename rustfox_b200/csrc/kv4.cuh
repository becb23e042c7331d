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

// Rows of sequences: sequence s has the rows row_start[s] ..
// row_start[s+1]-1, standing at the last of its kv_len[s] positions. Both as
// given place them, also where the block table holds fewer positions or the row
// arrays fewer rows: what lies outside is absent, and moves nothing else.
struct Kv4Rows {
  uint8_t* cache;
  const int* table;      // [n_seq][table_stride] pages
  const int* row_start;  // [n_seq + 1]
  const int* kv_len;     // [n_seq]
  int n_pages, n_kv, n_seq, table_stride, n_rows;
  int* err;
};

FOX_DEV void kv4_outside(const Kv4Rows& c) {
  if (c.err) atomicOr(c.err, KERR_PAGES);
}

// The length of sequence s as given, and what a block table holds.
FOX_DEV int kv4_len(const Kv4Rows& c, int s) { return max(__ldg(c.kv_len + s), 0); }
FOX_DEV int kv4_room(const Kv4Rows& c) { return c.table_stride * KV_PAGE; }

// The page of sequence s that holds position p (inside the table), or -1
// (reported) when the table names none of the cache's pages.
FOX_DEV int kv4_page(const Kv4Rows& c, int s, int p) {
  const int page = __ldg(c.table + (size_t)s * c.table_stride + p / KV_PAGE);
  if ((unsigned)page < (unsigned)c.n_pages) return page;
  kv4_outside(c);
  return -1;
}

// A row's page and position in it; page -1 for rows that have none (reported
// where the row stands behind the table's end). The last row reports rows that
// are not there.
struct Kv4Place { int page, at; };
FOX_DEV Kv4Place kv4_place(const Kv4Rows& c, int row) {
  Kv4Place x = {-1, 0};
  if (row == c.n_rows - 1 && __ldg(c.row_start + c.n_seq) > c.n_rows) kv4_outside(c);
  if (row >= c.n_rows || row < __ldg(c.row_start)) return x;
  int lo = 0, hi = c.n_seq;  // sequences that end at or before the row
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (__ldg(c.row_start + mid + 1) <= row) lo = mid + 1; else hi = mid;
  }
  if (lo >= c.n_seq) return x;
  const int pos = kv4_len(c, lo) - (__ldg(c.row_start + lo + 1) - row);
  if (pos < 0) return x;
  if (pos < kv4_room(c)) x.page = kv4_page(c, lo, pos);
  else kv4_outside(c);
  x.at = pos % KV_PAGE;
  return x;
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

// fmaxf and fminf that a NaN goes through.
FOX_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
FOX_DEV float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float KV4_F16_MAX = 65504.0f;

// The code of x: the k that is nearest to (x - m) / d, ties to even. x - m is
// rounded to s (its error e exact, by Knuth's two-sum), but a code near s / d
// leaves r = s - k d without rounding (both lie within d of each other), so
// |r| against d / 2 decides, and e where they are equal.
FOX_DEV float kv4_code(float x, float m, float d, float inv) {
  x = fminf(fmaxf(x, -KV4_F16_MAX), KV4_F16_MAX);
  const float s = __fsub_rn(x, m);
  float k = rintf(s * inv);
  const float r = __fmaf_rn(-k, d, s), half = 0.5f * d;
  if (fabsf(r) > half) {
    k += r > 0.0f ? 1.0f : -1.0f;
  } else if (fabsf(r) == half) {
    const float b = __fsub_rn(x, s), e = __fadd_rn(__fsub_rn(x, __fadd_rn(s, b)), __fsub_rn(b, m));
    const float off = r > 0.0f ? e : -e;  // beyond the border (> 0), short of it, or on it
    if (off > 0.0f || (off == 0.0f && ((int)k & 1))) k += r > 0.0f ? 1.0f : -1.0f;
  }
  return fminf(fmaxf(k, 0.0f), 15.0f);
}

// A group's 64 values over 8 lanes (8 each): its parameters, and this lane's 8
// codes (code i in bits 4i). All parameters are exact:
// - m: rounding down to fp16 is one instruction.
// - d: rounding up nests (to fp32, then to fp16), and a product with 1/15
//   rounded up is at most one fp16 too high, which 15 d' >= span tells.
// - The codes by a product with 1 / d are, too, unless some |r| (kv4_code)
//   reaches d / 2, where the careful form decides.
FOX_DEV uint32_t kv4_quantise(const float (&x)[8], __half2* pair) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) { lo = min_nan(lo, x[i]); hi = max_nan(hi, x[i]); }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (lo != lo) {
    *pair = __half2half2(__ushort_as_half(0x7fff));
    return 0;
  }
  const bool wide = lo < -KV4_F16_MAX || hi > KV4_F16_MAX;
  lo = fminf(fmaxf(lo, -KV4_F16_MAX), KV4_F16_MAX);
  hi = fminf(fmaxf(hi, -KV4_F16_MAX), KV4_F16_MAX);
  const __half m16 = __float2half_rd(lo);
  const float m = __half2float(m16), span = __fsub_ru(hi, m);
  __half d16 = __float2half_ru(__fmul_ru(span, 0x1.111112p-4f));
  const __half less = __ushort_as_half((unsigned short)(__half_as_ushort(d16) - 1));
  if (span > 0.0f && 15.0f * __half2float(less) >= span) d16 = less;
  const float d = __half2float(d16);
  *pair = __halves2half2(d16, m16);
  if (d == 0.0f) return 0;  // one value: every code is 0
  const float inv = __fdividef(1.0f, d), magic = 12582912.0f;  // adding 1.5 * 2^23 rounds to a whole number
  float k[8], far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = __fsub_rn(x[i], m);
    k[i] = __fsub_rn(__fmaf_rn(s, inv, magic), magic);
    far = fmaxf(far, fabsf(__fmaf_rn(-k[i], d, s)));
  }
  if (wide || far >= 0.5f * d) {
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = kv4_code(x[i], m, d, inv);
  }
  const float a = __fmaf_rn(__fmaf_rn(__fmaf_rn(k[3], 16.0f, k[2]), 16.0f, k[1]), 16.0f, k[0]);
  const float b = __fmaf_rn(__fmaf_rn(__fmaf_rn(k[7], 16.0f, k[6]), 16.0f, k[5]), 16.0f, k[4]);
  return (uint32_t)a | (uint32_t)b << 16;
}

// Byte offsets in a block: of the word that holds dimensions d .. d+7 of
// position `at` (K), of the half word of d .. d+3 (V), of a group's
// parameters; each is a sum of a part of the position and one of the dimension.
template <int HD>
struct Kv4Lay {
  static constexpr int SLAB = HD < 128 ? HD : 128, SG = SLAB / 64, NB = SLAB / 32, G = HD / KV4_GROUP;
  static FOX_DEV int k_row(int at) { return at * (SLAB / 2); }
  static FOX_DEV int k_dim(int d) {
    const int r = d % SLAB;
    return d / SLAB * (KV_PAGE * SLAB / 2) + r % 64 / 16 * 8 * SG + 8 * (r / 64) + 4 * (r % 16 / 8);
  }
  static FOX_DEV int v_row(int at) { return at / 2 * (8 * 4 * NB) + 2 * (at & 1); }
  static FOX_DEV int v_dim(int d) {
    const int r = d % SLAB;
    return d / SLAB * (KV_PAGE * SLAB / 2) + r % 32 / 4 * 4 * NB + 4 * (r / 32);
  }
  static FOX_DEV int pair_row(int at) { return kv4_codes_bytes(HD) + at * (4 * G); }
};

// 8 values from and to 16-byte aligned memory.
FOX_DEV void kv4_load8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
FOX_DEV void kv4_load8(const __half* p, float (&v)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
FOX_DEV void kv4_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
FOX_DEV void kv4_store8(__half* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct Kv4MoveParams {
  Kv4Rows c;
  void *k, *v;                // rows to write into the cache, or read back from it
  size_t k_stride, v_stride;  // elements between rows
};

// What a warp moves of each of its rows: pass q of the row, four groups, 8
// lanes each, a lane 8 dimensions. The groups are K and V of two heads (64
// dimensions), of one head (128), or K or V of one head (256).
template <int HD>
struct Kv4Pass {
  static constexpr int G = HD / KV4_GROUP;
  int head, side, d;
  bool live;       // the second head of an odd number's last pass is not
  size_t in_page;  // byte of the lane's block in a page
  int code_dim, code_dim4, pair_dim;
  FOX_DEV Kv4Pass(int q, int n_kv) {
    using Y = Kv4Lay<HD>;
    const int sub = (threadIdx.x & 31) >> 3;
    head = G == 1 ? 2 * q + (sub >> 1) : G == 2 ? q : q >> 1;
    side = G == 1 ? sub & 1 : G == 2 ? sub >> 1 : q & 1;
    live = head < n_kv;
    head = min(head, n_kv - 1);
    d = sub % G * KV4_GROUP + 8 * (threadIdx.x & 7);
    in_page = (size_t)(2 * head + side) * kv4_block_bytes(HD);
    code_dim = side ? Y::v_dim(d) : Y::k_dim(d);
    code_dim4 = Y::v_dim(d + 4);
    pair_dim = 4 * (sub % G);
  }
  static __host__ __device__ constexpr int passes(int n_kv) { return G == 1 ? (n_kv + 1) / 2 : G == 2 ? n_kv : 2 * n_kv; }
};
// A warp's rows: ROWS neighbouring ones, their places found by as many lanes
// at once. Unit u is pass u % passes of rows u / passes * ROWS on.
template <int ROWS>
FOX_DEV Kv4Place kv4_places(const Kv4Rows& c, int row0) {
  const int lane = threadIdx.x & 31;
  Kv4Place x = {-1, 0};
  if (lane < ROWS) x = kv4_place(c, row0 + lane);
  return x;
}

constexpr int KV4_AT_ONCE = 4;  // rows whose loads are in flight together

// Quantises rows into their positions: a group's minimum and maximum over the 8
// lanes that hold it, then every lane's codes. Bound by its instructions, 26 a
// value for the exact codes (28 from fp16, where one warp's groups in twelve hold
// a value on the border of two codes and take the careful form), and by the wait
// for a warp's rows in front of them, which few warps overlap: 4616 fp32 rows of
// 8 heads of 128 take 13.8 us (43 MB of values read and codes written, 3.1 TB/s)
// with 56 % of the issue slots, 32768 65 us (4.7 TB/s), 32768 from fp16 75 us
// (2.3 TB/s, 74 % of the slots). Padding rows are read before it is known that
// they are: 2808 rows among 4616 take 12.1 us. A step's 16 rows take 2.7 us: a
// launch, and the dependent loads of row, length and page.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4MoveParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using Y = Kv4Lay<HD>;
  constexpr int N = ROWS < KV4_AT_ONCE ? ROWS : KV4_AT_ONCE;
  const unsigned unit = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, passes = Kv4Pass<HD>::passes(p.c.n_kv);
  const int row0 = (int)(unit / passes) * ROWS;
  if (row0 >= p.c.n_rows) return;
  const Kv4Pass<HD> pass((int)(unit % passes), p.c.n_kv);
  const T* src = static_cast<const T*>(pass.side ? p.v : p.k) + pass.head * HD + pass.d;
  const size_t stride = pass.side ? p.v_stride : p.k_stride, page_bytes = (size_t)p.c.n_kv * 2 * kv4_block_bytes(HD);
  Kv4Place mine;
#pragma unroll
  for (int r0 = 0; r0 < ROWS; r0 += N) {
    float x[N][8];
#pragma unroll
    for (int i = 0; i < N; ++i) kv4_load8(src + min(row0 + r0 + i, p.c.n_rows - 1) * stride, x[i]);
    if (r0 == 0) mine = kv4_places<ROWS>(p.c, row0);  // while the first rows are on their way
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int page = __shfl_sync(0xffffffffu, mine.page, r0 + i), at = __shfl_sync(0xffffffffu, mine.at, r0 + i);
      if (page < 0) continue;
      __half2 pair;
      const uint32_t code = kv4_quantise(x[i], &pair);
      if (!pass.live) continue;
      uint8_t* block = p.c.cache + page * page_bytes + pass.in_page;
      if (pass.side) {
        uint8_t* dst = block + Y::v_row(at);
        *reinterpret_cast<uint16_t*>(dst + pass.code_dim) = (uint16_t)code;
        *reinterpret_cast<uint16_t*>(dst + pass.code_dim4) = (uint16_t)(code >> 16);
      } else {
        *reinterpret_cast<uint32_t*>(block + Y::k_row(at) + pass.code_dim) = code;
      }
      if ((threadIdx.x & 7) == 0) *reinterpret_cast<__half2*>(block + Y::pair_row(at) + pass.pair_dim) = pair;
    }
  }
}

// 8 codes (code i in bits 4i) as the values they stand for. A code in a half's
// mantissa is a subnormal, c * 2^-22 in bits 2-5 and c * 2^-18 in bits 6-9; d
// takes the power of two back, exactly.
FOX_DEV void kv4_decode(uint32_t code, __half2 pair, float (&v)[8]) {
  const float m = __high2float(pair), d0 = __low2float(pair) * 4194304.0f, d1 = d0 * 0.0625f;
  const uint32_t up = code << 2, down = code >> 6;
  const uint32_t w[4] = {up & 0x003c003cu, up & 0x03c003c0u, down & 0x003c003cu, down & 0x03c003c0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[i] = __fmaf_rn(i % 2 ? d1 : d0, f.x, m);
    v[i + 4] = __fmaf_rn(i % 2 ? d1 : d0, f.y, m);
  }
}

// The rows' values, x = m + d c with one rounding. Bound by its instructions, 15
// a value with their addresses (76 % of the issue slots), before the memory: 32768
// positions of 8 heads of 128 to fp16 take 39 us, 4.4 TB/s, to fp32 64 us, 4.8
// TB/s.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4MoveParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using Y = Kv4Lay<HD>;
  constexpr int N = ROWS < KV4_AT_ONCE ? ROWS : KV4_AT_ONCE;
  const unsigned unit = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, passes = Kv4Pass<HD>::passes(p.c.n_kv);
  const int row0 = (int)(unit / passes) * ROWS;
  if (row0 >= p.c.n_rows) return;
  const Kv4Pass<HD> pass((int)(unit % passes), p.c.n_kv);
  const Kv4Place mine = kv4_places<ROWS>(p.c, row0);
  const size_t page_bytes = (size_t)p.c.n_kv * 2 * kv4_block_bytes(HD);
  T* dst = static_cast<T*>(pass.side ? p.v : p.k) + ((size_t)row0 * p.c.n_kv + pass.head) * HD + pass.d;
#pragma unroll
  for (int r0 = 0; r0 < ROWS; r0 += N) {
    uint32_t code[N];
    __half2 pair[N];
    bool there[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int page = __shfl_sync(0xffffffffu, mine.page, r0 + i), at = __shfl_sync(0xffffffffu, mine.at, r0 + i);
      there[i] = page >= 0 && pass.live;
      const uint8_t* block = p.c.cache + max(page, 0) * page_bytes + pass.in_page;
      if (!there[i]) continue;
      if (pass.side) {
        const uint8_t* from = block + Y::v_row(at);
        code[i] = *reinterpret_cast<const uint16_t*>(from + pass.code_dim) |
                  (uint32_t) * reinterpret_cast<const uint16_t*>(from + pass.code_dim4) << 16;
      } else {
        code[i] = *reinterpret_cast<const uint32_t*>(block + Y::k_row(at) + pass.code_dim);
      }
      pair[i] = *reinterpret_cast<const __half2*>(block + Y::pair_row(at) + pass.pair_dim);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!there[i]) continue;
      float v[8];
      kv4_decode(code[i], pair[i], v);
      kv4_store8(dst + (size_t)(r0 + i) * p.c.n_kv * HD, v);
    }
  }
}

struct RopeParams {
  const void* x;  // rows of n_head query heads, then n_kv key heads
  const int* pos;
  const float *q_norm, *k_norm;  // [hd], or null: no norm
  const float *cos, *sin;        // [n_pos][hd / 2]
  void *q, *k;
  size_t x_stride, q_stride, k_stride;
  int n_rows, n_head, n_kv, n_pos;
  float eps;
  int* err;
};

// E neighbouring values as they lie in memory, and as floats.
template <typename T, int E>
struct RopeVec {
  uint4 u[E * sizeof(T) / 16];
  FOX_DEV void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  FOX_DEV void get(float (&v)[E]) const {
#pragma unroll
    for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          v[4 * i + j] = __uint_as_float(w[j]);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          v[2 * j] = f.x; v[2 * j + 1] = f.y;
        }
      }
    }
  }
};
template <int E>
FOX_DEV void rope_store(float* p, const float (&v)[E]) {
#pragma unroll
  for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
FOX_DEV void rope_store(__half* p, const float (&v)[8]) { kv4_store8(p, v); }

// RMSNorm of every query and key head and the rotation of its position:
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w
//   (a, b) -> (a cos - b sin, a sin + b cos) for the pairs (2i, 2i+1), or
//   (i, i + hd/2) with HALVES.
// A lane holds E neighbouring dimensions of a head (16 bytes, or 32 of 256
// fp32 dimensions), so the pairs lie in a lane and the halves LANES / 2 lanes
// apart. A warp takes BATCH such loads of one row's query or key heads, so that
// the row's sines, cosines and the weights are loaded once for all of them and
// the loads are in flight together. Without norms the result is that of the
// decode step's rotation, bit for bit. fp32 rows are bound by memory: 4096 of 32 +
// 8 heads of 128 take 28 us, 6.1 TB/s. fp16 rows, with twice the arithmetic a
// byte, are bound by their instructions (66 % of the issue slots, the rest waits
// for loads and exchanges): 4096 of 32 + 16 heads take 23 us, 4.5 TB/s. 1 to 100
// rows take 1.6 us, a launch.
template <typename T, int HD>
struct RopeLay {
  static constexpr int E = sizeof(T) == 2 || HD == 256 ? 8 : 4, LANES = HD / E, AT_ONCE = 32 / LANES;
  static __host__ __device__ int chunks(int heads, int batch) { return (heads + AT_ONCE * batch - 1) / (AT_ONCE * batch); }
};
template <typename T, int HD, bool HALVES, int BATCH>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const RopeParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using Y = RopeLay<T, HD>;
  constexpr int E = Y::E, LANES = Y::LANES, AT_ONCE = Y::AT_ONCE, C = HALVES ? E : E / 2;
  const int lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES;
  const int q_chunks = Y::chunks(p.n_head, BATCH), chunks = q_chunks + Y::chunks(p.n_kv, BATCH);
  const unsigned unit = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;  // below 2^20 rows * 2^11 chunks
  const int row = (int)(unit / chunks), chunk = (int)(unit - row * chunks);
  if (row >= p.n_rows) return;
  const bool is_q = chunk < q_chunks;
  const int heads = is_q ? p.n_head : p.n_kv, h0 = (is_q ? chunk : chunk - q_chunks) * (AT_ONCE * BATCH) + sub;
  const int pos = __ldg(p.pos + row);
  if (pos < 0) return;
  const T* x = static_cast<const T*>(p.x) + (size_t)row * p.x_stride + (size_t)(is_q ? 0 : p.n_head) * HD + l * E;
  RopeVec<T, E> raw[BATCH];
#pragma unroll
  for (int b = 0; b < BATCH; ++b) raw[b].load(x + (size_t)min(h0 + b * AT_ONCE, heads - 1) * HD);
  if (pos >= p.n_pos) {
    if (lane == 0 && p.err) atomicOr(p.err, KERR_PAGES);
    return;
  }
  float cs[C], sn[C];
  {
    const int i0 = HALVES ? l % (LANES / 2) * E : l * (E / 2);
    const float *c = p.cos + (size_t)pos * (HD / 2) + i0, *s = p.sin + (size_t)pos * (HD / 2) + i0;
#pragma unroll
    for (int i = 0; i < C; i += 2) {
      const float2 a = __ldg(reinterpret_cast<const float2*>(c + i)), b = __ldg(reinterpret_cast<const float2*>(s + i));
      cs[i] = a.x; cs[i + 1] = a.y; sn[i] = b.x; sn[i + 1] = b.y;
    }
  }
  const float* norm = is_q ? p.q_norm : p.k_norm;
  float w[E];
  if (norm) {
    RopeVec<float, E> f;
    f.load(norm + l * E);
    f.get(w);
  }
  T* out = is_q ? static_cast<T*>(p.q) + (size_t)row * p.q_stride : static_cast<T*>(p.k) + (size_t)row * p.k_stride;
  out += l * E;
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    const int h = h0 + b * AT_ONCE;
    float v[E];
    raw[b].get(v);
    if (norm) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float mean = fmaf(ss, 1.0f / HD, p.eps);
      float scale = rsqrtf(mean);
      scale = fmaf(0.5f * scale, fmaf(-mean * scale, scale, 1.0f), scale);  // a Newton step: the last bits
      // (an infinite mean, or zero with no eps, has nothing to refine)
      if (!(mean > 0.0f) || isinf(mean)) scale = rsqrtf(mean);
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], scale), w[i]);
    }
    float o[E];
    if (HALVES) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, v[i], LANES / 2);
        o[i] = l < LANES / 2 ? __fsub_rn(__fmul_rn(v[i], cs[i]), __fmul_rn(other, sn[i]))
                             : __fadd_rn(__fmul_rn(other, sn[i]), __fmul_rn(v[i], cs[i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        o[i] = __fsub_rn(__fmul_rn(v[i], cs[i / 2]), __fmul_rn(v[i + 1], sn[i / 2]));
        o[i + 1] = __fadd_rn(__fmul_rn(v[i], sn[i / 2]), __fmul_rn(v[i + 1], cs[i / 2]));
      }
    }
    if (h < heads) rope_store(out + (size_t)h * HD, o);
  }
}

}  // namespace fox
