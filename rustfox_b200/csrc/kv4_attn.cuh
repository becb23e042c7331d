// Attention over the 4-bit K/V cache of kv4.cuh (sm_100a).
//
// With x = m + d c for each group g of 64 dimensions,
//   s_j = scale * q . k_j = scale * sum_g (d_jg * (q_g . c_jg) + m_jg * sum(q_g))
//   p_j = 2^(s_j log2 e - M), l = sum_j p_j       (M the running maximum)
//   o_d = (sum_j (p_j d_jg) c_jd + sum_j p_j m_jg) / l
// so the codes enter both products as they are, and the matrix instructions
// (m16n8k16, fp16 in, fp32 sums) take them without a conversion: the 4 bits
// placed in a half's mantissa are a subnormal, c * 2^-22 in bits 2-5 and
// c * 2^-18 in bits 6-9. A 32-bit word of 8 codes becomes 4 operand registers
// by two shifts and four masks; the powers of two go into the other operand
// (K) or the result (V). (Bits 0-3 and 4-7 need one shift less, but products
// are aligned by the subnormal's nominal exponent before they are summed, and
// the leading zeros cost their low bits: 4e-6 of the result.)
//
// The codes are the 16-row operand (positions for K, dimensions for V), the
// columns hold query rows: a pair (row, head) takes two, the halves of q (and
// of p d) as hi + lo fp16, 22 bits, so the sums are near fp32's.
// - q is scaled by a power of two to [2^13, 2^14) before it is split, p d by
//   one (of the largest d seen) to at most 2^15: neither end of fp16's range
//   is met.
// - The scores of a 16-position step come out as (position, pair) per lane:
//   the softmax needs no exchange but the maximum's, and 8x8 transposes turn
//   its weights into the second product's operand.
// - Every second position of V is taken from its top level down, x = (m + 15
//   d) - d (15 - c), with the complement of the code (an xor that joins the
//   mask) and a negated weight, alternating within an operand and within what
//   a lane sums: both sums then stay near the result instead of 7.5 d away
//   from it. What cancels in the end must not pass through them: with all
//   positions counted from below the error was 1e-4 of the result at 32768
//   positions, now it is 1e-6.
//
// Bound by memory for long single tokens, with the issue of instructions close
// behind: 16 sequences of 32768 positions, 32 heads over 8 of 128, take 120 us,
// 5.0 TB/s of codes and parameters; 64 ragged fp16 ones over 16 KV heads 128 us,
// 4.7 TB/s. Short ones are bound by their chain of dependent loads (row, length,
// page, codes) and the launch: 576 positions 11 us, 65 positions 8 us. With many
// rows the products and the weights of every row bound it: 32 (row, head) pairs
// for each of 8 KV heads, 4 sequences of 8192 positions, 69 us; from 48 pairs on
// the tiles of kv4_wide.cuh are faster.
#pragma once

#include <cfloat>
#include <climits>

#include "kv4.cuh"

namespace fox {

constexpr int KV4_MAX_SEQ = 1024;

struct Kv4AttnParams {
  Kv4Rows c;
  const void* q;
  void* out;
  float* part;          // workspace: pieces of runs split between CTAs
  size_t q_stride;      // elements between rows
  int n_head, ctas;
  float scale;
};

// How the work is divided. A tile is PAIRS (row, head) pairs of one KV head of
// a sequence, a run all the pages of its sequence. The runs stand in a line
// (sequence, tile, KV head); every CTA takes an equal stretch of it, and every
// warp an equal stretch of its CTA's, so the load is even whatever the lengths
// and no warp waits for another before its end. A warp's stretch holds whole
// runs, whose results it writes, and at most two pieces: the end of one run and
// the beginning of another. The CTA joins its warps' pieces in shared memory,
// and a second kernel joins, in order, the CTAs' pieces of runs that are split
// between CTAs. That launch costs more than a few pages' work: a line without
// a run of more than KV4_WHOLE pages is divided between runs, and no second
// kernel follows where the block tables hold no more.
constexpr int KV4_WHOLE = 16;
// A run begins with KV4_HEAD units without a page: what its queries' loading
// and its results' writing take of a worker's time.
constexpr int KV4_HEAD = 2;
// Rows r0 .. r0 + T - 1, the first at position at (negative: it has none), and
// the L positions that the block table holds.
struct Kv4Seq { int r0, T, at, L, tiles, units; };

template <int PAIRS>
FOX_DEV Kv4Seq kv4_seq(const Kv4AttnParams& p, int s) {
  Kv4Seq q;
  q.r0 = min(max(__ldg(p.c.row_start + s), 0), p.c.n_rows);
  const int end = max(__ldg(p.c.row_start + s + 1), q.r0), len = kv4_len(p.c, s);
  q.T = min(end, p.c.n_rows) - q.r0;
  q.at = len - (end - q.r0);
  q.L = min(len, kv4_room(p.c));
  q.tiles = (q.T * (p.n_head / p.c.n_kv) + PAIRS - 1) / PAIRS;
  q.units = KV4_HEAD + (q.L + KV_PAGE - 1) / KV_PAGE;
  return q;
}

// n things in `parts` nearly equal stretches. The host keeps every count of
// units below 2^31.
struct Kv4Split {
  int base, rem;
  FOX_DEV Kv4Split(int n, int parts) : base(n / parts), rem(n - n / parts * parts) {}
  FOX_DEV int first(int i) const { return i * base + min(i, rem); }
  FOX_DEV int owner(int u) const {
    const int wide = rem * (base + 1);
    return u < wide ? u / (base + 1) : rem + (u - wide) / base;
  }
};

// The line: the first unit and run of each sequence (n_seq + 1 each, then the
// longest sequence's units), in shared memory.
struct Kv4Line {
  int *unit0, *run0;
  int U, runs, n_seq;
  bool whole;  // no run is split between CTAs
  static __host__ __device__ int bytes(int n_seq) { return (2 * n_seq + 3) * 4; }

  // By the CTA's first warp; every thread calls. Lengths beyond the block table
  // and rows beyond the row arrays are reported here. A row_start that falls
  // could count rows twice and the units past 2^31: it leaves the line empty.
  template <int PAIRS>
  FOX_DEV void build(const Kv4AttnParams& p, void* mem) {
    n_seq = p.c.n_seq;
    unit0 = static_cast<int*>(mem);
    run0 = unit0 + n_seq + 1;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
      int r0 = 0, u0 = 0, longest = 0;
      bool outside = false, falls = false;
      for (int s0 = 0; s0 < n_seq; s0 += 32) {
        const int s = s0 + lane;
        int r = 0, n = 0;
        if (s < n_seq) {
          const Kv4Seq q = kv4_seq<PAIRS>(p, s);
          const int end = __ldg(p.c.row_start + s + 1);
          falls = falls || end < __ldg(p.c.row_start + s);
          outside = outside || falls || end > p.c.n_rows || kv4_len(p.c, s) > q.L;
          r = q.tiles * p.c.n_kv;
          n = r * q.units;
          if (r) longest = max(longest, q.units);
        }
        int rs = r, ns = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int ru = __shfl_up_sync(0xffffffffu, rs, o), nu = __shfl_up_sync(0xffffffffu, ns, o);
          if (lane >= o) { rs += ru; ns += nu; }
        }
        if (s < n_seq) { run0[s] = r0 + rs - r; unit0[s] = u0 + ns - n; }
        r0 += __shfl_sync(0xffffffffu, rs, 31);
        u0 += __shfl_sync(0xffffffffu, ns, 31);
        if (__any_sync(0xffffffffu, falls)) {
          r0 = u0 = 0;
          break;
        }
      }
      if (outside) kv4_outside(p.c);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
      if (lane == 0) { run0[n_seq] = r0; unit0[n_seq] = u0; run0[n_seq + 1] = longest; }
    }
    __syncthreads();
    runs = run0[n_seq];
    U = unit0[n_seq];
    whole = run0[n_seq + 1] <= KV4_HEAD + KV4_WHOLE;
  }
  // The last sequence that begins at or before x (sequences without runs take
  // no room, so it is the one that holds x).
  FOX_DEV int find(const int* start, int x) const {
    int lo = 0, hi = n_seq - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (start[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
  FOX_DEV int ctas(int most) const { return min(most, whole ? runs : U / 2); }
};

FOX_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
FOX_DEV void mma16816_0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
FOX_DEV uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
FOX_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
FOX_DEV uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// (x & mask) ^ flip in one instruction, flip from a register.
template <uint32_t MASK>
FOX_DEV uint32_t kv4_pick(uint32_t x, uint32_t flip) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(x), "n"(MASK), "r"(flip));
  return r;
}
constexpr uint32_t KV4_E = 0x003c003cu, KV4_O = 0x03c003c0u;
// 8 codes of a word (nibble i in bits 4i) as four operand registers: codes
// (0, 4), (1, 5), (2, 6), (3, 7), the even ones as c * 2^-22, the odd ones as
// c * 2^-18; flip_e and flip_o: the masks' bits in the halves whose codes are
// complemented.
FOX_DEV void kv4_operands(uint32_t x, uint32_t (&a)[4]) {
  const uint32_t up = x << 2, down = x >> 6;
  a[0] = up & KV4_E;
  a[1] = up & KV4_O;
  a[2] = down & KV4_E;
  a[3] = down & KV4_O;
}
FOX_DEV void kv4_operands(uint32_t x, uint32_t flip_e, uint32_t flip_o, uint32_t (&a)[4]) {
  const uint32_t up = x << 2, down = x >> 6;
  a[0] = kv4_pick<KV4_E>(up, flip_e);
  a[1] = kv4_pick<KV4_O>(up, flip_o);
  a[2] = kv4_pick<KV4_E>(down, flip_e);
  a[3] = kv4_pick<KV4_O>(down, flip_o);
}
constexpr float KV4_EVEN = 4194304.0f;  // 2^22
constexpr int KV4_FLUSH = 4;  // pages whose sums stay in the matrix instructions' registers
// Sums of a query's dimensions are held at this, so that no finite ones pass
// fp32's range; what takes the scores of large queries back is held to it too.
constexpr float KV4_QSUM = 1.0f / 64.0f;
// A weight may exceed 1 by 2^SLACK before the sums are rescaled; times d it is
// scaled to at most 2^15.
constexpr float KV4_SLACK = 7.0f, KV4_WEIGHT = 256.0f;
// x as hi + lo fp16: hi keeps the leading 11 bits.
FOX_DEV uint32_t kv4_hi_lo(float x) {
  const float hi = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
  return half2_bits(__floats2half2_rn(hi, x - hi));
}

// A unit in line: page `page` of a run, or its head (negative).
struct Kv4Unit {
  Kv4Seq q;
  int seq, run, tile, kv, page;
};

FOX_DEV float4 kv4_quotient(float4 v, float l) {
  if (l == 0.0f) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // nothing to see
  return make_float4(__fdiv_rn(v.x, l), __fdiv_rn(v.y, l), __fdiv_rn(v.z, l), __fdiv_rn(v.w, l));
}

// Pieces of a pair's results joined one after the other: M, l and, of the
// sums, dimensions lane, lane + 32, ...
template <int HD>
struct Kv4Sum {
  float M = -INFINITY, l = 0.0f, v[HD / 32] = {};
  FOX_DEV void add(float m, float lm, const float (&x)[HD / 32]) {
    if (m == -INFINITY && lm == 0.0f) return;  // a piece that saw nothing
    const float to = fmaxf(M, m), old = M == -INFINITY ? 0.0f : exp2_approx(M - to), by = exp2_approx(m - to);
    M = to;
    l = fmaf(l, old, lm * by);
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) v[e] = fmaf(v[e], old, x[e] * by);
  }
  FOX_DEV void add(const float* piece) {
    const float2 ml = *reinterpret_cast<const float2*>(piece);
    float x[HD / 32];
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) x[e] = piece[4 + e * 32 + (threadIdx.x & 31)];
    add(ml.x, ml.y, x);
  }
  template <typename T>
  FOX_DEV void store(T* out) const {
#pragma unroll
    for (int e = 0; e < HD / 32; ++e)
      out[e * 32 + (threadIdx.x & 31)] = (T)(l == 0.0f ? 0.0f : __fdiv_rn(v[e], l));
  }
};

// HD: head dimension.
template <int HD>
struct Kv4Attn {
  static constexpr int SLAB = HD < 128 ? HD : 128, SLABS = HD / SLAB, SG = SLAB / 64, NB = SLAB / 32;
  static constexpr int G = HD / KV4_GROUP, BB = kv4_block_bytes(HD), PAGE_BYTES = 2 * BB;
  static constexpr int PAIRS = 4;            // (row, head) pairs of a tile
  static constexpr int SUM_VECS = SLABS * NB * 2;  // float4s of a lane's sums
  static constexpr int PART = HD + 4;        // floats of one pair's partial result: M, l, -, -, sums
  // warps of a CTA: what the registers (and for 256 dimensions shared memory)
  // hold. Each has room for a page's K and V, then for a piece of a run; for
  // its flushed sums; and for the piece it may end before that.
  static constexpr int NW = HD < 256 ? 12 : 7, PIECE_BYTES = PAIRS * PART * 4;
  static_assert(PIECE_BYTES <= PAGE_BYTES && PIECE_BYTES % 16 == 0, "a piece fits the ring");
  static constexpr size_t smem_bytes(int n_seq) {
    return (size_t)NW * (PAGE_BYTES + SUM_VECS * 512 + PIECE_BYTES) + NW * 2 * 8 + NW * 2 * 4 + Kv4Line::bytes(n_seq);
  }

  // A warp's share of a tile: q's operand registers, and the running maximum,
  // weights and sums of its pairs. Lane (g, t) = (lane / 4, lane % 4) holds
  // the scores of pair t at positions g and g + 8 of a step, and pair t's sums of
  // dimensions 4g .. 4g+3 of each block of 32.
  uint32_t qb[SLABS][SG][2][2][2];
  float f, qs[G];  // score = f * sum_g (d_g * product) + sum_g m_g * qs_g, in powers of 2
  float o[SLABS][NB][2][4], mx, l, mo[G], big;
  // The matrix instructions round their sums toward zero, 0.7 * 2^-24 of them
  // each time, so after KV4_FLUSH pages they move to shared memory (this
  // lane's float4s, 32 apart), added to the nearest. `flushed`: there are any.
  float4* sums;
  bool flushed;
  float sco[4][2];            // the page's scores
  int lim, lim_min, lim_max;  // the last position pair t sees (negative: none), and over the tile

  // The last position that any row of a tile sees.
  static FOX_DEV int last_seen(const Kv4Seq& q, int tile, int gqa) {
    return q.at + min(q.T - 1, (tile * PAIRS + PAIRS - 1) / gqa);
  }

  template <typename T>
  FOX_DEV void begin(const Kv4AttnParams& p, const Kv4Unit& it, int gqa) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    lim_min = max(0, it.q.at + it.tile * PAIRS / gqa);
    lim_max = last_seen(it.q, it.tile, gqa);
    lim = min(it.q.at + (it.tile * PAIRS + t) / gqa, lim_max);  // (no pair: as the tile)
    const float unit = p.scale * 1.44269504088896341f;
    const int pr = it.tile * PAIRS + (g >> 1);
    const bool live = pr < it.q.T * gqa;
    const int row = it.q.r0 + (live ? pr / gqa : 0), head = it.kv * gqa + (live ? pr % gqa : 0);
    const T* q = static_cast<const T*>(p.q) + (size_t)row * p.q_stride + (size_t)head * HD;
    float x[G][16], top = 0.0f, sum[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      sum[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (live) v = kv4_load4(q + j * 64 + t * 16 + i * 4);
        x[j][4 * i] = v.x; x[j][4 * i + 1] = v.y; x[j][4 * i + 2] = v.z; x[j][4 * i + 3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) { sum[j] = fmaf(x[j][i], KV4_QSUM, sum[j]); top = fmaxf(top, fabsf(x[j][i])); }
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the power of two that takes the largest |q| to [2^13, 2^14)
    const int e = min(13 - ((int)(__float_as_uint(top) >> 23) - 127), 100);
    const float sc = __uint_as_float((uint32_t)(e + 127) << 23);
    const float back = fminf(unit * KV4_EVEN * __uint_as_float((uint32_t)(127 - e) << 23), FLT_MAX);
    f = __shfl_sync(0xffffffffu, back, t * 8);
#pragma unroll
    for (int j = 0; j < G; ++j) qs[j] = __shfl_sync(0xffffffffu, sum[j], t * 8) * (unit / KV4_QSUM);
    auto part = [&](float v, float by) {
      v *= sc * by;
      const float hi = __uint_as_float(__float_as_uint(v) & 0xffffe000u);
      return g & 1 ? v - hi : hi;
    };
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* v = &x[j][8 * w + 2 * h];
          uint32_t* b = qb[j / SG][j % SG][w][h];
          b[0] = half2_bits(__floats2half2_rn(part(v[0], 1.0f), part(v[4], 1.0f)));
          b[1] = half2_bits(__floats2half2_rn(part(v[1], 0.0625f), part(v[5], 0.0625f)));
        }
#pragma unroll
    for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[sl][b][h][c] = 0.0f;
    mx = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < G; ++j) mo[j] = 0.0f;
    big = 0x1p-24f;  // a power of two above every d that pair t met
    flushed = false;
  }

  FOX_DEV float4 sum_of(int sl, int b, int h) const {
    const float(&c)[4] = o[sl][b][h];
    float4 v = make_float4(c[0], c[1], c[2], c[3]);
    if (flushed) {
      const float4 w = sums[32 * ((sl * NB + b) * 2 + h)];
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    return v;
  }
  FOX_DEV void flush() {
#pragma unroll
    for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sums[32 * ((sl * NB + b) * 2 + h)] = sum_of(sl, b, h);
#pragma unroll
          for (int c = 0; c < 4; ++c) o[sl][b][h][c] = 0.0f;
        }
    flushed = true;
  }

  // The scores of a page's K block.
  FOX_DEV void scores(const uint8_t* kb) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const __half2* dm = reinterpret_cast<const __half2*>(kb + kv4_codes_bytes(HD));
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int a = s * 16 + g;
      float prod[2], off[2];
#pragma unroll
      for (int sl = 0; sl < SLABS; ++sl) {
        uint32_t wa[2 * SG], wb[2 * SG];
        const uint8_t* base = kb + sl * (KV_PAGE * SLAB / 2) + t * (8 * SG);
        if constexpr (SG == 2) {
          *reinterpret_cast<uint4*>(wa) = *reinterpret_cast<const uint4*>(base + a * (SLAB / 2));
          *reinterpret_cast<uint4*>(wb) = *reinterpret_cast<const uint4*>(base + (a + 8) * (SLAB / 2));
        } else {
          *reinterpret_cast<uint2*>(wa) = *reinterpret_cast<const uint2*>(base + a * (SLAB / 2));
          *reinterpret_cast<uint2*>(wb) = *reinterpret_cast<const uint2*>(base + (a + 8) * (SLAB / 2));
        }
#pragma unroll
        for (int j = 0; j < SG; ++j) {
          const int gg = sl * SG + j;
          float c[4];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t x[4], y[4];
            kv4_operands(wa[2 * j + w], x);
            kv4_operands(wb[2 * j + w], y);
            const uint32_t(&b)[2][2] = qb[sl][j][w];
            if (w == 0) mma16816_0(c, x[0], y[0], x[1], y[1], b[0][0], b[0][1]);
            else mma16816(c, x[0], y[0], x[1], y[1], b[0][0], b[0][1]);
            mma16816(c, x[2], y[2], x[3], y[3], b[1][0], b[1][1]);
          }
          const float2 da = __half22float2(dm[a * G + gg]), db = __half22float2(dm[(a + 8) * G + gg]);
          const float ca = c[0] + c[1], cb = c[2] + c[3];
          prod[0] = gg ? fmaf(da.x, ca, prod[0]) : da.x * ca;
          prod[1] = gg ? fmaf(db.x, cb, prod[1]) : db.x * cb;
          off[0] = gg ? fmaf(da.y, qs[gg], off[0]) : da.y * qs[gg];
          off[1] = gg ? fmaf(db.y, qs[gg], off[1]) : db.y * qs[gg];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) sco[s][h] = fmaf(prod[h], f, off[h]);
    }
  }

  // The largest finite d of a page's parameters: an infinite one makes its own
  // group's sums what they are, and must not scale the others by it.
  static FOX_DEV float largest_finite(const __half2 (&dv)[4][2][G]) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * G; ++i) {
      const float d = __low2float(dv[i / (2 * G)][i / G % 2][i % G]);
      if (!isinf(d)) most = fmaxf(most, d);
    }
#pragma unroll
    for (int sh = 4; sh < 32; sh <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, sh));
    return most;
  }

  // Softmax weights of the page's scores and the sums over its V block. EDGE:
  // some of its positions are hidden from some pair; those count as zeros for it,
  // whatever the memory holds, in the scale of its weights too.
  template <bool EDGE>
  FOX_DEV void values(const uint8_t* vb, int pos0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const __half2* dm = reinterpret_cast<const __half2*>(vb + kv4_codes_bytes(HD));
    // this lane's parameters, the largest d that pair t sees, and its largest score
    __half2 dv[4][2][G], most = __half2half2(__ushort_as_half(0));
    float top;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = s * 16 + h * 8 + g;
        const bool hidden = EDGE && pos0 + at > lim;
#pragma unroll
        for (int j = 0; j < G; ++j) {
          dv[s][h][j] = dm[at * G + j];
          if (hidden) dv[s][h][j] = __half2half2(__ushort_as_half(0));
          most = __hmax2(most, dv[s][h][j]);
        }
        if (hidden) sco[s][h] = -INFINITY;
        top = s + h ? fmaxf(top, sco[s][h]) : sco[s][h];
      }
#pragma unroll
    for (int sh = 4; sh < 32; sh <<= 1) {
      most = __hmax2(most, __shfl_xor_sync(0xffffffffu, most, sh));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sh));
    }
    float dmax = __low2float(most);
    // The reference point of a pair's weights moves only when a score passes
    // it by 2^KV4_SLACK: the weights' scale leaves room for that.
    if (__any_sync(0xffffffffu, dmax >= big || top > mx + KV4_SLACK)) {
      if (__any_sync(0xffffffffu, isinf(dmax))) dmax = largest_finite(dv);  // (NaN it passes over)
      const float to = dmax >= big ? __uint_as_float((__float_as_uint(dmax) & 0x7f800000u) + 0x00800000u) : big;
      const float shrink = big / to;
      big = to;
      const float m = fmaxf(mx, top);
      const float al = m == -INFINITY ? 1.0f : exp2_approx(mx - m), all = al * shrink;
      mx = m;
      l *= al;
#pragma unroll
      for (int j = 0; j < G; ++j) mo[j] *= al;
#pragma unroll
      for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[sl][b][h][c] *= all;
      if (flushed)
#pragma unroll
        for (int i = 0; i < SUM_VECS; ++i) {
          float4& v = sums[32 * i];
          v = make_float4(v.x * all, v.y * all, v.z * all, v.w * all);
        }
    }

    // the weights, times d, as the second product's operand
    const float norm = ((g & 1) ? -KV4_WEIGHT : KV4_WEIGHT) / big, from_top = (g & 1) ? 15.0f : 0.0f;
    // which positions count from the top: odd ones of a step's first half and
    // even ones of its second, the other way round in the next step
    uint32_t flip[2][2] = {{KV4_E & 0xffff0000u, KV4_O & 0xffff0000u}, {KV4_E & 0xffffu, KV4_O & 0xffffu}};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+r"(flip[i / 2][i % 2]));  // held in registers
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint32_t pb[G][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool swap = (s + h) & 1;
        const float w = exp2_approx(sco[s][h] - (EDGE && mx == -INFINITY ? 0.0f : mx)), wn = w * (swap ? -norm : norm);
        l += w;
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const float2 d = __half22float2(dv[s][h][j]);
          const float m = fmaf(swap ? 15.0f - from_top : from_top, d.x, d.y);
          mo[j] = fmaf(w, m, mo[j]);
          pb[j][h] = transpose8x8(kv4_hi_lo(wn * d.x));
        }
      }
#pragma unroll
      for (int sl = 0; sl < SLABS; ++sl) {
        uint32_t u[NB], v[NB];
        const uint8_t* base = vb + ((((sl * 4 + s) * 2) * 4 + t) * 8 + g) * (4 * NB);
        if constexpr (NB == 4) {
          *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(base);
          *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(base + 32 * 4 * NB);
        } else {
          *reinterpret_cast<uint2*>(u) = *reinterpret_cast<const uint2*>(base);
          *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(base + 32 * 4 * NB);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int j = sl * SG + b / 2;
          uint32_t x[4], y[4];
          kv4_operands(u[b], flip[s & 1][0], flip[s & 1][1], x);
          kv4_operands(v[b], flip[1 - (s & 1)][0], flip[1 - (s & 1)][1], y);
          mma16816(o[sl][b][0], x[0], x[1], y[0], y[1], pb[j][0], pb[j][1]);
          mma16816(o[sl][b][1], x[2], x[3], y[2], y[3], pb[j][0], pb[j][1]);
        }
      }
    }
  }

  // The run's results: to `part` (PAIRS partial results), or to the rows of
  // out where that is null.
  template <typename T>
  FOX_DEV void end(const Kv4AttnParams& p, const Kv4Unit& it, int gqa, float* part) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float unit = big * (KV4_EVEN / KV4_WEIGHT);
#pragma unroll
    for (int sh = 4; sh < 32; sh <<= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, sh);
#pragma unroll
      for (int j = 0; j < G; ++j) mo[j] += __shfl_xor_sync(0xffffffffu, mo[j], sh);
    }
    const int pr = it.tile * PAIRS + t;
    if (pr >= it.q.T * gqa) return;
    T* out = static_cast<T*>(p.out) + ((size_t)(it.q.r0 + pr / gqa) * p.n_head + it.kv * gqa + pr % gqa) * HD;
    float* dst = part + (size_t)t * PART;
#pragma unroll
    for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float m = mo[sl * SG + b / 2];
        const float4 x = sum_of(sl, b, 0), y = sum_of(sl, b, 1);
        const float4 v = make_float4(fmaf(x.x + x.y, unit, m), fmaf(x.z + x.w, unit * 0.0625f, m),
                                     fmaf(y.x + y.y, unit, m), fmaf(y.z + y.w, unit * 0.0625f, m));
        const int d = sl * SLAB + b * 32 + g * 4;
        if (part) *reinterpret_cast<float4*>(dst + 4 + d) = v;
        else kv4_store4(out + d, kv4_quotient(v, l));
      }
    if (part && g == 0) *reinterpret_cast<float2*>(dst) = make_float2(mx, l);
  }
};

template <int HD, typename T>
__global__ void __launch_bounds__(Kv4Attn<HD>::NW * 32, 1) kv4_attend_kernel(const Kv4AttnParams p) {
  using A = Kv4Attn<HD>;
  constexpr int PAIRS = A::PAIRS, NW = A::NW, E = HD / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + (size_t)warp * A::PAGE_BYTES;
  uint8_t* heads = smem + (size_t)NW * (A::PAGE_BYTES + A::SUM_VECS * 512);
  uint8_t* behind = heads + (size_t)NW * A::PIECE_BYTES;
  uint64_t* bar = reinterpret_cast<uint64_t*>(behind) + warp * 2;
  int* piece_run = reinterpret_cast<int*>(behind + NW * 2 * 8);  // [2 NW], in line: the runs of the warps' pieces, or -1
  Kv4Line line;
  const int gqa = p.n_head / p.c.n_kv;

  if (lane == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 1, 1);
    mbar_fence_init();
    piece_run[2 * warp] = piece_run[2 * warp + 1] = -1;
  }
  __syncwarp();
  griddep_wait();
  griddep_launch_dependents();
  line.build<PAIRS>(p, piece_run + 2 * NW);
  const int ctas = line.ctas(gridDim.x);
  if ((int)blockIdx.x >= ctas) return;
  const Kv4Split split(line.whole ? line.runs : line.U, ctas);
  auto edge = [&](int c) {
    const int x = split.first(c);
    if (!line.whole) return x;
    if (x == line.runs) return line.U;
    const int s = line.find(line.run0, x);
    return line.unit0[s] + (x - line.run0[s]) * kv4_seq<PAIRS>(p, s).units;
  };
  const int a0 = edge(blockIdx.x), a1 = edge(blockIdx.x + 1);

  auto locate = [&](int u) {
    Kv4Unit x;
    x.seq = line.find(line.unit0, u);
    x.q = kv4_seq<PAIRS>(p, x.seq);
    const int at = u - line.unit0[x.seq], run = at / x.q.units;
    x.page = at - run * x.q.units - KV4_HEAD;
    x.run = line.run0[x.seq] + run;
    x.tile = run / p.c.n_kv;
    x.kv = run - x.tile * p.c.n_kv;
    return x;
  };
  // The K block of a run's page, or null where there is nothing to see: no row
  // of the tile reaches it, or the table names no page there.
  auto find = [&](int seq, int kv, int page, int seen) -> const uint8_t* {
    if (page < 0 || page * KV_PAGE > seen) return nullptr;
    const int at = kv4_page(p.c, seq, page * KV_PAGE);
    return at < 0 ? nullptr : kv4_block(p.c, at, kv, 0, A::BB);
  };
  auto ask = [&](const uint8_t* block, int side) {  // the ring's K or V
    if (block && lane == 0) {
      mbar_arrive_expect_tx(bar + side, A::BB);
      bulk_g2s(ring + side * A::BB, block + side * A::BB, A::BB, bar + side);
    }
  };
  unsigned phase = 0;  // of both barriers
  bool dead = false;   // a wait gave up: the results are not valid, and nothing more is asked for
  auto arrived = [&](int side) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar + side, phase))) return;
    if (__any_sync(0xffffffffu, !mbar_wait(bar + side, phase))) {
      if (lane == 0 && p.c.err) atomicOr(p.c.err, KERR_WAIT);
      dead = true;
    }
  };

  // the warp's stretch, behind the units that only stand ahead of a page
  Kv4Unit cur = locate(a0);
  const int from = a0 + min(max(0, -cur.page), min(a1 - a0, cur.q.units - KV4_HEAD - cur.page) - 1);  // of every run one is left
  const Kv4Split mine(a1 - from, NW);
  const int u0 = from + mine.first(warp), u1 = from + mine.first(warp + 1);
  if (u0 < u1) {
    A w;
    w.sums = reinterpret_cast<float4*>(smem + (size_t)NW * A::PAGE_BYTES) + warp * A::SUM_VECS * 32 + lane;
    int since = 0;  // pages whose sums are in registers
    if (u0 != a0) cur = locate(u0);
    int seq = cur.seq, kv = cur.kv, page = cur.page, end = cur.q.units - KV4_HEAD;
    const uint8_t* block = find(seq, kv, page, A::last_seen(cur.q, cur.tile, gqa));
    ask(block, 0);
    ask(block, 1);
    w.template begin<T>(p, cur, gqa);
    for (int u = u0; u < u1; ++u) {
      // the next page's address is known before this one's codes are used up
      const uint8_t* after = nullptr;
      const bool over = page + 1 == end, last = u + 1 == u1;  // the run's last unit, this warp's
      if (!last && !dead) {
        if (over) {
          const Kv4Unit nxt = locate(u + 1);
          after = find(nxt.seq, nxt.kv, nxt.page, A::last_seen(nxt.q, nxt.tile, gqa));
        } else {
          after = find(seq, kv, page + 1, w.lim_max);
        }
      }
      if (block) {
        const int pos0 = page * KV_PAGE;
        arrived(0);
        if (!dead) w.scores(ring);
        __syncwarp();  // every lane has read K
        if (!dead) ask(after, 0);
        arrived(1);
        if (!dead) {
          if (pos0 + KV_PAGE - 1 > w.lim_min) w.template values<true>(ring + A::BB, pos0);
          else w.template values<false>(ring + A::BB, pos0);
        }
        __syncwarp();
        if (!dead) ask(after, 1);
        phase ^= 1;
        if (++since == KV4_FLUSH) { w.flush(); since = 0; }
      } else {
        ask(after, 0);
        ask(after, 1);
      }
      block = dead ? nullptr : after;
      ++page;
      if (over || last) {
        cur = locate(u);
        const int run_first = u - (cur.page + KV4_HEAD);
        const bool whole = over && (run_first >= u0 || (u0 == from && run_first >= a0));
        float* part = reinterpret_cast<float*>(last ? ring : heads + (size_t)warp * A::PIECE_BYTES);
        w.template end<T>(p, cur, gqa, whole ? nullptr : part);
        if (!whole && lane == 0) piece_run[2 * warp + last] = cur.run;
        if (!last) {
          cur = locate(u + 1);
          seq = cur.seq; kv = cur.kv; page = cur.page; end = cur.q.units - KV4_HEAD;
          w.template begin<T>(p, cur, gqa);
          since = 0;
        }
      }
    }
  }
  if (dead)  // copies in flight end before their memory is used for something else
    for (int i = 0; i < 4; ++i) mbar_wait(bar + i / 2, i & 1);
  __syncthreads();

  // the pieces of each run, in line: piece 2w is one that warp w ended before
  // its last, which is 2w + 1 and in its ring
  for (int x = warp; x < 2 * NW * PAIRS; x += NW) {
    const int k = x / PAIRS, i = x % PAIRS, run = piece_run[k];
    if (run < 0) continue;
    int before = k - 1;
    while (before >= 0 && piece_run[before] < 0) --before;
    if (before >= 0 && piece_run[before] == run) continue;  // joined with that one
    const int s = line.find(line.run0, run);
    const Kv4Seq q = kv4_seq<PAIRS>(p, s);
    const int r = run - line.run0[s], kv = r % p.c.n_kv, pr = r / p.c.n_kv * PAIRS + i;
    if (pr >= q.T * gqa) continue;
    Kv4Sum<HD> sum;
    for (int j = k; j < 2 * NW && (piece_run[j] < 0 || piece_run[j] == run); ++j) {
      if (piece_run[j] < 0) continue;
      sum.add(reinterpret_cast<const float*>(j & 1 ? smem + (size_t)(j / 2) * A::PAGE_BYTES
                                                   : heads + (size_t)(j / 2) * A::PIECE_BYTES) + i * A::PART);
    }
    const int first = line.unit0[s] + r * q.units;
    if (first >= a0 && first + q.units <= a1) {
      sum.store(static_cast<T*>(p.out) + ((size_t)(q.r0 + pr / gqa) * p.n_head + kv * gqa + pr % gqa) * HD);
    } else {  // the end of a run that began earlier, or the beginning of one that goes on
      float* dst = p.part + (((size_t)blockIdx.x * 2 + (first >= a0)) * PAIRS + i) * A::PART;
      if (lane == 0) *reinterpret_cast<float2*>(dst) = make_float2(sum.M, sum.l);
#pragma unroll
      for (int e = 0; e < E; ++e) dst[4 + e * 32 + lane] = sum.v[e];
    }
  }
}

// Joins the CTAs' pieces of split runs, in the line's order. Bound by the
// blocks' way to their pieces, not by the bytes: alone and cold 10 us for the
// 128 runs of 16 sequences (0.6 MB from memory), 16 us for the 16 runs of 128
// pairs of 64 rows (11 MB); in a call its start overlaps the first kernel's end. A pair of a run
// takes 1, 2, 4 or 8 of the CTA's warps, by how many pieces a run has on
// average; each takes every such-th piece.
constexpr int KV4_JOIN_WARPS = 8;
template <int HD>
__host__ __device__ constexpr int kv4_join_smem(int n_seq) {
  return KV4_JOIN_WARPS * (HD + 2) * 4 + Kv4Line::bytes(n_seq);
}
template <int HD, typename T, int PAIRS>
__global__ void __launch_bounds__(KV4_JOIN_WARPS * 32) kv4_join_kernel(const Kv4AttnParams p) {
  constexpr int E = HD / 32, JW = KV4_JOIN_WARPS, PART = HD + 4;
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem);  // [JW][HD + 2]
  Kv4Line line;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gqa = p.n_head / p.c.n_kv;
  line.build<PAIRS>(p, red + JW * (HD + 2));  // of arrays that the attention does not write
  griddep_wait();  // by every thread: the end of this kernel stands for the end of the attention too
  const int ctas = line.ctas(p.ctas);
  if (line.whole || ctas == 0) return;
  const Kv4Split split(line.U, ctas);
  int team = 1;  // warps of a pair
  while (team < JW && team * 8 * line.runs < ctas) team *= 2;
  const int teams = JW / team, in_team = warp % team;
  const long long pairs = (long long)line.runs * PAIRS;
  for (long long x0 = (long long)blockIdx.x * teams; x0 < pairs; x0 += (long long)gridDim.x * teams) {
    const long long x = x0 + warp / team;
    const int run = (int)(x / PAIRS), i = (int)(x % PAIRS);
    Kv4Sum<HD> sum;
    T* out = nullptr;
    if (x < pairs) {
      const int s = line.find(line.run0, run);
      const Kv4Seq q = kv4_seq<PAIRS>(p, s);
      const int r = run - line.run0[s], kv = r % p.c.n_kv, pr = r / p.c.n_kv * PAIRS + i;
      const int first = line.unit0[s] + r * q.units;
      const int c0 = split.owner(first), c1 = split.owner(first + q.units - 1);
      if (c0 != c1 && pr < q.T * gqa) {
        out = static_cast<T*>(p.out) + ((size_t)(q.r0 + pr / gqa) * p.n_head + kv * gqa + pr % gqa) * HD;
#pragma unroll 4
        for (int c = c0 + in_team; c <= c1; c += team)
          sum.add(p.part + (((size_t)c * 2 + (c == c0)) * PAIRS + i) * PART);
      }
    }
    if (team > 1) {
      __syncthreads();  // red is free
#pragma unroll
      for (int e = 0; e < E; ++e) red[warp * (HD + 2) + e * 32 + lane] = sum.v[e];
      if (lane == 0) { red[warp * (HD + 2) + HD] = sum.M; red[warp * (HD + 2) + HD + 1] = sum.l; }
      __syncthreads();
      if (in_team) continue;
      for (int k = 1; k < team; ++k) {
        const float* from = red + (warp + k) * (HD + 2);
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = from[e * 32 + lane];
        sum.add(from[HD], from[HD + 1], v);
      }
    }
    if (out) sum.store(out);
  }
}

}  // namespace fox
