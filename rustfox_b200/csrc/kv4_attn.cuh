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
// - Odd positions of V are taken from their top level down, x = (m + 15 d) -
//   d (15 - c), with the complement of the code (an xor that joins the mask)
//   and a negated weight: the second product's sums then stay near the result
//   instead of 7.5 d away from it. They round toward zero, so what would
//   cancel in the end must not pass through them: at 32768 positions the error
//   was 1e-4 of the result with all positions counted from below. A page's
//   sums start at zero and join the rest in plain fp32 for the same reason.
#pragma once

#include <climits>

#include "kv4.cuh"

namespace fox {

constexpr int KV4_MAX_SEQ = 1024;

struct Kv4AttnParams {
  Kv4Rows c;
  const void* q;
  void* out;
  float* part;       // partial results of split sequences
  size_t q_stride;   // elements between rows
  int n_head, sms;
  float scale;
};

// How a sequence of L positions and T rows is cut, from its own numbers and
// the device's: tiles of `pairs` (row, head) pairs of a KV head, and segments
// of pages that different CTAs take when rows and heads alone do not fill the
// device.
constexpr int KV4_SEG_PAGES = 4;    // pages a segment has at least
struct Kv4Cut { int tiles, segs; };
__host__ __device__ inline Kv4Cut kv4_cut(int L, int T, int gqa, int n_kv, int pairs, int sms) {
  Kv4Cut k;
  k.tiles = (T * gqa + pairs - 1) / pairs;
  const int pages = (L + KV_PAGE - 1) / KV_PAGE;
  const int want = sms / max(1, n_kv * k.tiles), most = (pages + KV4_SEG_PAGES - 1) / KV4_SEG_PAGES;
  k.segs = max(1, min(want, most));
  return k;
}
// Slots of partial results a sequence can need beyond one for each row.
__host__ __device__ inline int kv4_extra_slots(int n_head, int pairs, int sms) {
  return (sms * pairs + n_head - 1) / n_head;
}

FOX_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// 8 codes of a word (nibble i in bits 4i) as four operand registers: codes
// (0, 4), (1, 5), (2, 6), (3, 7), the even ones as c * 2^-22, the odd ones as
// c * 2^-18. With ODD the upper half's codes are complemented.
template <bool ODD>
FOX_DEV void kv4_operands(uint32_t x, uint32_t (&a)[4]) {
  constexpr uint32_t E = 0x003c003cu, O = 0x03c003c0u, FE = ODD ? E & 0xffff0000u : 0, FO = ODD ? O & 0xffff0000u : 0;
  const uint32_t up = x << 2, down = x >> 6;
  a[0] = (up & E) ^ FE;
  a[1] = (up & O) ^ FO;
  a[2] = (down & E) ^ FE;
  a[3] = (down & O) ^ FO;
}
constexpr float KV4_EVEN = 4194304.0f;  // 2^22
// x as hi + lo fp16: hi keeps the leading 11 bits.
FOX_DEV uint32_t kv4_hi_lo(float x) {
  const float hi = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
  return half2_bits(__floats2half2_rn(hi, x - hi));
}

// What a warp's pages are: a range of pages of one sequence and KV head.
struct Kv4Item {
  int seq, kv, tile, seg, segs, first, last;  // pages first .. last-1
  int r0, T, L;
};

// HD: head dimension; NT: column tiles (of 4 pairs) of a warp.
template <int HD, int NT>
struct Kv4Attn {
  static constexpr int SLAB = HD < 128 ? HD : 128, SLABS = HD / SLAB, SG = SLAB / 64, NB = SLAB / 32;
  static constexpr int G = HD / KV4_GROUP, BB = kv4_block_bytes(HD), PAGE_BYTES = 2 * BB;
  static constexpr int PAIRS = 4 * NT;       // (row, head) pairs of a tile
  static constexpr int RED_STRIDE = HD + 4;  // floats of one pair of one warp
  // warps of a CTA and pages in flight per warp: what shared memory holds
  static constexpr int NW = HD == 64 ? 12 : HD == 128 ? 10 : 5, SLOTS = HD == 64 ? 3 : 2;
  static constexpr size_t ring_bytes() { return (size_t)NW * SLOTS * PAGE_BYTES; }
  static constexpr size_t red_bytes() { return (size_t)NW * PAIRS * RED_STRIDE * 4; }
  static constexpr size_t smem_bytes(int n_seq) {
    return ring_bytes() + red_bytes() + NW * PAIRS * 8 + NW * SLOTS * 8 + (size_t)(n_seq + 1) * 4 + 16;
  }

  // A warp's share of a tile: q's operand registers, and the running maximum,
  // weights and sums of its pairs. Lane (g, t) = (lane / 4, lane % 4) holds
  // the scores of pair t of each column tile at positions g and g + 8 of a
  // step, and the sums of dimensions 4g .. 4g+3 of each block of 32.
  uint32_t qb[NT][SLABS][SG][2][2][2];
  float f[NT], qs[NT][G];  // score = f * sum_g (d_g * product) + sum_g m_g * qs_g, in powers of 2
  float o[NT][SLABS][NB][2][4], mx[NT], l[NT], mo[NT][G], big;
  int lim[NT], lim_min, lim_max;  // the last position a pair sees (negative: none; no pair: all), and over the tile

  FOX_DEV void limits(const Kv4Item& it, int gqa) {
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int pr = it.tile * PAIRS + n * 4 + t;
      lim[n] = pr < it.T * gqa ? it.L - it.T + pr / gqa : INT_MAX;
    }
    lim_min = max(0, it.L - it.T + it.tile * PAIRS / gqa);
    lim_max = it.L - it.T + min(it.T - 1, (it.tile * PAIRS + PAIRS - 1) / gqa);
  }

  template <typename T>
  FOX_DEV void load_q(const Kv4AttnParams& p, const Kv4Item& it, int gqa) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float unit = p.scale * 1.44269504088896341f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int pr = it.tile * PAIRS + n * 4 + (g >> 1);
      const bool live = pr < it.T * gqa;
      const int row = it.r0 + (live ? pr / gqa : 0), head = it.kv * gqa + (live ? pr % gqa : 0);
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
        for (int i = 0; i < 16; ++i) { sum[j] += x[j][i]; top = fmaxf(top, fabsf(x[j][i])); }
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the power of two that takes the largest |q| to [2^13, 2^14)
      const int e = min(max(13 - ((int)(__float_as_uint(top) >> 23) - 127), -100), 100);
      const float sc = __uint_as_float((uint32_t)(e + 127) << 23);
      const float back = unit * KV4_EVEN * __uint_as_float((uint32_t)(127 - e) << 23);
      f[n] = __shfl_sync(0xffffffffu, back, t * 8);
#pragma unroll
      for (int j = 0; j < G; ++j) qs[n][j] = __shfl_sync(0xffffffffu, sum[j], t * 8) * unit;
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
            uint32_t* b = qb[n][j / SG][j % SG][w][h];
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
            for (int c = 0; c < 4; ++c) o[n][sl][b][h][c] = 0.0f;
      mx[n] = -INFINITY;
      l[n] = 0.0f;
#pragma unroll
      for (int j = 0; j < G; ++j) mo[n][j] = 0.0f;
    }
    big = 0x1p-24f;  // a power of two above every d met
  }

  // One page in shared memory. EDGE: some of its positions are hidden from
  // some pair (`absent`: all of them from all).
  template <bool EDGE>
  FOX_DEV void page(const uint8_t* kb, int pos0, bool absent) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint8_t* vb = kb + BB;
    const __half2* kdm = reinterpret_cast<const __half2*>(kb + kv4_codes_bytes(HD));
    const __half2* vdm = reinterpret_cast<const __half2*>(vb + kv4_codes_bytes(HD));
    float sco[NT][4][2];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int a = s * 16 + g;
      float prod[NT][2], off[NT][2];
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
          float c[NT][4] = {};
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t x[4], y[4];
            kv4_operands<false>(wa[2 * j + w], x);
            kv4_operands<false>(wb[2 * j + w], y);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma16816(c[n], x[0], y[0], x[1], y[1], qb[n][sl][j][w][0][0], qb[n][sl][j][w][0][1]);
              mma16816(c[n], x[2], y[2], x[3], y[3], qb[n][sl][j][w][1][0], qb[n][sl][j][w][1][1]);
            }
          }
          const float2 da = __half22float2(kdm[a * G + gg]), db = __half22float2(kdm[(a + 8) * G + gg]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float ca = c[n][0] + c[n][1], cb = c[n][2] + c[n][3];
            prod[n][0] = gg ? fmaf(da.x, ca, prod[n][0]) : da.x * ca;
            prod[n][1] = gg ? fmaf(db.x, cb, prod[n][1]) : db.x * cb;
            off[n][0] = gg ? fmaf(da.y, qs[n][gg], off[n][0]) : da.y * qs[n][gg];
            off[n][1] = gg ? fmaf(db.y, qs[n][gg], off[n][1]) : db.y * qs[n][gg];
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) sco[n][s][h] = fmaf(prod[n][h], f[n], off[n][h]);
    }

    // V's parameters of this lane's positions, the page's largest d, and the
    // maxima over its positions
    float2 dv[4][2][G];
    float dmax = 0.0f, top[NT];
    const float from_top = (g & 1) ? 15.0f : 0.0f;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = s * 16 + h * 8 + g;
        const bool nobody = EDGE && (absent || pos0 + at > lim_max);
#pragma unroll
        for (int j = 0; j < G; ++j) {
          dv[s][h][j] = __half22float2(vdm[at * G + j]);
          if (nobody) dv[s][h][j] = make_float2(0.0f, 0.0f);  // whatever the memory held
          dmax = fmaxf(dmax, dv[s][h][j].x);
          dv[s][h][j].y = fmaf(from_top, dv[s][h][j].x, dv[s][h][j].y);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (EDGE && (absent || pos0 + at > lim[n])) sco[n][s][h] = -INFINITY;
          top[n] = s + h ? fmaxf(top[n], sco[n][s][h]) : sco[n][s][h];
        }
      }
#pragma unroll
    for (int sh = 4; sh < 32; sh <<= 1) {
      dmax = fmaxf(dmax, __shfl_xor_sync(0xffffffffu, dmax, sh));
#pragma unroll
      for (int n = 0; n < NT; ++n) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], sh));
    }
    bool grew = dmax >= big;
#pragma unroll
    for (int n = 0; n < NT; ++n) grew = grew || top[n] > mx[n];
    if (__any_sync(0xffffffffu, grew)) {
      const float to = dmax >= big ? __uint_as_float((__float_as_uint(dmax) & 0x7f800000u) + 0x00800000u) : big;
      const float shrink = big / to;
      big = to;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float m = fmaxf(mx[n], top[n]);
        const float al = m == -INFINITY ? 1.0f : exp2_approx(mx[n] - m), all = al * shrink;
        mx[n] = m;
        l[n] *= al;
#pragma unroll
        for (int j = 0; j < G; ++j) mo[n][j] *= al;
#pragma unroll
        for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[n][sl][b][h][c] *= all;
      }
    }

    // the weights, times d, as the second product's operand
    const float norm = ((g & 1) ? -32768.0f : 32768.0f) / big;
    uint32_t pb[NT][4][G][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float base = EDGE && mx[n] == -INFINITY ? 0.0f : mx[n];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w = exp2_approx(sco[n][s][h] - base), wn = w * norm;
          l[n] += w;
#pragma unroll
          for (int j = 0; j < G; ++j) {
            float v = wn * dv[s][h][j].x, m = dv[s][h][j].y;
            if (EDGE && sco[n][s][h] == -INFINITY) v = m = 0.0f;  // hidden, whatever it is
            mo[n][j] = fmaf(w, m, mo[n][j]);
            pb[n][s][j][h] = transpose8x8(kv4_hi_lo(v));
          }
        }
    }
#pragma unroll
    for (int sl = 0; sl < SLABS; ++sl) {
      uint32_t u[4][NB], v[4][NB];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint8_t* base = vb + ((((sl * 4 + s) * 2) * 4 + t) * 8 + g) * (4 * NB);
        if constexpr (NB == 4) {
          *reinterpret_cast<uint4*>(u[s]) = *reinterpret_cast<const uint4*>(base);
          *reinterpret_cast<uint4*>(v[s]) = *reinterpret_cast<const uint4*>(base + 32 * 4 * NB);
        } else {
          *reinterpret_cast<uint2*>(u[s]) = *reinterpret_cast<const uint2*>(base);
          *reinterpret_cast<uint2*>(v[s]) = *reinterpret_cast<const uint2*>(base + 32 * 4 * NB);
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int j = sl * SG + b / 2;
        float c[NT][2][4] = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          uint32_t x[4], y[4];
          kv4_operands<true>(u[s][b], x);
          kv4_operands<true>(v[s][b], y);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816(c[n][0], x[0], x[1], y[0], y[1], pb[n][s][j][0], pb[n][s][j][1]);
            mma16816(c[n][1], x[2], x[3], y[2], y[3], pb[n][s][j][0], pb[n][s][j][1]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][sl][b][h][i] += c[n][h][i];
      }
    }
  }

  // The warp's sums over its lanes' positions, to its part of `red` (PAIRS
  // rows) and redm.
  FOX_DEV void park(float* red, float2* redm) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float unit = big * (KV4_EVEN / 32768.0f);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) {
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], sh);
#pragma unroll
        for (int j = 0; j < G; ++j) mo[n][j] += __shfl_xor_sync(0xffffffffu, mo[n][j], sh);
      }
      float* dst = red + (size_t)(n * 4 + t) * RED_STRIDE;
#pragma unroll
      for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float m = mo[n][sl * SG + b / 2];
          const float(&c)[2][4] = o[n][sl][b];
          *reinterpret_cast<float4*>(dst + sl * SLAB + b * 32 + g * 4) =
              make_float4(fmaf(c[0][0] + c[0][1], unit, m), fmaf(c[0][2] + c[0][3], unit * 0.0625f, m),
                          fmaf(c[1][0] + c[1][1], unit, m), fmaf(c[1][2] + c[1][3], unit * 0.0625f, m));
        }
      if (g == 0) redm[n * 4 + t] = make_float2(mx[n], l[n]);
    }
  }
};

// Prefix sums of every sequence's items (tiles x KV heads x segments) in
// shared memory, by the CTA's first warp.
template <int PAIRS>
FOX_DEV void kv4_schedule(const Kv4AttnParams& p, int* start) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int base = 0;
    for (int s0 = 0; s0 < p.c.n_seq; s0 += 32) {
      const int s = s0 + lane;
      int n = 0;
      if (s < p.c.n_seq) {
        const int a = min(max(__ldg(p.c.row_start + s), 0), p.c.n_rows);
        const int b = min(max(__ldg(p.c.row_start + s + 1), a), p.c.n_rows);
        if (b > a) {
          const Kv4Cut k = kv4_cut(kv4_len(p.c, s), b - a, p.n_head / p.c.n_kv, p.c.n_kv, PAIRS, p.sms);
          n = k.tiles * k.segs * p.c.n_kv;
        }
      }
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (s < p.c.n_seq) start[s] = base + sum - n;
      base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) start[p.c.n_seq] = base;
  }
  __syncthreads();
}

template <int PAIRS>
FOX_DEV Kv4Item kv4_item(const Kv4AttnParams& p, const int* start, int item) {
  int lo = 0, hi = p.c.n_seq - 1;  // the last sequence that starts at or before the item
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (start[mid] <= item) lo = mid; else hi = mid - 1;
  }
  Kv4Item it;
  it.seq = lo;
  it.r0 = min(max(__ldg(p.c.row_start + lo), 0), p.c.n_rows);
  it.T = min(max(__ldg(p.c.row_start + lo + 1), it.r0), p.c.n_rows) - it.r0;
  it.L = min(max(__ldg(p.c.kv_len + lo), 0), p.c.table_stride * KV_PAGE);
  const Kv4Cut k = kv4_cut(it.L, it.T, p.n_head / p.c.n_kv, p.c.n_kv, PAIRS, p.sms);
  int r = item - start[lo];
  it.segs = k.segs;
  it.seg = r % k.segs; r /= k.segs;
  it.kv = r % p.c.n_kv;
  it.tile = r / p.c.n_kv;
  const int pages = (it.L + KV_PAGE - 1) / KV_PAGE;
  it.first = (int)((long long)pages * it.seg / k.segs);
  it.last = (int)((long long)pages * (it.seg + 1) / k.segs);
  return it;
}

template <int HD, typename T, int NT>
__global__ void __launch_bounds__(Kv4Attn<HD, NT>::NW * 32, 1) kv4_attend_kernel(const Kv4AttnParams p) {
  using A = Kv4Attn<HD, NT>;
  constexpr int PAIRS = A::PAIRS, NW = A::NW, SLOTS = A::SLOTS;
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem + A::ring_bytes());
  float2* redm = reinterpret_cast<float2*>(smem + A::ring_bytes() + A::red_bytes());  // (M, l) of a warp's pair
  uint64_t* bars = reinterpret_cast<uint64_t*>(redm + NW * PAIRS);
  int* start = reinterpret_cast<int*>(bars + NW * SLOTS);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + (size_t)warp * SLOTS * A::PAGE_BYTES;
  uint64_t* bar = bars + warp * SLOTS;
  const int gqa = p.n_head / p.c.n_kv;

  if (lane == 0) {
    for (int i = 0; i < SLOTS; ++i) mbar_init(bar + i, 1);
    mbar_fence_init();
  }
  __syncwarp();
  griddep_wait();
  griddep_launch_dependents();
  kv4_schedule<PAIRS>(p, start);
  const int n_items = start[p.c.n_seq];

  A w;
  Kv4Item it;
  int issued = 0, taken = 0;  // pages this warp asked for and used, over all items
  int n_mine = 0;             // pages of the item this warp takes: first + warp, + NW, ...
  bool dead = false;          // a wait gave up: nothing more is asked for
  auto issue = [&](int i) {   // this warp's i-th page of the item
    if (lane == 0) {
      const int slot = issued % SLOTS;
      const int page = kv4_page(p.c, it.seq, (it.first + warp + i * NW) * KV_PAGE);
      // an absent page is not read: its positions are masked when taken
      mbar_arrive_expect_tx(bar + slot, page >= 0 ? A::PAGE_BYTES : 0);
      if (page >= 0)
        bulk_g2s(ring + (size_t)slot * A::PAGE_BYTES, kv4_block(p.c, page, it.kv, 0, A::BB), A::PAGE_BYTES, bar + slot);
    }
    ++issued;
  };
  auto begin = [&](int item) {
    it = kv4_item<PAIRS>(p, start, item);
    w.limits(it, gqa);
    const int last = min(it.last, w.lim_max < 0 ? 0 : w.lim_max / KV_PAGE + 1);
    n_mine = last > it.first + warp ? (last - it.first - warp + NW - 1) / NW : 0;
    for (int i = 0; i < min(n_mine, SLOTS) && !dead; ++i) issue(i);
  };
  if ((int)blockIdx.x < n_items) begin(blockIdx.x);
  for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
    w.template load_q<T>(p, it, gqa);
    for (int i = 0; i < n_mine && !dead; ++i) {
      const int slot = taken % SLOTS, pos0 = (it.first + warp + i * NW) * KV_PAGE;
      const int page = __ldg(p.c.table + (size_t)it.seq * p.c.table_stride + pos0 / KV_PAGE);
      const bool absent = (unsigned)page >= (unsigned)p.c.n_pages;
      dead = __any_sync(0xffffffffu, !mbar_wait(bar + slot, (taken / SLOTS) & 1));
      if (dead) {
        if (lane == 0 && p.c.err) atomicExch(p.c.err, KERR_WAIT);
        break;
      }
      ++taken;
      const uint8_t* kb = ring + (size_t)slot * A::PAGE_BYTES;
      if (absent || pos0 + KV_PAGE - 1 > w.lim_min) w.template page<true>(kb, pos0, absent);
      else w.template page<false>(kb, pos0, false);
      __syncwarp();  // every lane has read the slot
      if (i + SLOTS < n_mine) issue(i + SLOTS);
    }
    w.park(red + (size_t)warp * PAIRS * A::RED_STRIDE, redm + warp * PAIRS);
    const Kv4Item was = it;
    // the next item's pages are on their way while this one's warps are joined
    if (item + (int)gridDim.x < n_items) begin(item + gridDim.x);
    __syncthreads();
    for (int u = threadIdx.x; u < PAIRS * HD; u += NW * 32) {
      const int pr = u / HD, d = u % HD, pair = was.tile * PAIRS + pr;
      if (pair >= was.T * gqa) break;
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < NW; ++k) M = fmaxf(M, redm[k * PAIRS + pr].x);
      float sum = 0.0f, ls = 0.0f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float2 ml = redm[k * PAIRS + pr];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // nothing seen by this warp
        const float by = exp2_approx(ml.x - M);
        ls = fmaf(ml.y, by, ls);
        sum = fmaf(red[(size_t)(k * PAIRS + pr) * A::RED_STRIDE + d], by, sum);
      }
      const int row = pair / gqa, head = was.kv * gqa + pair % gqa;
      if (was.segs == 1) {
        const float r = ls == 0.0f ? 0.0f : __fdiv_rn(sum, ls);  // nothing to see: zeros
        static_cast<T*>(p.out)[((size_t)(was.r0 + row) * p.n_head + head) * HD + d] = (T)r;
      } else {
        const size_t slot = (size_t)was.r0 + (size_t)was.seq * kv4_extra_slots(p.n_head, PAIRS, p.sms) +
                            (size_t)row * was.segs + was.seg;
        float* dst = p.part + (slot * p.n_head + head) * (HD + 4);
        dst[4 + d] = sum;
        if (d == 0) { dst[0] = M; dst[1] = ls; }
      }
    }
    __syncthreads();  // red is free
  }
  // copies in flight end before the CTA does
  for (; taken < issued; ++taken) mbar_wait(bar + taken % SLOTS, (taken / SLOTS) & 1);
}

// Joins the segments of split sequences, one warp for a row's head, in
// segment order.
template <int HD, typename T, int PAIRS>
__global__ void __launch_bounds__(256) kv4_merge_kernel(const Kv4AttnParams p) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const size_t unit = blockIdx.x * (size_t)(blockDim.x / 32) + threadIdx.x / 32;
  griddep_wait();  // by every thread: the end of this kernel stands for the end of the one before it too
  if (unit >= (size_t)p.c.n_rows * p.n_head) return;
  const int row = (int)(unit / p.n_head), head = (int)(unit - (size_t)row * p.n_head);
  const int s = kv4_seq_of(p.c, row);
  if (s >= p.c.n_seq) return;
  const int r0 = min(max(__ldg(p.c.row_start + s), 0), p.c.n_rows);
  const int T_ = min(max(__ldg(p.c.row_start + s + 1), r0), p.c.n_rows) - r0;
  const int L = min(max(__ldg(p.c.kv_len + s), 0), p.c.table_stride * KV_PAGE);
  const Kv4Cut k = kv4_cut(L, T_, p.n_head / p.c.n_kv, p.c.n_kv, PAIRS, p.sms);
  if (k.segs == 1 || row < r0) return;
  const size_t slot = (size_t)r0 + (size_t)s * kv4_extra_slots(p.n_head, PAIRS, p.sms) + (size_t)(row - r0) * k.segs;
  const float* src = p.part + (slot * p.n_head + head) * (HD + 4);
  const size_t step = (size_t)p.n_head * (HD + 4);
  float M = -INFINITY;
  for (int j = lane; j < k.segs; j += 32) M = fmaxf(M, src[j * step]);
  M = warp_max(M);
  float ls = 0.0f, sum[E] = {};
  for (int j = 0; j < k.segs; ++j) {
    const float m = src[j * step], lj = src[j * step + 1];
    if (m == -INFINITY && lj == 0.0f) continue;
    const float by = exp2_approx(m - M);
    ls = fmaf(lj, by, ls);
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] = fmaf(src[j * step + 4 + lane * E + i], by, sum[i]);
  }
  T* out = static_cast<T*>(p.out) + unit * HD + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) out[i] = (T)(ls == 0.0f ? 0.0f : __fdiv_rn(sum[i], ls));
}

}  // namespace fox
