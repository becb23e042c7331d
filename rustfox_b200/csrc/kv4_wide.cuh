// Attention over the 4-bit cache for many rows of a sequence (sm_100a): both
// products on the 5th-generation tensor cores (tcgen05 kind::f16, fp32 sums in
// tensor memory).
//
// With c' = 2 c - 15 a cached value is x = m + d c = ((2 m + 15 d) + d c') / 2.
// d c' has 15 significant bits, so it is hi + lo in fp16 exactly (a product and
// the fused remainder), and the offsets 2 m + 15 d, one for each position and
// group, are hi + lo to 22 bits. So the unpacked page is a set of fp16
// operands, scaled by a power of two to fp16's range (kv4_level says what that
// costs beside values beyond 16384), and the parameters never meet the scores:
//   S = Qh Kh + Ql Kh + Qh Kl + (sums of q per group) (offsets of K)
//   O = Ph Vh + Pl Vh + Ph Vl,  with V's offsets as further columns
// with q and the weights as hi + lo fp16 too. (An earlier form multiplied the
// scores and weights by d, and added m, after the products: each of its threads
// loaded every position's parameters from shared memory, and that bounded it.)
//
// A CTA takes 128 (row, head) pairs of a KV head (the products' 128 rows) and
// walks their pages; its warps have roles:
// - 3 warps unpack a page's K, 4 its V, into 8 x 16-byte core matrices whose
//   strides keep the stores free of bank conflicts.
// - 1 warp loads pages and issues the products. q stands in tensor memory, and
//   a page's weights take the place of its scores there. The scores of page
//   j + 1 are formed while page j's weights are.
// - 8 warps form the weights: two threads share a pair, each with half of the
//   page's positions and of the pair's sums, and hold most of the registers.
//   The reference point of a pair's weights moves only when a score passes it
//   by 2^KV4_SLACK; then, and every KV4_WIDE_FLUSH pages, O leaves tensor
//   memory for the threads' registers, which bounds what the products' rounding
//   toward zero adds up to: 1.3e-6 of the result at every 4 pages, 2.1e-6 and
//   0.6 % of the time less at every 8.
// The work is divided as in kv4_attn.cuh, with a CTA for a warp.
//
// 64 rows behind 16384 positions, 32 heads over 8 of 128, take 83 us: 207
// TFLOP/s of the formula's products, of which this form issues three for one and
// the offsets. A page takes a tile about 4300 cycles, and K's three warps are
// what it waits for (1200 cycles for the parameters and their exchange, 1800 for
// the codes); the products take 1700, the weights 2000. With four warps for K
// and three for V, V's are waited for instead, in the same time. The time hardly
// depends on how many of the 128 pairs are live.
#pragma once

#include "kv4_attn.cuh"
#include "tcgen05.cuh"

#include <math_constants.h>

namespace fox {

constexpr unsigned long long KV4_WAIT_NS = 500000000;  // half a second
constexpr int KV4_WIDE_PAIRS = 128, KV4_WIDE_FLUSH = 4;

template <int HD>
struct Kv4Wide {
  static constexpr int G = HD / KV4_GROUP, BB = kv4_block_bytes(HD), PAGE_BYTES = 2 * BB, PART = HD + 4;
  static constexpr int PAIRS = KV4_WIDE_PAIRS, SHARE = 2, OWN = HD / SHARE, POS = KV_PAGE / SHARE;  // threads of a pair; their dimensions and positions
  static constexpr int SOFT = PAIRS * SHARE, THREADS = 512;
  // second operands, K [position][dimension] and V [dimension][position]: 8
  // rows are 1168 bytes, 8 fp16 along the contraction 144; V has 16 further
  // rows, (hi, lo) of each group's offsets and zeros
  static constexpr int LBO = 144, SBO = 8 * LBO + 16, TILE = 8 * SBO, V_ROWS = HD + 16;
  static constexpr int K_HALF = G * TILE, KM_SBO = 2 * LBO, KM_AT = 2 * K_HALF, K_BYTES = KM_AT + 8 * KM_SBO;  // hi, lo, offsets
  static constexpr int V_LO = V_ROWS / 8 * SBO, V_BYTES = V_LO + G * TILE;                                     // hi and offsets, lo
  // tensor memory's columns: S (then P) of two pages, O with the offsets, Q
  static constexpr int O_COL = 2 * KV_PAGE, Q_COL = O_COL + V_ROWS, QM_COL = Q_COL + HD, TMEM = 512;
  static_assert(QM_COL + 8 <= TMEM, "what is allocated");
  // warps by role, in groups of four that share a number of registers: 128 a
  // thread at launch, 8 x 176 + 8 x 80 = 16 x 128
  static constexpr int V_WARP = 8, K_WARP = 12, MMA_WARP = 15;
  static constexpr int SOFT_REGS = 176, OTHER_REGS = 80;
  static constexpr int RAW = 4;  // pages loaded ahead
  // shared memory
  static constexpr int K_AT = 0, V_AT = K_AT + 2 * K_BYTES, RAW_AT = V_AT + 2 * V_BYTES, D_AT = RAW_AT + RAW * PAGE_BYTES;
  static constexpr int EX_AT = D_AT + 4 * G * KV_PAGE * 2;  // [K, V][buffer][group][position] d; then the sharing threads' exchange
  static constexpr int LINE_AT = EX_AT + SOFT * 16;
  static_assert(RAW_AT % 16 == 0 && EX_AT % 16 == 0, "bulk copies and vectors");
  static size_t smem_bytes(int n_seq) { return LINE_AT + Kv4Line::bytes(n_seq); }
};

struct Kv4WideBars {
  // Of the pages that share a barrier, the later one's phase must not end before
  // all who wait for the earlier one's have seen it. K runs ahead of the weights
  // by more than the two buffers' turn, so it has four.
  uint64_t raw_full[4], k_full[4], v_full[2], s_full[2], p_full[2], pv_done[2], q_full;
  uint32_t tmem;
  int fresh[2];                         // the page's O does not add to what tensor memory holds
  float k_unit[4], v_unit[4];           // what 1 stands for in the page's operands
  unsigned v_bad[4][4];                 // positions whose V is not finite: [group][half of the page]
  int absent[8];                        // the block table names no page
  unsigned seen[2][2][4];               // K's and V's warps: the largest size of their parameters (its bits), all ones: gave up
  int dead;                             // a wait gave up
};

FOX_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A warp's wait: bounded, and at once when another wait of the CTA has given
// up. All lanes poll and leave together, which takes the fewest issue slots from
// the working roles: lanes that leave singly cost 4 % of the kernel's time, a
// longer sleep in the poll 4 % more, one lane polling for the others a quarter.
FOX_DEV bool kv4_warp_wait(Kv4WideBars& b, uint64_t* bar, unsigned parity) {
  unsigned long long since = 0, now;
  for (int i = 1;; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, ok)) return true;
    if (i & 63) continue;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (!since) since = now;
    if (now - since > KV4_WAIT_NS) *reinterpret_cast<volatile int*>(&b.dead) = 1;
    __syncwarp();
    if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&b.dead))) return false;
  }
}
// The first operand in tensor memory: two fp16 a column.
FOX_DEV void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  const uint32_t z = 0;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate), "r"(z), "r"(z), "r"(z), "r"(z)
      : "memory");
}
FOX_DEV void tmem_st8(uint32_t a, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(a), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
FOX_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Whether any of the 256 weight-forming threads says so (their barrier).
FOX_DEV bool kv4_soft_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 256, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}
FOX_DEV void kv4_soft_sync() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }

FOX_DEV bool kv4_elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}

// Two floats in one register pair: one instruction for both.
typedef unsigned long long f32x2;
FOX_DEV f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
FOX_DEV float2 unpack2(f32x2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
FOX_DEV f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 8 codes as fp16 2 c - 15, in the order (0, 4), (1, 5), (2, 6), (3, 7).
FOX_DEV void kv4_centred(uint32_t x, __half2 (&h)[4]) {
  const __half2 off = __half2half2(__ushort_as_half(0x6410));  // 1040
  const uint32_t s[4] = {x << 1, x >> 3, x >> 7, x >> 11};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = (s[i] & 0x001e001eu) | 0x64016401u;  // 1024 + 2 c + 1
    h[i] = __hsub2(*reinterpret_cast<const __half2*>(&u), off);
  }
}
// d c' as hi + lo, exactly.
FOX_DEV void kv4_product(__half2 d, __half2 c, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __hmul2(d, c);
  *hi = half2_bits(h);
  *lo = half2_bits(__hfma2(d, c, __hneg2(h)));
}
// x as hi + lo fp16, 22 bits.
FOX_DEV void kv4_split(float x, __half* hi, __half* lo) {
  *hi = __float2half_rn(x);
  *lo = __float2half_rn(x - __half2float(*hi));
}
// What a page's operands are scaled by, of the size |2 m + 15 d| + 15 |d| of its
// largest group. Unscaled (level 2) they are multiples of 2^-24, and d c' loses
// nothing; pages of small ones leave fp16's subnormal numbers, for which the
// products' sums keep fewer bits (level 3). Large ones must stay below 2^16: with
// values beyond 16384 (level 1) steps are rounded to multiples of 2^-22, so those
// below 2^-12 lose bits; steps beyond 8736, which no write gives, are level 0.
constexpr int KV4_LEVELS = 4;
FOX_DEV int kv4_level(float size) {
  return size < 1.0f / 16.0f ? 3 : size <= 32768.0f ? 2 : size <= 4.0f * 65504.0f ? 1 : 0;
}
FOX_DEV float kv4_scale_of(int level) {
  return level == 3 ? 65536.0f : level == 2 ? 1.0f : level == 1 ? 1.0f / 4.0f : 1.0f / 128.0f;
}

template <int HD, typename T>
__global__ void __launch_bounds__(Kv4Wide<HD>::THREADS, 1) kv4_wide_kernel(const Kv4AttnParams p) {
  using A = Kv4Wide<HD>;
  constexpr int G = A::G, PAIRS = A::PAIRS, OWN = A::OWN;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) Kv4WideBars bars;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gqa = p.n_head / p.c.n_kv;
  constexpr int MMA_WARP = A::MMA_WARP;
  if (tid == 0) {
    for (int i = 0; i < A::RAW; ++i) mbar_init(&bars.raw_full[i], 1);
    for (int i = 0; i < 4; ++i) mbar_init(&bars.k_full[i], MMA_WARP - A::K_WARP);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.v_full[i], A::K_WARP - A::V_WARP);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], A::SOFT / 32);
      mbar_init(&bars.pv_done[i], 1);
    }
    mbar_init(&bars.q_full, A::SOFT / 32);
    mbar_fence_init();
    bars.dead = 0;
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&bars.tmem, A::TMEM);
    tmem_relinquish();
  }
  for (int i = tid * 16; i < A::RAW_AT; i += A::THREADS * 16)  // the operands' rows and columns that stay zero
    *reinterpret_cast<uint4*>(smem + i) = make_uint4(0, 0, 0, 0);
  griddep_wait();
  griddep_launch_dependents();
  Kv4Line line;
  line.build<PAIRS>(p, smem + A::LINE_AT);  // ends with a barrier of the CTA
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  const int ctas = line.ctas(gridDim.x);
  int a0 = 0, a1 = 0;
  if ((int)blockIdx.x < ctas) {
    const Kv4Split split(line.whole ? line.runs : line.U, ctas);
    auto edge = [&](int c) {
      const int x = split.first(c);
      if (!line.whole) return x;
      if (x == line.runs) return line.U;
      const int s = line.find(line.run0, x);
      return line.unit0[s] + (x - line.run0[s]) * kv4_seq<PAIRS>(p, s).units;
    };
    a0 = edge(blockIdx.x);
    a1 = edge(blockIdx.x + 1);
  }

  // A run's part in this CTA's stretch: pages first .. last - 1 that some row
  // of the tile sees. Every role walks the same parts and counts their pages.
  struct Part {
    Kv4Unit x;
    int first, last, lim_max, next;  // next: the unit behind the part
    bool begins, ends;
  };
  auto part_at = [&](int u) {
    Part r;
    r.x.seq = line.find(line.unit0, u);
    r.x.q = kv4_seq<PAIRS>(p, r.x.seq);
    const int at = u - line.unit0[r.x.seq], run = at / r.x.q.units;
    r.x.run = line.run0[r.x.seq] + run;
    r.x.tile = run / p.c.n_kv;
    r.x.kv = run - r.x.tile * p.c.n_kv;
    const int in_run = at - run * r.x.q.units, run_end = u - in_run + r.x.q.units;
    r.x.page = in_run - KV4_HEAD;
    r.next = min(run_end, a1);
    r.begins = in_run == 0;
    r.ends = r.next == run_end;
    r.lim_max = r.x.q.at + min(r.x.q.T - 1, (r.x.tile * PAIRS + PAIRS - 1) / gqa);
    r.first = max(r.x.page, 0);
    r.last = max(r.first, min(r.x.page + (r.next - u), r.lim_max < 0 ? 0 : r.lim_max / KV_PAGE + 1));
    return r;
  };

  if (warp < A::V_WARP) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(A::SOFT_REGS));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(A::OTHER_REGS));

  if (warp < A::V_WARP) {
    // ---- the weights
    static_assert(A::SOFT == 256, "the barriers' count");
    const int share = warp >> 2, pair = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    float4* ex = reinterpret_cast<float4*>(smem + A::EX_AT) + pair;  // [share * PAIRS]
    int j = 0;
    bool ok = true;
    for (int u = a0; u < a1 && ok;) {
      const Part r = part_at(u);
      const int pr = r.x.tile * PAIRS + pair;
      const bool live = pr < r.x.q.T * gqa;
      const int row = live ? pr / gqa : 0, head = r.x.kv * gqa + (live ? pr - row * gqa : 0);
      const int lim = live ? r.x.q.at + row : INT_MAX, lim_min = max(0, r.x.q.at + r.x.tile * PAIRS / gqa);
      float f = 0.0f;
      // q's operand: this thread's OWN dimensions of its pair
      if (r.last > r.first) {
        const T* q = static_cast<const T*>(p.q) + (size_t)(r.x.q.r0 + row) * p.q_stride + (size_t)head * HD + share * OWN;
        float x[OWN], top = 0.0f, sum = 0.0f, qs[G];
#pragma unroll
        for (int i = 0; i < OWN; i += 4) {
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (live) v = kv4_load4(q + i);
          x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < OWN; ++i) { sum = fmaf(x[i], KV4_QSUM, sum); top = fmaxf(top, fabsf(x[i])); }
        ex[share * PAIRS] = make_float4(sum, top, 0.0f, 0.0f);
        kv4_soft_sync();
#pragma unroll
        for (int g = 0; g < G; ++g) qs[g] = 0.0f;
#pragma unroll
        for (int k = 0; k < A::SHARE; ++k) {
          const float4 e = ex[k * PAIRS];
          qs[k * G / A::SHARE] += e.x;
          top = fmaxf(top, e.y);
        }
        // scaled by a power of two to below 2^8: a group's sum stays in range
        const int e = min(7 - ((int)(__float_as_uint(top) >> 23) - 127), 100);
        const float sc = __uint_as_float((uint32_t)(e + 127) << 23);
        f = fminf(p.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - e) << 23), FLT_MAX);
        // The score of a hidden position is -inf times f and a page's unit (2^-16
        // at least), so their product must not fall to zero. No score that this
        // changes exceeds 2^-60: the operands' products stay below 2^40.
        f = fmaxf(f, 0x1p-100f);
#pragma unroll
        for (int c = 0; c < OWN / 16; ++c) {
          constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = 16 * c + 8 * (i / 4);
            const float v0 = x[at + order[2 * (i % 4)]] * sc, v1 = x[at + order[2 * (i % 4) + 1]] * sc;
            const float h0 = __uint_as_float(__float_as_uint(v0) & 0xffffe000u);
            const float h1 = __uint_as_float(__float_as_uint(v1) & 0xffffe000u);
            hi[i] = half2_bits(__floats2half2_rn(h0, h1));
            lo[i] = half2_bits(__floats2half2_rn(v0 - h0, v1 - h1));
          }
          tmem_st8(tmem + lanes + A::Q_COL + share * (OWN / 2) + 8 * c, hi);
          tmem_st8(tmem + lanes + A::Q_COL + HD / 2 + share * (OWN / 2) + 8 * c, lo);
        }
        if (share == 0) {  // against K's offsets (hi, hi, lo) of each group
          __half h[2], l[2];
          h[1] = l[1] = __ushort_as_half(0);
#pragma unroll
          for (int g = 0; g < G; ++g) kv4_split(qs[g] * (sc / KV4_QSUM), &h[g], &l[g]);
          const uint32_t m[8] = {half2_bits(__halves2half2(h[0], l[0])), half2_bits(__halves2half2(h[0], h[1])),
                                 half2_bits(__halves2half2(l[1], h[1])), 0, 0, 0, 0, 0};
          tmem_st8(tmem + lanes + A::QM_COL, m);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full);
      }
      float o[OWN], off = 0.0f, mx = -INFINITY, l = 0.0f, unit = 1.0f;
#pragma unroll
      for (int i = 0; i < OWN; ++i) o[i] = 0.0f;
      int since = 0;     // pages in tensor memory's sums
      unsigned nan = 0;  // groups whose V was not finite
      auto take_sums = [&]() {  // O of the pages up to j - 1, into the registers
        if (since && !kv4_warp_wait(bars, &bars.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1)) ok = false;
        if (!since || !ok) return;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < OWN; c += 16) {
          uint32_t v[16];
          TmemLd<16>::run(tmem + lanes + A::O_COL + share * OWN + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[c + i] += __uint_as_float(v[i]);
        }
        uint32_t m[4];  // the offsets' sums of both groups
        TmemLd<4>::run(tmem + lanes + A::O_COL + HD, m);
        tmem_wait_ld();
        const bool second = share * G / A::SHARE;
        off += __uint_as_float(second ? m[2] : m[0]) + __uint_as_float(second ? m[3] : m[1]);
        tc_fence_before();
        since = 0;
      };
      for (int page = r.first; page < r.last; ++page, ++j) {
        const int b = j & 1, pos0 = page * KV_PAGE + share * A::POS;
        const unsigned ph = (j >> 1) & 1;
        ok = kv4_warp_wait(bars, &bars.k_full[j & 3], (j >> 2) & 1) && kv4_warp_wait(bars, &bars.v_full[b], ph) &&
             kv4_warp_wait(bars, &bars.s_full[b], ph);
        tc_fence_after();
        const uint32_t s_at = tmem + lanes + b * KV_PAGE;
        const float fj = f * bars.k_unit[j & 3], new_unit = bars.v_unit[j & 3];
        const bool absent = bars.absent[j & 7], edge = absent || page * KV_PAGE + KV_PAGE - 1 > lim_min;
        uint32_t d[A::POS];
        float top = -INFINITY;
        if (ok) {
          TmemLd<A::POS>::run(s_at + share * A::POS, d);
          tmem_wait_ld();
          if (edge) {
#pragma unroll
            for (int i = 0; i < A::POS; ++i)
              if (absent || pos0 + i > lim) d[i] = 0xff800000u;  // -inf: hidden
          }
#pragma unroll
          for (int i = 0; i < A::POS; ++i) top = fmaxf(top, __uint_as_float(d[i]));
          top *= fj;
        }
        // the barrier of this vote also stands between the scores' loads and the weights' stores
        if (kv4_soft_any(!ok || new_unit != unit || top > mx + KV4_SLACK || since == KV4_WIDE_FLUSH)) {
          if (*reinterpret_cast<volatile int*>(&bars.dead)) ok = false;
          take_sums();
          ex[share * PAIRS] = make_float4(top, 0.0f, 0.0f, 0.0f);
          if (kv4_soft_any(!ok)) { ok = false; break; }
          float m = mx;
#pragma unroll
          for (int k = 0; k < A::SHARE; ++k) m = fmaxf(m, ex[k * PAIRS].x);
          const float al = m == -INFINITY ? 1.0f : exp2_approx(mx - m), all = al * (unit / new_unit);
          mx = m;
          unit = new_unit;
          l *= al;
          off *= all;
#pragma unroll
          for (int i = 0; i < OWN; ++i) o[i] *= all;
        }
        if (tid == 0) bars.fresh[b] = since == 0;
        // Weights are scaled by 2^7, out of fp16's small numbers; with the slack
        // they reach 2^14. The product is rounded before the sum, as the
        // reference point was, so that the largest of scores of any size has a
        // weight of 1 to 2^14: a fused one differed from it by more than 2^7
        // from scores of 10^8 on. (7 - mx, rounded, is off by less than 4 where
        // scores are that coarse, and those above mx by no more than the slack
        // are then equal to it.)
        const float base = 7.0f - (mx == -INFINITY ? 0.0f : mx);
        static_assert(KV4_SLACK == 7.0f, "2^14, and not fp16's 2^16");
        uint32_t hi[A::POS / 2], lo[A::POS / 2];
        f32x2 l2 = 0;
#pragma unroll
        for (int i = 0; i < A::POS; i += 2) {
          // (a packed product and sum were fused by the assembler; these are not)
          const float w0 = exp2_approx(__fadd_rn(__fmul_rn(__uint_as_float(d[i]), fj), base));
          const float w1 = exp2_approx(__fadd_rn(__fmul_rn(__uint_as_float(d[i + 1]), fj), base));
          l2 = add2(l2, pack2(w0, w1));
          const float h0 = __uint_as_float(__float_as_uint(w0) & 0xffffe000u), h1 = __uint_as_float(__float_as_uint(w1) & 0xffffe000u);
          const float2 r = unpack2(add2(pack2(w0, w1), pack2(-h0, -h1)));
          hi[i / 2] = half2_bits(__floats2half2_rn(h0, h1));
          lo[i / 2] = half2_bits(__floats2half2_rn(r.x, r.y));
        }
        l += unpack2(l2).x + unpack2(l2).y;
#pragma unroll
        for (int c = 0; c < A::POS / 2; c += 8) {
          const uint32_t(&h)[8] = *reinterpret_cast<const uint32_t(*)[8]>(hi + c);
          const uint32_t(&q)[8] = *reinterpret_cast<const uint32_t(*)[8]>(lo + c);
          tmem_st8(s_at + share * (A::POS / 2) + c, h);
          tmem_st8(s_at + KV_PAGE / 2 + share * (A::POS / 2) + c, q);
        }
        // V that is not finite was left out of the product: it reaches who sees it here
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const unsigned bad = bars.v_bad[j & 3][2 * g + share];
          if (bad) {
#pragma unroll
            for (int i = 0; i < A::POS; ++i)
              if ((bad >> i & 1) && d[i] != 0xff800000u) nan |= 1u << g;
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[b]);
        ++since;
      }
      take_sums();
      ex[share * PAIRS] = make_float4(l, __uint_as_float(nan), 0.0f, 0.0f);
      if (kv4_soft_any(!ok)) { ok = false; break; }
      float total = 0.0f;
#pragma unroll
      for (int k = 0; k < A::SHARE; ++k) {
        total += ex[k * PAIRS].x;
        nan |= __float_as_uint(ex[k * PAIRS].y);
      }
      if (nan >> (share * G / A::SHARE) & 1) off = CUDART_NAN_F;
      kv4_soft_sync();  // the exchange is free
      if (live) {
        T* out = static_cast<T*>(p.out) + ((size_t)(r.x.q.r0 + row) * p.n_head + head) * HD + share * OWN;
        float* dst = p.part + (((size_t)blockIdx.x * 2 + r.begins) * PAIRS + pair) * A::PART;
        const bool whole = r.begins && r.ends;
        if (!whole && share == 0) *reinterpret_cast<float2*>(dst) = make_float2(mx, total);
#pragma unroll
        for (int i = 0; i < OWN; i += 4) {
          const float4 v = make_float4((o[i] + off) * unit, (o[i + 1] + off) * unit, (o[i + 2] + off) * unit, (o[i + 3] + off) * unit);
          if (whole) kv4_store4(out + i, kv4_quotient(v, total));
          else *reinterpret_cast<float4*>(dst + 4 + share * OWN + i) = v;
        }
      }
      u = r.next;
    }
    if (!ok && tid == 0 && p.c.err) atomicOr(p.c.err, KERR_WAIT);
  } else if (warp < MMA_WARP) {
    // ---- a page's operands. Their loops stay rolled: four roles share a
    // scheduler's instruction cache, and copies of the bodies cost 6 %.
    const int side = warp < A::K_WARP, t0 = tid - (side ? A::V_WARP : A::K_WARP) * 32;  // K 0, V 1
    constexpr int NK = (MMA_WARP - A::K_WARP) * 32, NV = (A::K_WARP - A::V_WARP) * 32, EACH = (KV_PAGE * G + NK - 1) / NK;
    static_assert(KV_PAGE * G <= NV, "a thread for each position and group of V");
    const int n = side ? NV : NK;
    uint64_t* freed = side ? bars.pv_done : bars.s_full;  // the products that used the buffers last
    auto sync = [&]() {
      if (side) asm volatile("barrier.cta.sync 3, %0;" ::"n"(NV) : "memory");
      else asm volatile("barrier.cta.sync 2, %0;" ::"n"(NK) : "memory");
    };
    int j = 0;
    bool ok = true;
    for (int u = a0; u < a1 && ok;) {
      const Part r = part_at(u);
      int level = KV4_LEVELS - 1;  // V's only falls within a run: its sums have one scale
      for (int page = r.first; page < r.last; ++page, ++j) {
        const int b = j & 1, left = r.lim_max - page * KV_PAGE;  // positions 0 .. left of the page are seen
        const uint8_t* raw = smem + A::RAW_AT + (j % A::RAW) * A::PAGE_BYTES + side * A::BB;
        uint8_t* tile = smem + (side ? A::V_AT + b * A::V_BYTES : A::K_AT + b * A::K_BYTES);
        __half* dd = reinterpret_cast<__half*>(smem + A::D_AT) + (side * 2 + b) * G * KV_PAGE;  // [group][position]
        ok = kv4_warp_wait(bars, &bars.raw_full[j % A::RAW], (j / A::RAW) & 1) &&
             (j < 2 || kv4_warp_wait(bars, &freed[b], ((j - 2) >> 1) & 1));
        // the parameters: position i % 64 of group i / 64; zero where the
        // position is nobody's, whatever the memory held
        float d[EACH], off[EACH];
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
          const int i = t0 + k * n, pos = i % KV_PAGE, g = i / KV_PAGE;
          bool bad = false;
          d[k] = off[k] = 0.0f;
          if (ok && g < G && !bars.absent[j & 7] && pos <= left) {
            const float2 dm = __half22float2(reinterpret_cast<const __half2*>(raw + kv4_codes_bytes(HD))[pos * G + g]);
            d[k] = dm.x;
            off[k] = fmaf(15.0f, dm.x, 2.0f * dm.y);
            const float size = fmaf(15.0f, fabsf(d[k]), fabsf(off[k]));
            bad = !(size < 1e30f);  // not finite
            if (!bad) top = fmaxf(top, size);
            else if (side) d[k] = off[k] = 0.0f;
          }
          const unsigned bads = __ballot_sync(0xffffffffu, bad);
          if (side && k == 0 && lane == 0) bars.v_bad[j & 3][warp & 3] = bads;
        }
        auto store = [&]() {
          const float sc = kv4_scale_of(level);
#pragma unroll
          for (int k = 0; k < EACH; ++k) {
            const int i = t0 + k * n, pos = i % KV_PAGE, g = i / KV_PAGE;
            if (g >= G) continue;
            __half hi, lo;
            dd[i] = __float2half_rn(d[k] * sc);
            kv4_split(off[k] * sc, &hi, &lo);
            if (side) {  // rows HD + 2 g (hi) and the next (lo)
              __half* m = reinterpret_cast<__half*>(tile + HD / 8 * A::SBO + pos / 8 * A::LBO + 2 * g * 16) + pos % 8;
              m[0] = hi;
              m[8] = lo;
            } else {     // hi, hi, lo: against q's sum's hi, lo, hi
              __half* m = reinterpret_cast<__half*>(tile + A::KM_AT + pos / 8 * A::KM_SBO + pos % 8 * 16) + 3 * g;
              m[0] = hi;
              m[1] = hi;
              m[2] = lo;
            }
          }
          if (t0 == 0) (side ? bars.v_unit : bars.k_unit)[j & 3] = 0.5f / sc;
        };
        // as the last page's, until all have been seen
        if (ok) store();
        const unsigned seen = __reduce_max_sync(0xffffffffu, __float_as_uint(top));  // (never negative)
        if (lane == 0) bars.seen[side][b][warp & 3] = ok ? seen : ~0u;
        sync();
        unsigned all = 0;
        for (int k = 0; k < n / 32; ++k) all = max(all, bars.seen[side][b][k]);
        if (all == ~0u) { ok = false; break; }
        const int now = min(side ? level : KV4_LEVELS - 1, kv4_level(__uint_as_float(all)));
        if (now != level) {
          level = now;
          store();
          sync();
        }
        if (!side) {
#pragma unroll 1
          for (int k = 0; k < (KV_PAGE * 4 + NK - 1) / NK; ++k) {  // position i / 4, 16 dimensions of every group
            const int i = t0 + k * NK;
            if (i >= KV_PAGE * 4) break;
            const int pos = i >> 2, t = i & 3;
            uint32_t w[2 * G];
            if constexpr (G == 2) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(raw + i * 16);
            else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(raw + i * 8);
#pragma unroll
            for (int x = 0; x < 2 * G; ++x) {
              const __half2 d = __half2half2(dd[x / 2 * KV_PAGE + pos]);
              __half2 c[4];
              uint32_t hi[4], lo[4];
              kv4_centred(w[x], c);
#pragma unroll
              for (int z = 0; z < 4; ++z) kv4_product(d, c[z], &hi[z], &lo[z]);
              uint8_t* dst = tile + x / 2 * A::TILE + pos / 8 * A::SBO + (2 * t + x % 2) * A::LBO + pos % 8 * 16;
              *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              *reinterpret_cast<uint4*>(dst + A::K_HALF) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < G; ++k) {  // 4 dimensions (g) of a block of 32, 8 positions
            const int i = t0 + k * NV, g = i & 7, blk = i / 8 % (2 * G), chunk = i / (16 * G);
            const uint4 d4 = *reinterpret_cast<const uint4*>(dd + blk / 2 * KV_PAGE + chunk * 8);
            const uint32_t d[4] = {d4.x, d4.y, d4.z, d4.w};
            uint32_t hi[4][4], lo[4][4];  // [dimension][pair of positions]
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              __half2 c[4];
              kv4_centred(*reinterpret_cast<const uint32_t*>(raw + ((chunk * 4 + t) * 8 + g) * (8 * G) + 4 * blk), c);
#pragma unroll
              for (int z = 0; z < 4; ++z) kv4_product(*reinterpret_cast<const __half2*>(&d[t]), c[z], &hi[z][t], &lo[z][t]);
            }
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const int dim = blk * 32 + 4 * g + z;
              uint8_t* dst = tile + dim / 8 * A::SBO + chunk * A::LBO + dim % 8 * 16;
              *reinterpret_cast<uint4*>(dst) = make_uint4(hi[z][0], hi[z][1], hi[z][2], hi[z][3]);
              *reinterpret_cast<uint4*>(dst + A::V_LO) = make_uint4(lo[z][0], lo[z][1], lo[z][2], lo[z][3]);
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(side ? &bars.v_full[b] : &bars.k_full[j & 3]);
      }
      u = r.next;
    }
  } else {
    // ---- the loads and the products. The whole warp walks (its values stay in
    // uniform registers, which the instructions want them in), one lane issues.
    const bool leader = kv4_elect();
    // fp32 sums of fp16, both along the contraction: N columns
    constexpr auto idesc = [](int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(PAIRS >> 4) << 24); };
    constexpr uint32_t S_DESC = idesc(KV_PAGE), O_DESC = idesc(A::V_ROWS), O_LO_DESC = idesc(HD);
    int pages = 0;  // of the whole stretch
    for (int u = a0; u < a1;) {
      const Part r = part_at(u);
      pages += r.last - r.first;
      u = r.next;
    }
    // the load cursor runs ahead of the products, and the block table's entry
    // ahead of the load
    int lu = a0, lp = 0, loaded = 0, next = -1;
    Part lr;
    if (a0 < a1) { lr = part_at(a0); lp = lr.first; }
    auto look = [&]() {
      if (loaded >= pages) return;
      while (lp >= lr.last) {
        lu = lr.next;
        lr = part_at(lu);
        lp = lr.first;
      }
      next = __ldg(p.c.table + (size_t)lr.x.seq * p.c.table_stride + lp);  // looked at when it is used
    };
    auto load = [&]() {
      uint64_t* bar = &bars.raw_full[loaded % A::RAW];
      // a page outside the cache is not read: its positions count for nothing
      const bool there = (unsigned)next < (unsigned)p.c.n_pages;
      if (leader) {
        bars.absent[loaded & 7] = !there;
        mbar_arrive_expect_tx(bar, there ? A::PAGE_BYTES : 0);
        if (!there) kv4_outside(p.c);
      }
      if (leader && there)
        bulk_g2s(smem + A::RAW_AT + (loaded % A::RAW) * A::PAGE_BYTES, kv4_block(p.c, next, lr.x.kv, 0, A::BB), A::PAGE_BYTES, bar);
      ++lp;
      ++loaded;
      look();
    };
    look();
    while (loaded < min(pages, A::RAW)) load();
    const uint32_t k0 = smem_u32(smem + A::K_AT), v0 = smem_u32(smem + A::V_AT);
    int j = 0, runs = 0, done = -1;
    bool ok = true;
    auto pv = [&](int i) {  // O += P . V of page i
      const int b = i & 1;
      const unsigned ph = (i >> 1) & 1;
      ok = ok && kv4_warp_wait(bars, &bars.v_full[b], ph) && kv4_warp_wait(bars, &bars.p_full[b], ph);
      if (!ok) return;
      tc_fence_after();
      const uint32_t add = *reinterpret_cast<volatile int*>(&bars.fresh[b]) ? 0u : 1u;
      if (leader) {
        const uint64_t v = umma_desc(v0 + b * A::V_BYTES, A::LBO, A::SBO);
        const uint32_t o_at = tmem + A::O_COL, p_at = tmem + b * KV_PAGE;
#pragma unroll
        for (int s = 0; s < 4; ++s) {  // 16 positions each
          const uint64_t vs = v + ((s * 2 * A::LBO) >> 4);
          mma_f16_ts(o_at, p_at + s * 8, vs, O_DESC, s ? 1u : add);
          mma_f16_ts(o_at, p_at + KV_PAGE / 2 + s * 8, vs, O_DESC, 1u);
          mma_f16_ts(o_at, p_at + s * 8, vs + (A::V_LO >> 4), O_LO_DESC, 1u);
        }
        mma_commit(&bars.pv_done[b]);
      }
      done = i;
      if (loaded < pages) load();  // the slot of page i: its codes have been unpacked
    };
    for (int u = a0; u < a1 && ok;) {
      const Part r = part_at(u);
      for (int page = r.first; page < r.last && ok; ++page, ++j) {
        const int b = j & 1;
        if (page == r.first) {  // the queries change once the last run's sums are taken
          if (j) pv(j - 1);
          ok = ok && kv4_warp_wait(bars, &bars.q_full, runs & 1);
          ++runs;
        }
        // (the buffer's last weights were used by the products of page j - 2)
        ok = ok && kv4_warp_wait(bars, &bars.k_full[j & 3], (j >> 2) & 1) && (j < 2 || kv4_warp_wait(bars, &bars.pv_done[b], ((j - 2) >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint64_t k = umma_desc(k0 + b * A::K_BYTES, A::LBO, A::SBO);
          const uint32_t s_at = tmem + b * KV_PAGE, q_at = tmem + A::Q_COL;
#pragma unroll
          for (int s = 0; s < HD / 16; ++s) {  // 16 dimensions each, the small terms first
            const uint64_t ks = k + ((s / 4 * A::TILE + s % 4 * 2 * A::LBO) >> 4);
            mma_f16_ts(s_at, q_at + HD / 2 + s * 8, ks, S_DESC, s ? 1u : 0u);
            mma_f16_ts(s_at, q_at + s * 8, ks + (A::K_HALF >> 4), S_DESC, 1u);
          }
#pragma unroll
          for (int s = 0; s < HD / 16; ++s)
            mma_f16_ts(s_at, q_at + s * 8, k + ((s / 4 * A::TILE + s % 4 * 2 * A::LBO) >> 4), S_DESC, 1u);
          mma_f16_ts(s_at, tmem + A::QM_COL, umma_desc(k0 + b * A::K_BYTES + A::KM_AT, A::LBO, A::KM_SBO), S_DESC, 1u);
          mma_commit(&bars.s_full[b]);
        }
        if (page > r.first) pv(j - 1);
      }
      u = r.next;
    }
    if (ok && j) pv(j - 1);
    // copies and products in flight end before the CTA does
    if (done >= 0) mbar_wait(&bars.pv_done[done & 1], (done >> 1) & 1);
    if (!ok) {
      for (int i = 0; i < 2; ++i) { mbar_wait(&bars.s_full[i], 0); mbar_wait(&bars.s_full[i], 1); }
      for (int i = 0; i < min(loaded, A::RAW); ++i) mbar_wait(&bars.raw_full[(loaded - 1 - i) % A::RAW], ((loaded - 1 - i) / A::RAW) & 1);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, A::TMEM);
}

}  // namespace fox
