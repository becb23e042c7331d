// Attention over the 4-bit cache for many rows of a sequence (sm_100a): the
// mathematics of kv4_attn.cuh with both products on the 5th-generation tensor
// cores (tcgen05 kind::f16, fp32 sums in tensor memory).
//
// A CTA takes 128 (row, head) pairs of a KV head (the products' 128 rows) and
// walks their pages; its warps have roles:
// - 4 warps unpack a page's K codes and 2 its V codes to fp16 2 c - 15 (exact;
//   centred, so the sums stay near their results) as the products' second operands: K [position]
//   [dimension], V [dimension][position], in 8 x 16-byte core matrices whose
//   strides keep the stores free of bank conflicts. The positions' parameters
//   are laid out as (d / 2, m + 7.5 d) in fp32, V's by a warp of its own.
// - 1 thread loads pages and issues the products: S_g = Q_g . K_g^T for each
//   group g of 64 dimensions, q as hi + lo fp16 (the two add up in one
//   accumulator), and O_g += P_g . V_g^T, P_g = p d_g as hi + lo fp16, which
//   replaces S_g in tensor memory. The scores of page j + 1 are formed while
//   page j's weights are.
// - 8 warps form the weights: two threads share a pair, each with half of the
//   page's positions and of the pair's sums, and hold most of the registers.
//   The reference point of a pair's weights moves only when a score
//   passes it by 2^KV4_SLACK; then, and every KV4_WIDE_FLUSH pages, O leaves
//   tensor memory for the thread's registers, which bounds what the products'
//   rounding toward zero adds up to.
// The work is divided as in kv4_attn.cuh, with a CTA for a warp.
#pragma once

#include "kv4_attn.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace fox {

constexpr int KV4_WIDE_PAIRS = 128, KV4_WIDE_FLUSH = 8;

template <int HD>
struct Kv4Wide {
  static constexpr int G = HD / KV4_GROUP, BB = kv4_block_bytes(HD), PAGE_BYTES = 2 * BB, PART = HD + 4;
  static constexpr int SHARE = 2, OWN = HD / SHARE, POS = KV_PAGE / SHARE;  // threads of a pair; their dimensions and positions
  static constexpr int PAIRS = KV4_WIDE_PAIRS, SOFT = PAIRS * SHARE, THREADS = 512;
  // second operands: 64 rows x 64 fp16, 8 core matrices along each side; one
  // step along the contraction is 144 bytes, eight rows 1168
  static constexpr int LBO = 144, SBO = 8 * LBO + 16, TILE = 8 * SBO;
  static constexpr int QLBO = 128, QSBO = 1024, QTILE = PAIRS / 8 * QSBO;  // the first: 128 rows x 64 fp16
  // tensor memory's columns: S of two pages, O, the page's scores
  static constexpr int S_COLS = 64 * G, O_COL = 2 * S_COLS, SCORE_COL = O_COL + HD, TMEM = HD == 64 ? 256 : 512;
  static_assert(SCORE_COL + KV_PAGE <= TMEM, "what is allocated");
  // warps by role, in groups of four that share a number of registers: 128 a
  // thread at launch, 8 x 176 + 8 x 80 = 16 x 128
  static constexpr int K_WARP = 8, V_WARP = 12, V_PAR_WARP = 14, MMA_WARP = 15;
  static constexpr int SOFT_REGS = 176, OTHER_REGS = 80;
  static constexpr int RAW = 3, PAR = 4;  // pages loaded ahead; pages whose parameters are kept
  // shared memory
  static constexpr int Q_AT = 0, K_AT = Q_AT + 2 * G * QTILE, V_AT = K_AT + 2 * G * TILE, RAW_AT = V_AT + 2 * G * TILE;
  static constexpr int PAR_AT = RAW_AT + RAW * PAGE_BYTES, PAR_BYTES = 2 * KV_PAGE * G * 8;  // [K, V][group][d / 2, m + 7.5 d][position] floats
  static constexpr int EX_AT = PAR_AT + PAR * PAR_BYTES;                                    // the sharing threads' exchange: [SHARE][PAIRS] float4
  static constexpr int LINE_AT = EX_AT + SOFT * 16;
  static size_t smem_bytes(int n_seq) { return LINE_AT + Kv4Line::bytes(n_seq); }
};

struct Kv4WideBars {
  uint64_t raw_full[3], k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2], q_full;
  uint32_t tmem;
  int fresh[2];    // the page's O does not add to what tensor memory holds
  float vmax[4];   // the page's largest d of V
  int absent[4];   // the block table names no page
  int dead;        // a wait gave up
};

FOX_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Bounded, and at once when another wait of the CTA has given up. A poll may
// sleep in the barrier's unit for up to 20 us, so that the waiting roles leave
// the schedulers to the working ones.
FOX_DEV bool kv4_wait(Kv4WideBars& b, uint64_t* bar, unsigned parity) {
  for (int i = 0; i < (1 << 16); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (*reinterpret_cast<volatile int*>(&b.dead)) return false;
  }
  *reinterpret_cast<volatile int*>(&b.dead) = 1;
  return false;
}
// The same by a warp. Every lane polls: one polling for the others was slower
// by a quarter of the kernel's time.
FOX_DEV bool kv4_warp_wait(Kv4WideBars& b, uint64_t* bar, unsigned parity) {
  return __all_sync(0xffffffffu, kv4_wait(b, bar, parity));
}
FOX_DEV void mma_f16(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  const uint32_t z = 0;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(z), "r"(z), "r"(z), "r"(z)
      : "memory");
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
FOX_DEV void tmem_st16(uint32_t a, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
FOX_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Whether any of the 256 weight-forming threads says so (their barrier).
FOX_DEV bool kv4_any(bool x) {
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
FOX_DEV f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
FOX_DEV f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 8 codes as fp16 2 c - 15, in the order (0, 4), (1, 5), (2, 6), (3, 7).
FOX_DEV void kv4_centred(uint32_t x, uint32_t (&h)[4]) {
  const __half2 off = __half2half2(__ushort_as_half(0x6410));  // 1040
  const uint32_t s[4] = {x << 1, x >> 3, x >> 7, x >> 11};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = (s[i] & 0x001e001eu) | 0x64016401u;  // 1024 + 2 c + 1
    h[i] = half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&u), off));
  }
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
    for (int i = 0; i < 3; ++i) mbar_init(&bars.raw_full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], A::V_WARP - A::K_WARP);
      mbar_init(&bars.v_full[i], MMA_WARP - A::V_WARP);
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
  griddep_wait();
  griddep_launch_dependents();
  Kv4Line line;
  line.build<PAIRS>(p, smem + A::LINE_AT);  // ends with a barrier of the CTA
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
    r.lim_max = r.x.q.L - r.x.q.T + min(r.x.q.T - 1, (r.x.tile * PAIRS + PAIRS - 1) / gqa);
    r.first = max(r.x.page, 0);
    r.last = max(r.first, min(r.x.page + (r.next - u), r.lim_max < 0 ? 0 : r.lim_max / KV_PAGE + 1));
    return r;
  };

  if (warp < A::K_WARP) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(A::SOFT_REGS));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(A::OTHER_REGS));

  if (warp < A::K_WARP) {
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
      const int lim = live ? r.x.q.L - r.x.q.T + row : INT_MAX, lim_min = max(0, r.x.q.L - r.x.q.T + r.x.tile * PAIRS / gqa);
      float f = 0.0f, qs[G];
      // q's operand: this thread's OWN dimensions of its pair
      if (r.last > r.first) {
        const T* q = static_cast<const T*>(p.q) + (size_t)(r.x.q.r0 + row) * p.q_stride + (size_t)head * HD + share * OWN;
        float x[OWN], top = 0.0f, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < OWN; i += 4) {
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (live) v = kv4_load4(q + i);
          x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < OWN; ++i) { sum += x[i]; top = fmaxf(top, fabsf(x[i])); }
        ex[share * PAIRS] = make_float4(sum, top, 0.0f, 0.0f);
        kv4_soft_sync();
        const float unit = p.scale * 1.44269504088896341f;
#pragma unroll
        for (int g = 0; g < G; ++g) qs[g] = 0.0f;
#pragma unroll
        for (int k = 0; k < A::SHARE; ++k) {
          const float4 e = ex[k * PAIRS];
          qs[k * G / A::SHARE] += e.x;
          top = fmaxf(top, e.y);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) qs[g] *= unit;
        const int e = min(max(13 - ((int)(__float_as_uint(top) >> 23) - 127), -100), 100);
        const float sc = __uint_as_float((uint32_t)(e + 127) << 23);
        f = unit * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int c = 0; c < OWN / 8; ++c) {
          constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v0 = x[8 * c + order[2 * i]] * sc, v1 = x[8 * c + order[2 * i + 1]] * sc;
            const float h0 = __uint_as_float(__float_as_uint(v0) & 0xffffe000u);
            const float h1 = __uint_as_float(__float_as_uint(v1) & 0xffffe000u);
            hi[i] = half2_bits(__floats2half2_rn(h0, h1));
            lo[i] = half2_bits(__floats2half2_rn(v0 - h0, v1 - h1));
          }
          const int d = share * OWN + 8 * c, at = d / 64 * A::QTILE + pair / 8 * A::QSBO + d % 64 / 8 * A::QLBO + pair % 8 * 16;
          *reinterpret_cast<uint4*>(smem + A::Q_AT + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(smem + A::Q_AT + G * A::QTILE + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full);
      }
      float o[OWN], mx = -INFINITY, big = 0x1p-24f;
      f32x2 l = 0, mo[G];  // of every other position
#pragma unroll
      for (int i = 0; i < OWN; ++i) o[i] = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) mo[g] = 0;
      int since = 0;  // pages in tensor memory's sums
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
        tc_fence_before();
        since = 0;
      };
      for (int page = r.first; page < r.last; ++page, ++j) {
        const int b = j & 1, pos0 = page * KV_PAGE + share * A::POS;
        const unsigned ph = (j >> 1) & 1;
        ok = kv4_warp_wait(bars, &bars.k_full[b], ph) && kv4_warp_wait(bars, &bars.v_full[b], ph) &&
             kv4_warp_wait(bars, &bars.s_full[b], ph);
        tc_fence_after();
        // this thread's positions' parameters: K's, then V's; four at once
        const float* kp = reinterpret_cast<const float*>(smem + A::PAR_AT + (j & 3) * A::PAR_BYTES) + share * A::POS;
        const float* vp = kp + 2 * G * KV_PAGE;
        auto par4 = [](const float* p) { return *reinterpret_cast<const ulonglong2*>(p); };
        const uint32_t s_at = tmem + lanes + b * A::S_COLS;
        const bool absent = bars.absent[j & 3], edge = absent || page * KV_PAGE + KV_PAGE - 1 > lim_min;
        const uint32_t mine = tmem + lanes + A::SCORE_COL + share * A::POS;
        float top = -INFINITY;
        // Rolled loops, the scores parked in tensor memory in between: so the
        // instruction cache holds all roles' code.
        auto scores = [&](auto at_edge) {
#pragma unroll 1
          for (int c = 0; c < A::POS; c += 16) {
            uint32_t d[G][16];
#pragma unroll
            for (int g = 0; g < G; ++g) TmemLd<16>::run(s_at + g * 64 + share * A::POS + c, d[g]);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              f32x2 prod[2], off[2];
#pragma unroll
              for (int g = 0; g < G; ++g) {
                const ulonglong2 dd = par4(kp + 2 * g * KV_PAGE + c + i), mm = par4(kp + (2 * g + 1) * KV_PAGE + c + i);
                const f32x2 q2 = pack2(qs[g], qs[g]), dk[2] = {dd.x, dd.y}, mk[2] = {mm.x, mm.y};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const f32x2 x = pack2(__uint_as_float(d[g][i + 2 * k]), __uint_as_float(d[g][i + 2 * k + 1]));
                  prod[k] = g ? fma2(dk[k], x, prod[k]) : mul2(dk[k], x);
                  off[k] = g ? fma2(mk[k], q2, off[k]) : mul2(mk[k], q2);
                }
              }
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float2 s = unpack2(fma2(pack2(f, f), prod[k], off[k]));
                const int at = pos0 + c + i + 2 * k;
                if (at_edge.value && (absent || at > lim)) s.x = -INFINITY;
                if (at_edge.value && (absent || at + 1 > lim)) s.y = -INFINITY;
                top = fmaxf(top, fmaxf(s.x, s.y));
                d[0][i + 2 * k] = __float_as_uint(s.x);
                d[0][i + 2 * k + 1] = __float_as_uint(s.y);
              }
            }
            tmem_st16(mine + c, d[0]);
          }
          tmem_wait_st();
        };
        if (ok) {
          if (edge) scores(std::true_type());
          else scores(std::false_type());
        }
        const float dmax = bars.vmax[j & 3];
        // the barrier of this vote also stands between the scores' loads and the weights' stores
        if (kv4_any(!ok || dmax >= big || top > mx + KV4_SLACK || since == KV4_WIDE_FLUSH)) {
          if (*reinterpret_cast<volatile int*>(&bars.dead)) ok = false;
          take_sums();
          ex[share * PAIRS] = make_float4(top, 0.0f, 0.0f, 0.0f);
          if (kv4_any(!ok)) { ok = false; break; }
          float m = mx;
#pragma unroll
          for (int k = 0; k < A::SHARE; ++k) m = fmaxf(m, ex[k * PAIRS].x);
          const float to = dmax >= big ? __uint_as_float((__float_as_uint(dmax) & 0x7f800000u) + 0x00800000u) : big;
          const float al = m == -INFINITY ? 1.0f : exp2_approx(mx - m), all = al * (big / to);
          mx = m;
          big = to;
          l = mul2(l, pack2(al, al));
#pragma unroll
          for (int g = 0; g < G; ++g) mo[g] = mul2(mo[g], pack2(al, al));
#pragma unroll
          for (int i = 0; i < OWN; ++i) o[i] *= all;
        }
        if (tid == 0) bars.fresh[b] = since == 0;
        const float norm = KV4_WEIGHT / big, base = mx == -INFINITY ? 0.0f : mx;
        auto weights = [&](auto at_edge) {
#pragma unroll 1
          for (int c = 0; c < A::POS; c += 16) {
            uint32_t s[16], hi[G][8], lo[G][8];
            TmemLd<16>::run(mine + c, s);
            tmem_wait_ld();
            const f32x2 below = pack2(-base, -base), norm2 = pack2(norm, norm);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              f32x2 w[2], wn[2];
              bool hidden[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)  // whatever the position holds
                hidden[k] = at_edge.value && __uint_as_float(s[i + k]) == -INFINITY;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float2 x = unpack2(add2(pack2(__uint_as_float(s[i + 2 * k]), __uint_as_float(s[i + 2 * k + 1])), below));
                w[k] = pack2(exp2_approx(x.x), exp2_approx(x.y));
                wn[k] = mul2(w[k], norm2);
                l = add2(l, w[k]);
              }
#pragma unroll
              for (int g = 0; g < G; ++g) {
                const ulonglong2 dd = par4(vp + 2 * g * KV_PAGE + c + i), mm = par4(vp + (2 * g + 1) * KV_PAGE + c + i);
                const f32x2 dk[2] = {dd.x, dd.y};
                f32x2 mk[2] = {mm.x, mm.y};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  float2 v = unpack2(mul2(wn[k], dk[k]));
                  if (at_edge.value) {
                    float2 m = unpack2(mk[k]);
                    if (hidden[2 * k]) v.x = m.x = 0.0f;
                    if (hidden[2 * k + 1]) v.y = m.y = 0.0f;
                    mk[k] = pack2(m.x, m.y);
                  }
                  mo[g] = fma2(w[k], mk[k], mo[g]);
                  const float h0 = __uint_as_float(__float_as_uint(v.x) & 0xffffe000u);
                  const float h1 = __uint_as_float(__float_as_uint(v.y) & 0xffffe000u);
                  const float2 rest = unpack2(add2(pack2(v.x, v.y), pack2(-h0, -h1)));
                  hi[g][i / 2 + k] = half2_bits(__floats2half2_rn(h0, h1));
                  lo[g][i / 2 + k] = half2_bits(__floats2half2_rn(rest.x, rest.y));
                }
              }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
              tmem_st8(s_at + g * 64 + (share * A::POS + c) / 2, hi[g]);
              tmem_st8(s_at + g * 64 + 32 + (share * A::POS + c) / 2, lo[g]);
            }
          }
        };
        if (edge) weights(std::true_type());
        else weights(std::false_type());
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[b]);
        ++since;
      }
      take_sums();
      // the shares of l and the offsets, and the result
      {
        const float2 a = unpack2(l), m0 = unpack2(mo[0]), m1 = unpack2(mo[G - 1]);
        ex[share * PAIRS] = make_float4(a.x + a.y, m0.x + m0.y, m1.x + m1.y, 0.0f);
      }
      if (kv4_any(!ok)) { ok = false; break; }
      float off = 0.0f, total = 0.0f;
#pragma unroll
      for (int k = 0; k < A::SHARE; ++k) {
        const float4 e = ex[k * PAIRS];
        total += e.x;
        off += share * G / A::SHARE ? e.z : e.y;
      }
      const float unit = big / KV4_WEIGHT;
      kv4_soft_sync();  // the exchange is free
      if (live) {
        T* out = static_cast<T*>(p.out) + ((size_t)(r.x.q.r0 + row) * p.n_head + head) * HD + share * OWN;
        float* dst = p.part + (((size_t)blockIdx.x * 2 + r.begins) * PAIRS + pair) * A::PART;
        const bool whole = r.begins && r.ends;
        if (!whole && share == 0) *reinterpret_cast<float2*>(dst) = make_float2(mx, total);
#pragma unroll
        for (int i = 0; i < OWN; i += 4) {
          const float4 v = make_float4(fmaf(o[i], unit, off), fmaf(o[i + 1], unit, off), fmaf(o[i + 2], unit, off),
                                       fmaf(o[i + 3], unit, off));
          if (whole) kv4_store4(out + i, kv4_quotient(v, total));
          else *reinterpret_cast<float4*>(dst + 4 + share * OWN + i) = v;
        }
      }
      u = r.next;
    }
    if (!ok && tid == 0 && p.c.err) atomicExch(p.c.err, KERR_WAIT);
  } else if (warp < MMA_WARP) {
    // ---- the codes and the parameters
    const int side = warp >= A::V_WARP;
    uint64_t* freed = side ? bars.pv_done : bars.s_full;  // the products that used the buffers last
    uint64_t* full = side ? bars.v_full : bars.k_full;
    const int t0 = tid - (side ? A::V_WARP : A::K_WARP) * 32;
    int j = 0;
    bool ok = true;
    for (int u = a0; u < a1 && ok;) {
      const Part r = part_at(u);
      for (int page = r.first; page < r.last; ++page, ++j) {
        const int b = j & 1, left = r.lim_max - page * KV_PAGE;  // positions 0 .. left of the page are seen
        const uint8_t* raw = smem + A::RAW_AT + (j % 3) * A::PAGE_BYTES + side * A::BB;
        const int at = __ldg(p.c.table + (size_t)r.x.seq * p.c.table_stride + page);
        const bool absent = (unsigned)at >= (unsigned)p.c.n_pages;
        ok = kv4_warp_wait(bars, &bars.raw_full[j % 3], (j / 3) & 1) &&
             (j < 2 || kv4_warp_wait(bars, &freed[b], ((j - 2) >> 1) & 1));
        if (!ok) break;
        float* par = reinterpret_cast<float*>(smem + A::PAR_AT + (j & 3) * A::PAR_BYTES) + side * 2 * G * KV_PAGE;
        auto param = [&](int i) {  // position i % 64, group i / 64: its d
          const int pos = i % KV_PAGE, g = i / KV_PAGE;
          const float2 dm = __half22float2(reinterpret_cast<const __half2*>(raw + kv4_codes_bytes(HD))[pos * G + g]);
          const bool seen = !absent && pos <= left;  // else whatever the memory held
          par[2 * g * KV_PAGE + pos] = seen ? 0.5f * dm.x : 0.0f;
          par[(2 * g + 1) * KV_PAGE + pos] = seen ? fmaf(7.5f, dm.x, dm.y) : 0.0f;
          return seen ? dm.x : 0.0f;
        };
        if (!side) {
          uint8_t* k = smem + A::K_AT + b * G * A::TILE;
#pragma unroll
          for (int n = 0; n < 2; ++n) {  // position i / 4, 16 dimensions of every group
            const int i = t0 + n * 128, pos = i >> 2, t = i & 3;
            uint32_t w[2 * G];
            if constexpr (G == 2) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(raw + i * 16);
            else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(raw + i * 8);
#pragma unroll
            for (int x = 0; x < 2 * G; ++x) {
              uint32_t h[4];
              kv4_centred(w[x], h);
              *reinterpret_cast<uint4*>(k + x / 2 * A::TILE + pos / 8 * A::SBO + (2 * t + x % 2) * A::LBO + pos % 8 * 16) =
                  make_uint4(h[0], h[1], h[2], h[3]);
            }
          }
          if (t0 < KV_PAGE * G) param(t0);
        } else if (warp < A::V_PAR_WARP) {
          uint8_t* v = smem + A::V_AT + b * G * A::TILE;
          const int chunk = t0 >> 3, g = t0 & 7;  // 8 positions, 4 dimensions of every block of 32
          uint32_t w[4][2 * G];                   // [pair of positions][block]
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint8_t* from = raw + ((chunk * 4 + t) * 8 + g) * (8 * G);
            if constexpr (G == 2) *reinterpret_cast<uint4*>(w[t]) = *reinterpret_cast<const uint4*>(from);
            else *reinterpret_cast<uint2*>(w[t]) = *reinterpret_cast<const uint2*>(from);
          }
#pragma unroll
          for (int blk = 0; blk < 2 * G; ++blk) {
            uint32_t h[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) kv4_centred(w[t][blk], h[t]);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int d = blk % 2 * 32 + 4 * g + n;
              *reinterpret_cast<uint4*>(v + blk / 2 * A::TILE + d / 8 * A::SBO + chunk * A::LBO + d % 8 * 16) =
                  make_uint4(h[0][n], h[1][n], h[2][n], h[3][n]);
            }
          }
        } else {
          float dmax = 0.0f;
#pragma unroll
          for (int i = 0; i < KV_PAGE * G / 32; ++i) dmax = fmaxf(dmax, param(lane + 32 * i));
          dmax = warp_max(dmax);
          if (lane == 0) {
            bars.vmax[j & 3] = dmax;
            bars.absent[j & 3] = absent;
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[b]);
      }
      u = r.next;
    }
  } else {
    // ---- the loads and the products. The whole warp walks (its values stay in
    // uniform registers, which the instructions want them in), one lane issues.
    const bool leader = kv4_elect();
    constexpr uint32_t IDESC = (1u << 4) | ((64u >> 3) << 17) | ((uint32_t)(PAIRS >> 4) << 24);  // fp32 sums of fp16, both K-major
    int pages = 0;  // of the whole stretch
    for (int u = a0; u < a1;) {
      const Part r = part_at(u);
      pages += r.last - r.first;
      u = r.next;
    }
    // the load cursor runs ahead of the products
    int lu = a0, lp = 0, loaded = 0;
    Part lr;
    if (a0 < a1) { lr = part_at(a0); lp = lr.first; }
    auto load = [&]() {
      while (lp >= lr.last) {
        lu = lr.next;
        lr = part_at(lu);
        lp = lr.first;
      }
      const int page = kv4_page(p.c, lr.x.seq, lp * KV_PAGE);
      uint64_t* bar = &bars.raw_full[loaded % 3];
      // an absent page is not read: its positions count for nothing
      if (leader) mbar_arrive_expect_tx(bar, page >= 0 ? A::PAGE_BYTES : 0);
      if (leader && page >= 0)
        bulk_g2s(smem + A::RAW_AT + (loaded % 3) * A::PAGE_BYTES, kv4_block(p.c, page, lr.x.kv, 0, A::BB), A::PAGE_BYTES, bar);
      ++lp;
      ++loaded;
    };
    while (loaded < min(pages, 3)) load();
    const uint32_t q0 = smem_u32(smem + A::Q_AT), k0 = smem_u32(smem + A::K_AT), v0 = smem_u32(smem + A::V_AT);
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
        const uint64_t v = umma_desc(v0 + b * G * A::TILE, A::LBO, A::SBO);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int s = 0; s < 8; ++s)  // hi, then lo; 16 positions each
            mma_f16_ts(tmem + A::O_COL + g * 64, tmem + b * A::S_COLS + g * 64 + s * 8,
                       v + ((g * A::TILE + (s & 3) * 2 * A::LBO) >> 4), IDESC, s ? 1u : add);
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
        ok = ok && kv4_warp_wait(bars, &bars.k_full[b], (j >> 1) & 1) && (j < 2 || kv4_warp_wait(bars, &bars.pv_done[b], ((j - 2) >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint64_t q = umma_desc(q0, A::QLBO, A::QSBO), k = umma_desc(k0 + b * G * A::TILE, A::LBO, A::SBO);
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int s = 0; s < 8; ++s)  // hi, then lo; 16 dimensions each
              mma_f16(tmem + b * A::S_COLS + g * 64, q + ((((s >> 2) * G + g) * A::QTILE + (s & 3) * 2 * A::QLBO) >> 4),
                      k + ((g * A::TILE + (s & 3) * 2 * A::LBO) >> 4), IDESC, s ? 1u : 0u);
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
      for (int i = 0; i < min(loaded, 3); ++i) mbar_wait(&bars.raw_full[(loaded - 1 - i) % 3], ((loaded - 1 - i) / 3) & 1);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, A::TMEM);
}

}  // namespace fox
