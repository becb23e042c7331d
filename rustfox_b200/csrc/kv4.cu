// The 4-bit paged K/V cache's entry points (include/foxcuda.h): argument
// checks and launches of kv4.cuh and kv4_attn.cuh.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "../../include/foxcuda.h"
#include "common.cuh"
#include "host.cuh"
#include "kv4.cuh"
#include "kv4_attn.cuh"
#include "kv4_wide.cuh"

using namespace fox;

// Attention takes the 5th-generation tensor cores' tiles from this many (row,
// head) pairs a sequence and KV head on: their time hardly depends on the rows.
// 4 sequences of 16384 positions, 8 KV heads of 128: 32 pairs 120 us either way,
// 48 pairs 170 us narrow and 121 wide, 128 pairs 423 and 130; of 64: 32 pairs 77
// and 83, 48 pairs 110 and 84. The rule sees what the host knows, a call's average
// with its padding rows, so a call of unlike sequences can be better as two: 64
// rows beside 15 single tokens, 16384 positions each, take 268 us in one call and
// 85 + 67 in two; 16 tokens of 4096 positions take 33 us, in 1024 row places 137.
// Heads of 256 dimensions stay with the narrow tiles (64 rows of 16 heads over 4
// behind 8192 positions: 134 us): S of two pages, O with the offsets and both
// halves of q would take 664 of tensor memory's 512 columns.
constexpr int KV4_WIDE_FROM = 48;
// Where no run is split, a tile has one SM for its pages, so there must also be
// this many pairs an SM: one sequence of 1000 positions, 128 pairs for each of 8
// KV heads, 18 us narrow and 42 wide; 16 of 512, 48 pairs, 41 and 27. (A longer
// table may hold short sequences all the same: 128 pairs behind 1000 positions
// under one of 512 pages take 47 us.)
constexpr int KV4_WIDE_FILL = 32;

static_assert(FOXCUDA_KV_PAGE == KV_PAGE, "the header's page size is the kernels'");

static bool kv4_hd_ok(uint32_t hd) { return hd == 64 || hd == 128 || hd == 256; }
static bool kv4_type_ok(int t) { return t == T_F32 || t == T_F16; }
static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
static bool aligned4(const void* p) { return (uintptr_t)p % 4 == 0; }
// The arrays that every call on a cache reads, and the cache.
static Rows cache_of(const foxcuda_kv4* c) {
  return {c->cache, (size_t)c->n_pages * c->n_head_kv * 2 * kv4_block_bytes((int)c->head_dim)};
}
static Rows table_of(const foxcuda_kv4* c) { return {c->table, (size_t)c->n_seq * c->table_stride * 4}; }
static Rows starts_of(const foxcuda_kv4* c) { return {c->row_start, ((size_t)c->n_seq + 1) * 4}; }
static Rows lens_of(const foxcuda_kv4* c) { return {c->kv_len, (size_t)c->n_seq * 4}; }
static bool stride_ok(size_t stride, size_t row, int type) {
  return stride >= row && stride * (type == T_F32 ? 4 : 2) % 16 == 0 && stride <= ((size_t)1 << 32);
}

extern "C" size_t foxcuda_kv4_block_bytes(uint32_t head_dim) {
  return kv4_hd_ok(head_dim) ? (size_t)kv4_block_bytes((int)head_dim) : 0;
}

// The checks every call on a cache makes; *none is set when there is no row.
static foxcuda_status check_kv4(const foxcuda_kv4* c, int type, const char* what, Kv4Rows* r, bool* none) {
  if (!c) return fail(FOXCUDA_ERR_ARG, "%s: null cache", what);
  if (!kv4_type_ok(type)) return fail(FOXCUDA_ERR_UNSUPPORTED, "%s: rows of ggml type %d are not covered", what, type);
  if (!kv4_hd_ok(c->head_dim))
    return fail(FOXCUDA_ERR_UNSUPPORTED, "%s: head_dim %u is not 64, 128 or 256", what, c->head_dim);
  if (!c->n_head_kv || c->n_head_kv > 1024) return fail(FOXCUDA_ERR_ARG, "%s: %u KV heads", what, c->n_head_kv);
  if (c->n_seq > (uint32_t)KV4_MAX_SEQ || c->n_rows > (1u << 20))
    return fail(FOXCUDA_ERR_ARG, "%s: %u sequences / %u rows are beyond %d and 2^20", what, c->n_seq, c->n_rows,
                KV4_MAX_SEQ);
  if (c->table_stride > (1u << 24) || c->n_pages > (uint32_t)INT_MAX)
    return fail(FOXCUDA_ERR_ARG, "%s: %u pages a sequence / %u pages", what, c->table_stride, c->n_pages);
  *none = c->n_rows == 0 || c->n_seq == 0;
  if (*none) return FOXCUDA_OK;
  if (!c->cache || !c->table || !c->row_start || !c->kv_len) return fail(FOXCUDA_ERR_ARG, "%s: null pointer", what);
  if (!aligned16(c->cache)) return fail(FOXCUDA_ERR_ARG, "%s: the cache must be 16-byte aligned", what);
  if (!aligned4(c->table) || !aligned4(c->row_start) || !aligned4(c->kv_len))
    return fail(FOXCUDA_ERR_ARG, "%s: table, row_start and kv_len must be 4-byte aligned", what);
  r->cache = static_cast<uint8_t*>(c->cache);
  r->table = c->table; r->row_start = c->row_start; r->kv_len = c->kv_len;
  r->n_pages = (int)c->n_pages; r->n_kv = (int)c->n_head_kv; r->n_seq = (int)c->n_seq;
  r->table_stride = (int)c->table_stride; r->n_rows = (int)c->n_rows;
  r->err = kernel_err_ptr();
  return FOXCUDA_OK;
}

// f(type tag, head dimension) for the combination asked for.
template <typename F>
static cudaError_t by_type_hd(int type, uint32_t hd, F f) {
  auto with = [&](auto tag) {
    switch (hd) {
      case 64: return f(tag, std::integral_constant<int, 64>());
      case 128: return f(tag, std::integral_constant<int, 128>());
      default: return f(tag, std::integral_constant<int, 256>());
    }
  };
  return type == T_F32 ? with(float()) : with(__half());
}

// One row a warp where the rows are few, so that they spread over the device (16
// fp32 rows written: 2.7 us, 4.1 with four rows a warp; read 2.9 and 4.3); four,
// for one search for their places and more loads in flight, where they fill it
// anyway (32768 read to fp16: 39 us, 71 with one; 4616 written: 13.7 and 15.0).
template <int HD, typename F>
static cudaError_t by_rows(const Kv4Rows& c, F f) {
  const int passes = Kv4Pass<HD>::passes(c.n_kv);
  const auto grid = [&](int rows) { return (unsigned)(((size_t)((c.n_rows + rows - 1) / rows) * passes + 7) / 8); };
  if ((long long)c.n_rows * passes > 32LL * current_sms()) f(std::integral_constant<int, 4>(), grid(4));
  else f(std::integral_constant<int, 1>(), grid(1));
  return cudaGetLastError();
}

extern "C" foxcuda_status foxcuda_kv4_write(const foxcuda_kv4* c, int type, const void* k, size_t k_stride,
                                            const void* v, size_t v_stride, void* stream) {
  Kv4MoveParams p{};
  bool none = false;
  foxcuda_status st = check_kv4(c, type, "kv4_write", &p.c, &none);
  if (st || none) return st;
  const size_t row = (size_t)c->n_head_kv * c->head_dim;
  if (!k || !v) return fail(FOXCUDA_ERR_ARG, "kv4_write: null pointer");
  if (!aligned16(k) || !aligned16(v) || !stride_ok(k_stride, row, type) || !stride_ok(v_stride, row, type))
    return fail(FOXCUDA_ERR_ARG, "kv4_write: rows must be 16-byte aligned and at least a row apart");
  const size_t size = type == T_F32 ? 4 : 2;
  if (overlap(cache_of(c), {{k, row * size, c->n_rows, k_stride * size}, {v, row * size, c->n_rows, v_stride * size},
                            table_of(c), starts_of(c), lens_of(c)}))
    return fail(FOXCUDA_ERR_ARG, "kv4_write: the cache overlaps what is read");
  p.k = const_cast<void*>(k); p.v = const_cast<void*>(v); p.k_stride = k_stride; p.v_stride = v_stride;
  CK(by_type_hd(type, c->head_dim, [&](auto tag, auto hd) {
       return by_rows<hd.value>(p.c, [&](auto rows, unsigned grid) {
         kv4_write_kernel<decltype(tag), hd.value, rows.value><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
       });
     }), "kv4_write launch");
  return FOXCUDA_OK;
}

extern "C" foxcuda_status foxcuda_kv4_read(const foxcuda_kv4* c, int type, void* k, void* v, void* stream) {
  Kv4MoveParams p{};
  bool none = false;
  foxcuda_status st = check_kv4(c, type, "kv4_read", &p.c, &none);
  if (st || none) return st;
  if (!k || !v) return fail(FOXCUDA_ERR_ARG, "kv4_read: null pointer");
  if (!aligned16(k) || !aligned16(v)) return fail(FOXCUDA_ERR_ARG, "kv4_read: rows must be 16-byte aligned");
  const size_t bytes = (size_t)c->n_rows * c->n_head_kv * c->head_dim * (type == T_F32 ? 4 : 2);
  if (overlap(Rows{k, bytes}, {{v, bytes}, cache_of(c), table_of(c), starts_of(c), lens_of(c)}) ||
      overlap(Rows{v, bytes}, {cache_of(c), table_of(c), starts_of(c), lens_of(c)}))
    return fail(FOXCUDA_ERR_ARG, "kv4_read: the outputs overlap one another or what is read");
  p.k = k; p.v = v;
  CK(by_type_hd(type, c->head_dim, [&](auto tag, auto hd) {
       return by_rows<hd.value>(p.c, [&](auto rows, unsigned grid) {
         kv4_read_kernel<decltype(tag), hd.value, rows.value><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
       });
     }), "kv4_read launch");
  return FOXCUDA_OK;
}

template <typename T, int HD, bool HALVES, int BATCH>
static cudaError_t launch_rope_b(const RopeParams& p, cudaStream_t s) {
  using Y = RopeLay<T, HD>;
  const size_t warps = (size_t)p.n_rows * (Y::chunks(p.n_head, BATCH) + Y::chunks(p.n_kv, BATCH));
  qk_norm_rope_kernel<T, HD, HALVES, BATCH><<<(unsigned)((warps + 7) / 8), 256, 0, s>>>(p);
  return cudaGetLastError();
}
// One load a warp where the rows are few, so that they spread over the device (1
// row of 40 heads: 1.6 us, 2.2 with four); four, each row's tables loaded once
// for them, where they fill it anyway (4096 fp16 rows of 48 heads: 23 us, 38 with
// one).
template <typename T, int HD, bool HALVES>
static cudaError_t launch_rope(const RopeParams& p, cudaStream_t s) {
  const long long bytes = (long long)p.n_rows * (p.n_head + p.n_kv) * HD * sizeof(T);
  return bytes > 512LL * 16 * current_sms() ? launch_rope_b<T, HD, HALVES, 4>(p, s) : launch_rope_b<T, HD, HALVES, 1>(p, s);
}

extern "C" foxcuda_status foxcuda_qk_norm_rope(int type, const void* x, size_t x_stride, uint32_t n_rows,
                                               uint32_t n_head, uint32_t n_head_kv, uint32_t head_dim,
                                               const float* q_norm, const float* k_norm, float eps,
                                               const float* cos, const float* sin, uint32_t n_pos, int halves,
                                               const int32_t* pos, void* q_out, size_t q_stride, void* k_out,
                                               size_t k_stride, void* stream) {
  if (!kv4_type_ok(type)) return fail(FOXCUDA_ERR_UNSUPPORTED, "qk_norm_rope: rows of ggml type %d are not covered", type);
  if (!kv4_hd_ok(head_dim)) return fail(FOXCUDA_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %u is not 64, 128 or 256", head_dim);
  if (!n_head || !n_head_kv || n_head > 1024 || n_head_kv > 1024)
    return fail(FOXCUDA_ERR_ARG, "qk_norm_rope: %u query heads / %u KV heads", n_head, n_head_kv);
  if (halves != 0 && halves != 1) return fail(FOXCUDA_ERR_ARG, "qk_norm_rope: halves %d", halves);
  if (n_rows > (1u << 20) || n_pos > (uint32_t)INT_MAX)
    return fail(FOXCUDA_ERR_ARG, "qk_norm_rope: %u rows / %u positions", n_rows, n_pos);
  if (n_rows == 0) return FOXCUDA_OK;
  if (!x || !cos || !sin || !pos || !q_out || !k_out) return fail(FOXCUDA_ERR_ARG, "qk_norm_rope: null pointer");
  if (!aligned4(pos)) return fail(FOXCUDA_ERR_ARG, "qk_norm_rope: pos must be 4-byte aligned");
  const size_t nq = (size_t)n_head * head_dim, nk = (size_t)n_head_kv * head_dim;
  if (!aligned16(x) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(cos) || !aligned16(sin) ||
      (q_norm && !aligned16(q_norm)) || (k_norm && !aligned16(k_norm)) || !stride_ok(x_stride, nq + nk, type) ||
      !stride_ok(q_stride, nq, type) || !stride_ok(k_stride, nk, type))
    return fail(FOXCUDA_ERR_ARG, "qk_norm_rope: rows and tables must be 16-byte aligned, rows at least a row apart");
  const size_t size = type == T_F32 ? 4 : 2;
  const Rows xq = {x, nq * size, n_rows, x_stride * size}, xk = {(const char*)x + nq * size, nk * size, n_rows, x_stride * size};
  const Rows qo = {q_out, nq * size, n_rows, q_stride * size}, ko = {k_out, nk * size, n_rows, k_stride * size};
  const Rows angles[3] = {{cos, (size_t)n_pos * (head_dim / 2) * 4}, {sin, (size_t)n_pos * (head_dim / 2) * 4}, {pos, (size_t)n_rows * 4}};
  const Rows norms[2] = {{q_norm, (size_t)head_dim * 4}, {k_norm, (size_t)head_dim * 4}};
  const auto in_place = [&](const Rows& out, const Rows& in) { return out.p == in.p && (out.stride == in.stride || n_rows == 1); };
  if ((!in_place(qo, xq) && overlap(qo, xq)) || (!in_place(ko, xk) && overlap(ko, xk)) ||
      overlap(qo, {ko, xk, angles[0], angles[1], angles[2], norms[0], norms[1]}) ||
      overlap(ko, {xq, angles[0], angles[1], angles[2], norms[0], norms[1]}))
    return fail(FOXCUDA_ERR_ARG, "qk_norm_rope: the outputs overlap one another or what is read (each may be its own rows of x)");
  RopeParams p{};
  p.x = x; p.pos = pos; p.q_norm = q_norm; p.k_norm = k_norm; p.cos = cos; p.sin = sin; p.q = q_out; p.k = k_out;
  p.x_stride = x_stride; p.q_stride = q_stride; p.k_stride = k_stride;
  p.n_rows = (int)n_rows; p.n_head = (int)n_head; p.n_kv = (int)n_head_kv; p.n_pos = (int)n_pos;
  p.eps = eps; p.err = kernel_err_ptr();
  CK(by_type_hd(type, head_dim, [&](auto tag, auto hd) {
       return halves ? launch_rope<decltype(tag), hd.value, true>(p, (cudaStream_t)stream)
                     : launch_rope<decltype(tag), hd.value, false>(p, (cudaStream_t)stream);
     }), "qk_norm_rope launch");
  return FOXCUDA_OK;
}

// Two pieces of a tile for every CTA.
template <int HD>
static size_t kv4_work_bytes(int ctas) {
  constexpr int wide = HD < 256 ? KV4_WIDE_PAIRS : 0;
  return (size_t)ctas * 2 * std::max(wide, Kv4Attn<HD>::PAIRS) * (HD + 4) * 4;
}

extern "C" size_t foxcuda_kv4_attention_workspace(uint32_t head_dim, uint32_t table_stride) {
  if (table_stride <= KV4_WHOLE) return 0;  // no run is split between CTAs
  const int ctas = current_sms();
  switch (head_dim) {
    case 64: return kv4_work_bytes<64>(ctas);
    case 128: return kv4_work_bytes<128>(ctas);
    case 256: return kv4_work_bytes<256>(ctas);
    default: return 0;
  }
}

// The join of split runs, its launch overlapped with the attention.
template <typename T, int HD, int PAIRS>
static cudaError_t launch_kv4_join(const Kv4AttnParams& p, cudaStream_t s) {
  static size_t marks[kMaxDevices] = {};
  const size_t most = ((size_t)p.c.n_rows * (p.n_head / p.c.n_kv) / PAIRS + p.c.n_seq) * p.c.n_kv * PAIRS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<size_t>(most, (size_t)p.ctas * 8));
  cfg.blockDim = dim3(KV4_JOIN_WARPS * 32);
  cfg.dynamicSmemBytes = kv4_join_smem<HD>(p.c.n_seq);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = opt_in_smem(kv4_join_kernel<HD, T, PAIRS>, cfg.dynamicSmemBytes, marks);
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<HD, T, PAIRS>, p);
}

template <typename T, int HD>
static cudaError_t launch_kv4_attend(const Kv4AttnParams& p, bool wide, cudaStream_t s) {
  static size_t marks[2][kMaxDevices] = {};
  const bool join = p.c.table_stride > KV4_WHOLE;  // else no run is split between CTAs
  cudaError_t e;
  if constexpr (HD < 256) {
    if (wide) {
      using A = Kv4Wide<HD>;
      const size_t smem = A::smem_bytes(p.c.n_seq);
      if ((e = opt_in_smem(kv4_wide_kernel<HD, T>, smem, marks[1])) != cudaSuccess) return e;
      kv4_wide_kernel<HD, T><<<p.ctas, A::THREADS, smem, s>>>(p);
      if ((e = cudaGetLastError()) != cudaSuccess || !join) return e;
      return launch_kv4_join<T, HD, A::PAIRS>(p, s);
    }
  }
  using A = Kv4Attn<HD>;
  const size_t smem = A::smem_bytes(p.c.n_seq);
  if ((e = opt_in_smem(kv4_attend_kernel<HD, T>, smem, marks[0])) != cudaSuccess) return e;
  kv4_attend_kernel<HD, T><<<p.ctas, A::NW * 32, smem, s>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess || !join) return e;
  return launch_kv4_join<T, HD, A::PAIRS>(p, s);
}

extern "C" foxcuda_status foxcuda_kv4_attention(const foxcuda_kv4* c, int type, const void* q, size_t q_stride,
                                                uint32_t n_head, float scale, void* workspace,
                                                size_t workspace_bytes, void* out, void* stream) {
  Kv4AttnParams p{};
  bool none = false;
  foxcuda_status st = check_kv4(c, type, "kv4_attention", &p.c, &none);
  if (st) return st;
  const uint32_t gqa = n_head / c->n_head_kv;
  if (!n_head || n_head > 1024 || n_head % c->n_head_kv || gqa > 8)
    return fail(FOXCUDA_ERR_UNSUPPORTED, "kv4_attention: %u heads over %u KV heads are not covered", n_head, c->n_head_kv);
  if (!(scale >= 0.0f) || scale > 3.0e38f) return fail(FOXCUDA_ERR_ARG, "kv4_attention: scale %g", (double)scale);
  if (none) return FOXCUDA_OK;
  const size_t need = foxcuda_kv4_attention_workspace(c->head_dim, c->table_stride);
  if (!q || !out || (need && !workspace)) return fail(FOXCUDA_ERR_ARG, "kv4_attention: null pointer");
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) ||
      !stride_ok(q_stride, (size_t)n_head * c->head_dim, type))
    return fail(FOXCUDA_ERR_ARG, "kv4_attention: rows and workspace must be 16-byte aligned, rows at least a row apart");
  const size_t size = type == T_F32 ? 4 : 2, row = (size_t)n_head * c->head_dim;
  const Rows queries = {q, row * size, c->n_rows, q_stride * size};
  if (overlap(Rows{out, c->n_rows * row * size},
              {queries, {workspace, need}, cache_of(c), table_of(c), starts_of(c), lens_of(c)}) ||
      overlap(Rows{workspace, need}, {queries, cache_of(c), table_of(c), starts_of(c), lens_of(c)}))
    return fail(FOXCUDA_ERR_ARG, "kv4_attention: out or the workspace overlap what is read, or one another");
  // tiles of at least 4 (row, head) pairs, each with every page of its sequence
  const double units = ((double)c->n_rows * gqa / 4 + c->n_seq) * c->n_head_kv * ((double)c->table_stride + KV4_HEAD);
  if (units >= 2147483648.0)
    return fail(FOXCUDA_ERR_ARG, "kv4_attention: %u rows over %u pages a sequence are too many for one call",
                c->n_rows, c->table_stride);
  if (workspace_bytes < need)
    return fail(FOXCUDA_ERR_ARG, "kv4_attention: the workspace holds %zu bytes, %zu are needed", workspace_bytes, need);
  p.q = q; p.out = out; p.part = static_cast<float*>(workspace); p.q_stride = q_stride;
  p.n_head = (int)n_head; p.ctas = current_sms();
  p.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)c->head_dim);
  // many rows a sequence: the tensor cores' 128-row tiles
  const bool wide = c->head_dim < 256 && (size_t)c->n_rows * gqa >= (size_t)KV4_WIDE_FROM * c->n_seq &&
                    (c->table_stride > KV4_WHOLE || (size_t)c->n_rows * n_head >= (size_t)KV4_WIDE_FILL * p.ctas);
  CK(by_type_hd(type, c->head_dim, [&](auto tag, auto hd) {
       return launch_kv4_attend<decltype(tag), hd.value>(p, wide, (cudaStream_t)stream);
     }), "kv4_attention launch");
  return FOXCUDA_OK;
}
