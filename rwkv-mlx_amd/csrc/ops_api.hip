// C ABI of the routing from logits (route.hip) and of the 8-bit products
// (fp8.hip, fp8_gemm.hip): argument checks, workspaces and launch sequences.
// Every argument error is detected here, on the host, before any HIP call.
#include <stdint.h>

#include <algorithm>

#include "../../include/rwkvmoe.h"
#include "fp8.h"
#include "route.h"

using namespace rwkvmoe;

namespace {

bool aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }
size_t elem_size(int dtype) { return dtype == RWKVMOE_F32 ? 4 : 2; }

#define TRY(expr)                       \
  do {                                  \
    const int _st = (expr);             \
    if (_st != RWKVMOE_OK) return _st;  \
  } while (0)

#define HIPTRY(expr)                          \
  do {                                        \
    const hipError_t _e = (expr);             \
    if (_e != hipSuccess) return (int)_e;     \
  } while (0)

// A required pointer of the given alignment.
int need(const void* p, size_t a) {
  return !p ? RWKVMOE_ERR_NULL_PTR : aligned(p, a) ? RWKVMOE_OK : RWKVMOE_ERR_ALIGN;
}
int maybe(const void* p, size_t a) { return !p || aligned(p, a) ? RWKVMOE_OK : RWKVMOE_ERR_ALIGN; }
int check_dtype(int dt) { return dt >= RWKVMOE_F32 && dt <= RWKVMOE_BF16 ? RWKVMOE_OK : RWKVMOE_ERR_DTYPE; }

// A launch has fewer than 2^32 threads, of 256 a workgroup (of 512, where
// fewer workgroups are launched).
constexpr long long kMaxBlocks = (1ll << 24) - 1;

// ---- routing ----

constexpr int kMaxRouteRows = (1 << 26) - 64;  // (up to 64 threads a row)

int check_route(const rwkvmoe_route_desc* d, Route* r) {
  if (!d) return RWKVMOE_ERR_NULL_DESC;
  TRY(check_dtype(d->dtype));
  if (d->rows < 0 || d->rows > kMaxRouteRows || d->n_experts < 1 || d->n_experts > kRouteMaxE)
    return RWKVMOE_ERR_SHAPE;
  if (d->n_groups < 1 || d->n_groups > kRouteMaxGroups || d->n_experts % d->n_groups || d->top_groups < 1 ||
      d->top_groups > d->n_groups || d->logits_stride < d->n_experts)
    return RWKVMOE_ERR_SHAPE;
  if (d->top_k < 1 || d->top_k > kRouteMaxK || d->top_k > d->top_groups * (d->n_experts / d->n_groups))
    return RWKVMOE_ERR_TOPK;
  if (d->score < 0 || d->score > RWKVMOE_SCORE_SIGMOID || d->group_score < 0 || d->group_score > RWKVMOE_GROUP_TOP2)
    return RWKVMOE_ERR_MODE;
  if (d->flags & ~RWKVMOE_ROUTE_RENORM) return RWKVMOE_ERR_FLAGS;
  *r = Route{};
  r->rows = d->rows;
  r->E = d->n_experts;
  r->k = d->top_k;
  r->groups = d->n_groups;
  r->top_groups = d->top_groups;
  r->dtype = d->dtype;
  r->sigmoid = d->score == RWKVMOE_SCORE_SIGMOID;
  r->top2 = d->group_score == RWKVMOE_GROUP_TOP2;
  r->renorm = d->flags & RWKVMOE_ROUTE_RENORM;
  r->scale = d->scale;
  r->stride = d->logits_stride;
  return RWKVMOE_OK;
}

// ---- 8-bit products ----

constexpr int kMaxRows = 65535 * kFp8Block, kMaxK = 1 << 23, kMaxGroups = 1024;
constexpr int kMaxN = 1 << 22;  // (a tile's rows of out lie within 4 GB)

int check_fp8(const rwkvmoe_fp8_desc* d, bool product) {
  if (!d) return RWKVMOE_ERR_NULL_DESC;
  TRY(check_dtype(d->dtype));
  if (d->block != RWKVMOE_FP8_ROWS && d->block != RWKVMOE_FP8_TILES) return RWKVMOE_ERR_MODE;
  if (d->rows < 0 || d->rows > kMaxRows || d->k < 1 || d->k > kMaxK || d->groups < 0 || d->groups > kMaxGroups)
    return RWKVMOE_ERR_SHAPE;
  // (the workgroups of a launch: 16 rows of one slice of k)
  if ((d->rows / 16 + 1ll) * fp8_blocks(d->k) > kMaxBlocks) return RWKVMOE_ERR_SHAPE;
  if (product) {
    if (d->n < 1 || d->n > kMaxN) return RWKVMOE_ERR_SHAPE;
    // (the tiles of a launch)
    if ((long long)(fp8_blocks(d->rows) + d->groups) * fp8_blocks(d->n) >= 0x7fffffffll) return RWKVMOE_ERR_SHAPE;
    if (d->groups && d->block != RWKVMOE_FP8_TILES) return RWKVMOE_ERR_MODE;
  }
  return RWKVMOE_OK;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t q_bytes(size_t rows, int k) { return rows * fp8_pad(k); }
size_t s_bytes(size_t rows, int k) { return rows * fp8_blocks(k) * sizeof(float); }

Fp8Gemm gemm_of(const rwkvmoe_fp8_desc* d, const void* a, const float* sa, const void* b, const float* sb,
                const int32_t* off, void* out) {
  Fp8Gemm g{};
  g.a = (const unsigned char*)a;
  g.sa = sa;
  g.b = (const unsigned char*)b;
  g.sb = sb;
  g.off = d->groups ? off : nullptr;
  g.groups = d->groups;
  g.m = d->rows;
  g.n = d->n;
  g.k = d->k;
  g.b_kind = d->block == RWKVMOE_FP8_TILES ? FP8_TILES : FP8_ROWS;
  g.out_kind = d->dtype == RWKVMOE_F32 ? FP8_OUT_F32 : d->dtype == RWKVMOE_F16 ? FP8_OUT_F16 : FP8_OUT_BF16;
  g.exact = d->dtype == RWKVMOE_F32;
  g.out = out;
  return g;
}

struct ExpertsLayout {
  size_t dcounts, perm, inv, offsets, xq, xs, hq, hs, rows, total;
};

int check_experts(const rwkvmoe_desc* d, ExpertsLayout* L) {
  if (!d) return RWKVMOE_ERR_NULL_DESC;
  TRY(check_dtype(d->dtype));
  if (d->batch < 0 || d->seq_len < 0 || d->d_model < 4 || d->d_model % 4 || d->d_model > kMaxN || d->d_ffn < 1 ||
      d->d_ffn > kMaxN || d->n_experts < 1 || d->n_experts > 64)
    return RWKVMOE_ERR_SHAPE;
  if (d->top_k < 1 || d->top_k > std::min(d->n_experts, 8)) return RWKVMOE_ERR_TOPK;
  if (d->flags & ~(RWKVMOE_HAS_PREV | RWKVMOE_ADD_RESIDUAL)) return RWKVMOE_ERR_FLAGS;
  const long long N = (long long)d->batch * d->seq_len, nk = N * d->top_k;
  if (nk > kMaxRows || (nk / 16 + 1) * fp8_blocks(d->d_model) > kMaxBlocks ||
      N * (d->d_model / 4) > kMaxBlocks * 256 ||
      (nk / kFp8Block + 1 + d->n_experts) * fp8_blocks(std::max(d->d_ffn, d->d_model)) >= 0x7fffffffll)
    return RWKVMOE_ERR_SHAPE;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += up256(bytes);
    return at;
  };
  L->dcounts = take((size_t)dispatch_blocks((int)nk) * d->n_experts * sizeof(int));
  L->perm = take((size_t)nk * sizeof(int));
  L->inv = take((size_t)nk * sizeof(int));
  L->offsets = take((d->n_experts + 1) * sizeof(int));
  L->xq = take(q_bytes(nk, d->d_model));
  L->xs = take(s_bytes(nk, d->d_model));
  L->hq = take(q_bytes(nk, d->d_ffn));
  L->hs = take(s_bytes(nk, d->d_ffn));
  L->rows = take((size_t)nk * d->d_model * sizeof(float));
  L->total = off;
  return RWKVMOE_OK;
}

}  // namespace

extern "C" {

int rwkvmoe_route(const rwkvmoe_route_desc* desc, const void* logits, const float* bias, int32_t* inds, float* gates,
                  void* stream) {
  Route r;
  TRY(check_route(desc, &r));
  if (r.rows == 0) return RWKVMOE_OK;
  TRY(need(logits, elem_size(r.dtype))); TRY(maybe(bias, 4)); TRY(need(inds, 4)); TRY(need(gates, 4));
  r.logits = logits;
  r.bias = bias;
  r.inds = inds;
  r.gates = gates;
  HIPTRY(launch_route(r, (hipStream_t)stream));
  return RWKVMOE_OK;
}

int rwkvmoe_route_backward(const rwkvmoe_route_desc* desc, const void* logits, const int32_t* inds, const float* gates,
                           const float* d_gates, void* d_logits, void* stream) {
  Route r;
  TRY(check_route(desc, &r));
  if (r.rows == 0) return RWKVMOE_OK;
  TRY(need(logits, elem_size(r.dtype))); TRY(need(inds, 4)); TRY(need(gates, 4)); TRY(need(d_gates, 4));
  TRY(need(d_logits, 16));
  r.logits = logits;
  r.inds_in = inds;
  r.gates_in = gates;
  r.d_gates = d_gates;
  r.d_logits = d_logits;
  HIPTRY(launch_route_backward(r, (hipStream_t)stream));
  return RWKVMOE_OK;
}

int rwkvmoe_fp8_quantize(const rwkvmoe_fp8_desc* desc, const void* x, void* q, float* scales, void* q_t,
                         float* scales_t, void* stream) {
  TRY(check_fp8(desc, false));
  if (desc->stride < desc->k || (desc->groups && desc->block == RWKVMOE_FP8_ROWS)) return RWKVMOE_ERR_SHAPE;
  if (!q && !q_t) return RWKVMOE_ERR_NULL_PTR;
  if (desc->rows == 0) return RWKVMOE_OK;
  TRY(need(x, elem_size(desc->dtype))); TRY(maybe(q, 16)); TRY(maybe(q_t, 16));
  if (q) TRY(need(scales, 4));
  if (q_t) TRY(need(scales_t, 4));
  const Fp8Quant p{x, desc->dtype, std::max(desc->groups, 1), desc->rows, desc->k, desc->stride,
                   (unsigned char*)q, scales, (unsigned char*)q_t, scales_t};
  HIPTRY(desc->block == RWKVMOE_FP8_TILES ? launch_fp8_quant_tiles(p, (hipStream_t)stream)
                                          : launch_fp8_quant_rows(p, (hipStream_t)stream));
  return RWKVMOE_OK;
}

int rwkvmoe_fp8_layout(const rwkvmoe_fp8_desc* desc, const void* src, const float* src_scales, void* q, float* scales,
                       void* q_t, float* scales_t, void* stream) {
  TRY(check_fp8(desc, true));
  if (desc->block != RWKVMOE_FP8_TILES) return RWKVMOE_ERR_MODE;
  TRY(need(src, 1)); TRY(need(src_scales, 4)); TRY(need(q, 16)); TRY(need(scales, 4)); TRY(maybe(q_t, 16));
  if (q_t) TRY(need(scales_t, 4));
  if (fp8_blocks(desc->n) > 65535) return RWKVMOE_ERR_SHAPE;
  const Fp8Quant p{nullptr, desc->dtype, std::max(desc->groups, 1), desc->n, desc->k, desc->k,
                   (unsigned char*)q, scales, (unsigned char*)q_t, scales_t};
  HIPTRY(launch_fp8_layout((const unsigned char*)src, src_scales, p, (hipStream_t)stream));
  return RWKVMOE_OK;
}

int rwkvmoe_fp8_matmul(const rwkvmoe_fp8_desc* desc, const void* a, const float* a_scales, const void* b,
                       const float* b_scales, const int32_t* offsets, void* out, void* stream) {
  TRY(check_fp8(desc, true));
  if (desc->rows == 0) return RWKVMOE_OK;
  TRY(need(a, 16)); TRY(need(a_scales, 4)); TRY(need(b, 16)); TRY(need(b_scales, 4)); TRY(need(out, 16));
  if (desc->groups) TRY(need(offsets, 4));
  HIPTRY(launch_fp8_gemm(gemm_of(desc, a, a_scales, b, b_scales, offsets, out), (hipStream_t)stream));
  return RWKVMOE_OK;
}

int rwkvmoe_fp8_linear_workspace_bytes(const rwkvmoe_fp8_desc* desc, size_t* bytes) {
  TRY(check_fp8(desc, true));
  if (!bytes) return RWKVMOE_ERR_NULL_PTR;
  *bytes = fp8_few(desc->rows) ? 0 : up256(q_bytes(desc->rows, desc->k)) + up256(s_bytes(desc->rows, desc->k));
  return RWKVMOE_OK;
}

int rwkvmoe_fp8_linear(const rwkvmoe_fp8_desc* desc, const void* x, const void* b, const float* b_scales,
                       const int32_t* offsets, void* out, void* ws, size_t ws_bytes, void* stream) {
  TRY(check_fp8(desc, true));
  if (desc->block != RWKVMOE_FP8_TILES) return RWKVMOE_ERR_MODE;
  if (desc->stride < desc->k) return RWKVMOE_ERR_SHAPE;
  if (desc->rows == 0) return RWKVMOE_OK;
  TRY(need(x, elem_size(desc->dtype))); TRY(need(b, 16)); TRY(need(b_scales, 4)); TRY(need(out, 16));
  if (desc->groups) TRY(need(offsets, 4));
  if (fp8_few(desc->rows)) {  // rounded in the product's launch
    Fp8Gemm g = gemm_of(desc, nullptr, nullptr, b, b_scales, offsets, out);
    g.x = x;
    g.ldx = desc->stride;
    HIPTRY(launch_fp8_gemm(g, (hipStream_t)stream));
    return RWKVMOE_OK;
  }
  const size_t qb = up256(q_bytes(desc->rows, desc->k)), sb = up256(s_bytes(desc->rows, desc->k));
  if (!ws || ws_bytes < qb + sb || !aligned(ws, 256)) return RWKVMOE_ERR_WORKSPACE;
  unsigned char* q = (unsigned char*)ws;
  float* s = (float*)(q + qb);
  const Fp8Quant p{x, desc->dtype, 1, desc->rows, desc->k, desc->stride, q, s, nullptr, nullptr};
  HIPTRY(launch_fp8_quant_rows(p, (hipStream_t)stream));
  HIPTRY(launch_fp8_gemm(gemm_of(desc, q, s, b, b_scales, offsets, out), (hipStream_t)stream));
  return RWKVMOE_OK;
}

int rwkvmoe_fp8_experts_workspace_bytes(const rwkvmoe_desc* desc, size_t* bytes) {
  ExpertsLayout L;
  TRY(check_experts(desc, &L));
  if (!bytes) return RWKVMOE_ERR_NULL_PTR;
  *bytes = L.total;
  return RWKVMOE_OK;
}

int rwkvmoe_fp8_experts_forward(const rwkvmoe_desc* desc, const rwkvmoe_fp8_experts* t, void* ws, size_t ws_bytes,
                                void* stream) {
  ExpertsLayout L;
  TRY(check_experts(desc, &L));
  if (!t) return RWKVMOE_ERR_NULL_DESC;
  if (t->struct_size != sizeof(rwkvmoe_fp8_experts)) return RWKVMOE_ERR_VERSION;
  const int N = desc->batch * desc->seq_len, C = desc->d_model, F = desc->d_ffn, E = desc->n_experts, k = desc->top_k;
  if (N == 0) return RWKVMOE_OK;
  const bool prev = desc->flags & RWKVMOE_HAS_PREV, resid = desc->flags & RWKVMOE_ADD_RESIDUAL;
  if ((prev && !t->x_prev) || (resid && !t->residual)) return RWKVMOE_ERR_FLAGS;
  const size_t es = elem_size(desc->dtype);
  TRY(need(t->x, es)); TRY(need(t->x_k, es)); TRY(need(t->key_q, 16)); TRY(need(t->key_scales, 4));
  TRY(need(t->value_q, 16)); TRY(need(t->value_scales, 4)); TRY(need(t->inds, 4)); TRY(need(t->gates, 4));
  TRY(need(t->out, es)); TRY(maybe(t->x_prev, es)); TRY(maybe(t->residual, es));
  if (!ws || ws_bytes < L.total || !aligned(ws, 256)) return RWKVMOE_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  unsigned char* w = (unsigned char*)ws;
  const int nk = N * k;
  int *perm = (int*)(w + L.perm), *inv = (int*)(w + L.inv), *off = (int*)(w + L.offsets);
  HIPTRY(launch_dispatch(t->inds, nk, E, (int*)(w + L.dcounts), perm, inv, off, s, nullptr, 0, k));
  HIPTRY(launch_fp8_mix(desc->dtype, t->x, prev ? t->x_prev : nullptr, t->x_k, perm, t->inds, off, N, desc->seq_len, C,
                        E, k, w + L.xq, (float*)(w + L.xs), s));
  Fp8Gemm g{};
  g.a = w + L.xq;
  g.sa = (const float*)(w + L.xs);
  g.b = (const unsigned char*)t->key_q;
  g.sb = t->key_scales;
  g.off = off;
  g.groups = E;
  g.m = nk;
  g.n = F;
  g.k = C;
  g.b_kind = FP8_TILES;
  g.out_kind = FP8_OUT_RELU2Q;
  // a hidden value that lies on a border of e4m3 moves by a whole step: with
  // fp16 or fp32 results the sums before it are fp32's
  g.exact = desc->dtype != RWKVMOE_BF16;
  g.out = w + L.hq;
  g.out_s = (float*)(w + L.hs);
  HIPTRY(launch_fp8_gemm(g, s));
  g.a = w + L.hq;
  g.sa = (const float*)(w + L.hs);
  g.b = (const unsigned char*)t->value_q;
  g.sb = t->value_scales;
  g.n = C;
  g.k = F;
  g.out_kind = FP8_OUT_F32;
  g.exact = desc->dtype == RWKVMOE_F32;
  g.out = w + L.rows;
  g.out_s = nullptr;
  HIPTRY(launch_fp8_gemm(g, s));
  HIPTRY(launch_fp8_combine(desc->dtype, (const float*)(w + L.rows), t->gates, inv, resid ? t->residual : nullptr,
                            t->out, N, C, k, s));
  return RWKVMOE_OK;
}

}  // extern "C"
