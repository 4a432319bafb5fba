// paged_prep.hip -- the per-head q/k norm, RoPE and the cache write of a ragged
// batch into pages (gfx950), and the checks every paged entry point shares.
#include "paged.h"

namespace pq {

int paged_view(const pq_paged_kv *kv, const char *who, PagedView *out) {
  PQ_REQUIRE(kv, PQ_ERR_ARG, "%s: null pointer (kv)", who);
  PQ_REQUIRE(kv->k && kv->v && kv->table && kv->kv_len, PQ_ERR_ARG, "%s: null pointer in the paged cache", who);
  PQ_REQUIRE(kv->hd == 64 || kv->hd == 128, PQ_ERR_ARG, "%s: head_dim %d (64 or 128)", who, kv->hd);
  PQ_REQUIRE(kv->dtype == PQ_DTYPE_F16 || kv->dtype == PQ_DTYPE_BF16, PQ_ERR_ARG, "%s: cache type %d (fp16 or bf16)",
             who, kv->dtype);
  PQ_REQUIRE(kv->page >= 8 && kv->page <= 65536 && (kv->page & (kv->page - 1)) == 0, PQ_ERR_ARG,
             "%s: page of %d positions (a power of two, 8 .. 65536)", who, kv->page);
  PQ_REQUIRE(kv->nkv > 0 && kv->nkv <= 1024 && kv->npages > 0 && kv->table_pages > 0 && kv->table_stride >= kv->table_pages &&
                 kv->nseq > 0 && kv->nseq <= 65535, PQ_ERR_ARG,
             "%s: nkv=%d npages=%d table %d pages of %d, nseq=%d", who, kv->nkv, kv->npages, kv->table_pages, kv->table_stride,
             kv->nseq);
  PQ_REQUIRE(kv->page_stride >= (long long)kv->page * kv->nkv * kv->hd && kv->page_stride % 8 == 0, PQ_ERR_ARG,
             "%s: page stride %lld (a multiple of 8, at least a page)", who, kv->page_stride);
  PQ_REQUIRE(aligned(kv->k, 16) && aligned(kv->v, 16), PQ_ERR_ALIGN, "%s: the pools must be 16-byte aligned", who);
  out->k = kv->k;
  out->v = kv->v;
  out->page_stride = kv->page_stride;
  out->table = kv->table;
  out->kv_len = kv->kv_len;
  out->q_start = kv->q_start;
  out->npages = kv->npages;
  out->lg_page = __builtin_ctz((unsigned)kv->page);
  out->nkv = kv->nkv;
  out->nseq = kv->nseq;
  out->table_stride = kv->table_stride;
  const long long cap = (long long)kv->table_pages * kv->page;
  out->cap = cap < 0x7fffff00LL ? (int)cap : 0x7fffff00;   // room for a tile's end in an int
  return PQ_OK;
}

int paged_attn_check(const char *who, const uint16_t *q, int q_stride, const pq_paged_kv *kv, const uint16_t *gate,
                     int gate_stride, const uint16_t *out, int out_stride, const int8_t *qx, const float *dx, int nh,
                     int win, int sinks, int max_kv, PagedView *v) {
  PQ_REQUIRE(q && (out || qx) && (!qx || dx), PQ_ERR_ARG, "%s: null pointer", who);
  const int rc = paged_view(kv, who, v);
  if (rc) return rc;
  PQ_REQUIRE((long long)v->nseq * v->nkv <= 1 << 23, PQ_ERR_ARG, "%s: nseq=%d x nkv=%d (at most 2^23)", who, v->nseq, v->nkv);
  PQ_REQUIRE(nh > 0 && nh % v->nkv == 0 && nh / v->nkv <= 16 && win >= 0 && sinks >= 0 && max_kv > 0, PQ_ERR_ARG,
             "%s: nh=%d nkv=%d win=%d sinks=%d max_kv=%d", who, nh, v->nkv, win, sinks, max_kv);
  PQ_REQUIRE(q_stride >= nh * kv->hd && (!out || out_stride >= nh * kv->hd) && (!gate || gate_stride >= nh), PQ_ERR_ARG,
             "%s: row strides %d, %d and %d too small", who, q_stride, out_stride, gate_stride);
  return PQ_OK;
}

// One wave per (head, row); lane l holds dimensions l + 64e.
template <int HD, bool BF>
__global__ __launch_bounds__(256) void paged_prep_kernel(const uint16_t *qkv, int row_stride, uint16_t *q_out,
                                                         int q_stride, const float *__restrict__ qn,
                                                         const float *__restrict__ kn, const float *__restrict__ cs,
                                                         int rope_rows, PagedView kv, int nh, int rot, float eps) {
  constexpr int E = HD / 64;
  const int head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x;
  const int l = threadIdx.x & 63, nkv = kv.nkv, kvd = nkv * HD;
  if (head >= nh + 2 * nkv) return;
  int first, count;
  const int b = paged_seq_of_row(kv, row, first, count);
  if (b < 0) return;
  const int pos = kv.kv_len[b] - count + (row - first);
  if (pos < 0 || pos >= rope_rows) return;
  const uint16_t *xr = qkv + (size_t)row * row_stride + head * HD;
  float x[E], r[E];
#pragma unroll
  for (int e = 0; e < E; e++) r[e] = x[e] = bf2f(xr[l + 64 * e]);
  if (head < nh + nkv) {
    const float *w = head < nh ? qn : kn;
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) ss = __builtin_fmaf(x[e], x[e], ss);
    const float rs = 1.0f / sqrtf(wave_pairwise_sum(ss) * (1.0f / (float)HD) + eps);
#pragma unroll
    for (int e = 0; e < E; e++) r[e] = w[l + 64 * e] * (x[e] * rs);
    const int half = rot / 2;
    const float *c = cs + (size_t)pos * rot;
    if constexpr (HD == 64) {
      const float other = __shfl_xor(r[0], 32, 64);
      const int i = l & 31;
      if (i < half) r[0] = r[0] * c[2 * i] + (l < 32 ? -other : other) * c[2 * i + 1];
    } else if (l < half) {
      const float a = r[0], b2 = r[1];
      r[0] = a * c[2 * l] - b2 * c[2 * l + 1];
      r[1] = b2 * c[2 * l] + a * c[2 * l + 1];
    }
  }
  if (head < nh) {
#pragma unroll
    for (int e = 0; e < E; e++) q_out[(size_t)row * q_stride + head * HD + l + 64 * e] = f2bf(r[e]);
    return;
  }
  const long long at = paged_row(kv, b, pos, kvd);
  if (at < 0) return;
  const int g = head < nh + nkv ? head - nh : head - nh - nkv;
  uint16_t *dst = (head < nh + nkv ? kv.k : kv.v) + at + g * HD;
#pragma unroll
  for (int e = 0; e < E; e++) dst[l + 64 * e] = BF ? f2bf(r[e]) : f2h(r[e]);
}

}  // namespace pq

using namespace pq;

extern "C" int pq_paged_qk_prep(const uint16_t *qkv, int row_stride, uint16_t *q_out, int q_stride,
                                const float *q_norm, const float *k_norm, const float *rope_cs, int rope_rows,
                                const pq_paged_kv *kv, int nh, int rot, int T, float eps, void *stream) {
  PQ_REQUIRE(qkv && q_out && q_norm && k_norm && (rope_cs || rot == 0), PQ_ERR_ARG, "pq_paged_qk_prep: null pointer");
  PagedView v;
  const int rc = paged_view(kv, "pq_paged_qk_prep", &v);
  if (rc) return rc;
  PQ_REQUIRE(nh > 0 && nh <= 16 * v.nkv && nh % v.nkv == 0 && rot >= 0 && rot <= kv->hd && rot % 2 == 0 && T > 0 && T <= 1 << 23 &&
                 rope_rows > 0,
             PQ_ERR_ARG, "pq_paged_qk_prep: nh=%d nkv=%d rot=%d T=%d rope_rows=%d", nh, v.nkv, rot, T, rope_rows);
  PQ_REQUIRE(row_stride >= (nh + 2 * v.nkv) * kv->hd && q_stride >= nh * kv->hd, PQ_ERR_ARG,
             "pq_paged_qk_prep: row strides %d and %d too small", row_stride, q_stride);
  PQ_REQUIRE(q_out != qkv || q_stride == row_stride, PQ_ERR_ARG, "pq_paged_qk_prep: q in place needs one row stride");
  PQ_REQUIRE(kv->q_start || T == kv->nseq, PQ_ERR_ARG, "pq_paged_qk_prep: %d rows for %d sequences without q_start", T,
             kv->nseq);
  const dim3 grid(T, (nh + 2 * v.nkv + 3) / 4), block(256);
#define PQ_PREP(HH, BB)                                                                                              \
  launch(paged_prep_kernel<HH, BB>, grid, block, 0, as_stream(stream), qkv, row_stride, q_out, q_stride, q_norm, k_norm, \
         rope_cs, rope_rows, v, nh, rot, eps)
  const bool bf = kv->dtype == PQ_DTYPE_BF16;
  if (kv->hd == 64) {
    if (bf) PQ_PREP(64, true);
    else PQ_PREP(64, false);
  } else {
    if (bf) PQ_PREP(128, true);
    else PQ_PREP(128, false);
  }
#undef PQ_PREP
  return check_launch("pq_paged_qk_prep");
}
