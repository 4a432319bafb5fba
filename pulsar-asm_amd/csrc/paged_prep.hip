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
  out->cap = cap < kPagedCap ? (int)cap : kPagedCap;
  return PQ_OK;
}

int paged_attn_check(const char *who, const uint16_t *q, int q_stride, const pq_paged_kv *kv, const uint16_t *gate,
                     int gate_stride, const uint16_t *out, int out_stride, const int8_t *qx, const float *dx, int nh,
                     int win, int sinks, int max_kv, PagedView *v) {
  PQ_REQUIRE(q && (out || qx) && (!qx || dx), PQ_ERR_ARG, "%s: null pointer", who);
  const int rc = paged_view(kv, who, v);
  if (rc) return rc;
  PQ_REQUIRE((long long)v->nseq * v->nkv <= 1 << 23, PQ_ERR_ARG, "%s: nseq=%d x nkv=%d (at most 2^23)", who, v->nseq, v->nkv);
  PQ_REQUIRE(nh > 0 && nh % v->nkv == 0 && nh / v->nkv <= 16 && win >= 0 && win <= 1 << 30 && sinks >= 0 && max_kv > 0,
             PQ_ERR_ARG,
             "%s: nh=%d nkv=%d win=%d sinks=%d max_kv=%d", who, nh, v->nkv, win, sinks, max_kv);
  PQ_REQUIRE(q_stride >= nh * kv->hd && (!out || out_stride >= nh * kv->hd) && (!gate || gate_stride >= nh), PQ_ERR_ARG,
             "%s: row strides %d, %d and %d too small", who, q_stride, out_stride, gate_stride);
  return PQ_OK;
}

// y = w x / sqrt(mean(x^2) + eps) of each q and k head, then the rotation of the
// pairs (i, i + hd/2), i < rot/2, by the row's position; v as it is. fp32 from the
// bf16 inputs to the one rounding of the stores.
//
// A wave takes one row and U heads of it a turn: lane (u, c) = (lane / TH, lane %
// TH), TH = HD / 16 lanes a head, holds dims 8 c .. + 7 and HD / 2 + 8 c .. + 7 of
// head u, so that a rotation pair lies in one lane, each load is 16 bytes, and the
// row's cosines and sines and the norm weights, the same for every head, are read
// once a wave. The sum of squares is the lane's 16, then a butterfly over TH lanes.
//
// What bounds it is memory: each row read and written once. 19487 rows of 32 q and 8 kv
// heads of 64 52 us (240 MB, 4.65 TB/s; a large copy reaches 4.7 to 5.0), a wave a head
// row with 2-byte lanes 269, the norm weights read each turn 61. turns: a row's heads by
// one wave where the rows fill the chip, else a turn a wave (few rows are bound by the
// call: 8.5 us, the kernel 3.4).
template <int HD, bool BF>
__global__ __launch_bounds__(256) void paged_prep_kernel(const uint16_t *qkv, int row_stride, uint16_t *q_out,
                                                         int q_stride, const float *__restrict__ qn,
                                                         const float *__restrict__ kn, const float *__restrict__ cs,
                                                         int rope_rows, PagedView kv, int nh, int rot, float eps, int T,
                                                         int turns, int vec) {
  constexpr int TH = HD / 16, U = 64 / TH;   // lanes a head, heads a turn
  const int lane = threadIdx.x & 63, u = lane / TH, c = lane % TH;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nkv = kv.nkv, kvd = nkv * HD, heads = nh + 2 * nkv;
  const int parts = (heads + U * turns - 1) / (U * turns);   // waves a row
  const long long id = (long long)blockIdx.x * 4 + w;
  const int row = (int)(id / parts), h0 = (int)(id % parts) * U * turns;
  if (row >= T) return;
  int left;
  const int b = paged_seq_of_row(kv, row, left);
  if (b < 0) return;
  const int len = kv.kv_len[b];
  if (len < left || len - left >= rope_rows) return;
  const int pos = len - left;
  const long long at = paged_row(kv, b, pos, kvd);
  const int half = rot / 2;
  // the cosines and sines of this lane's pairs; 1 and 0 past the rotated dims
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 8; i++) co[i] = 1.0f, si[i] = 0.0f;
  const float *cr = cs + (size_t)pos * rot + 16 * c;
  if (vec && 8 * c + 8 <= half) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float4 v = *reinterpret_cast<const float4 *>(cr + 2 * i);
      co[i] = v.x, si[i] = v.y, co[i + 1] = v.z, si[i + 1] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (8 * c + i < half) co[i] = cr[2 * i], si[i] = cr[2 * i + 1];
  }
  float wq[2][8], wk[2][8];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const float *a = qn + e * (HD / 2) + 8 * c, *d = kn + e * (HD / 2) + 8 * c;
    if (vec) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 va = *reinterpret_cast<const float4 *>(a + i), vd = *reinterpret_cast<const float4 *>(d + i);
        wq[e][i] = va.x, wq[e][i + 1] = va.y, wq[e][i + 2] = va.z, wq[e][i + 3] = va.w;
        wk[e][i] = vd.x, wk[e][i + 1] = vd.y, wk[e][i + 2] = vd.z, wk[e][i + 3] = vd.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) wq[e][i] = a[i], wk[e][i] = d[i];
    }
  }
  for (int t = 0; t < turns; t++) {
    const int head = h0 + t * U + u;
    if (h0 + t * U >= heads) break;
    const bool on = head < heads, norm = head < nh + nkv;
    const uint16_t *xr = qkv + (size_t)row * row_stride + (on ? head : 0) * HD + 8 * c;
    uint32_t xw[2][4];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (vec) {
        const uint4 v = *reinterpret_cast<const uint4 *>(xr + e * (HD / 2));
        xw[e][0] = v.x, xw[e][1] = v.y, xw[e][2] = v.z, xw[e][3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) xw[e][i] = xr[e * (HD / 2) + 2 * i] | (uint32_t)xr[e * (HD / 2) + 2 * i + 1] << 16;
      }
    }
    float x[2][8], ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[e][i] = __uint_as_float(i & 1 ? xw[e][i >> 1] & 0xffff0000u : xw[e][i >> 1] << 16);
        ss = __builtin_fmaf(x[e][i], x[e][i], ss);
      }
    ss += dpp_f<kDppXor1>(ss);
    ss += dpp_f<kDppXor2>(ss);
    if constexpr (TH == 8) ss += dpp_f<kDppHalfMirror>(ss);
    if (norm) {
      const float rs = 1.0f / sqrtf(ss * (1.0f / (float)HD) + eps);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float a = (head < nh ? wq[0][i] : wk[0][i]) * (x[0][i] * rs), d = (head < nh ? wq[1][i] : wk[1][i]) * (x[1][i] * rs);
        x[0][i] = a * co[i] - d * si[i];
        x[1][i] = d * co[i] + a * si[i];
      }
    }
    if (!on) continue;
    const int g = head < nh + nkv ? head - nh : head - nh - nkv;
    if (head >= nh && at < 0) continue;
    uint16_t *dst = head < nh ? q_out + (size_t)row * q_stride + head * HD : (norm ? kv.k : kv.v) + at + g * HD;
    const bool wide = head >= nh || vec;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      uint32_t y[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = x[e][2 * i], d = x[e][2 * i + 1];
        y[i] = head < nh || BF ? f2bf2(a, d) : (uint32_t)f2h(a) | (uint32_t)f2h(d) << 16;
      }
      uint16_t *to = dst + e * (HD / 2) + 8 * c;
      if (wide) {
        *reinterpret_cast<uint4 *>(to) = make_uint4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) to[2 * i] = (uint16_t)y[i], to[2 * i + 1] = (uint16_t)(y[i] >> 16);
      }
    }
  }
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
  // 16-byte loads and stores of whole lanes where the rows allow it (the pools always do)
  const int vec = aligned(qkv, 16) && row_stride % 8 == 0 && aligned(q_out, 16) && q_stride % 8 == 0 &&
                  aligned(rope_cs, 16) && rot % 4 == 0 && aligned(q_norm, 16) && aligned(k_norm, 16);
  const int heads = nh + 2 * v.nkv, U = 64 / (kv->hd / 16), groups = (heads + U - 1) / U;
  const int turns = (long long)T * groups > 8192 ? groups : 1;
  const long long waves = (long long)T * ((heads + U * turns - 1) / (U * turns));
  PQ_REQUIRE((waves + 3) / 4 <= 1 << 24, PQ_ERR_ARG, "pq_paged_qk_prep: %d rows of %d heads are too many for one call", T, heads);
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
#define PQ_PREP(HH, BB)                                                                                              \
  launch(paged_prep_kernel<HH, BB>, grid, block, 0, as_stream(stream), qkv, row_stride, q_out, q_stride, q_norm, k_norm, \
         rope_cs, rope_rows, v, nh, rot, eps, T, turns, vec)
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
