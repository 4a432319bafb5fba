// paged_attn.hip -- attention over a paged cache (gfx950): one new token a
// sequence, and prompt rows of a ragged batch.
//
// A row at position p sees keys j <= p with win == 0, or j > p - win, or j <
// sinks: sinks [0, ns), ns = min(sinks, lo), and the window [lo, p], lo =
// max(0, p + 1 - win). s_j = scale q.k_j; the softmax is kept online, a running
// maximum m, sum l = sum e^(s_j - m) and value sum o = sum e^(s_j - m) v_j, all
// fp32.
#include "paged.h"

namespace pq {

// One workgroup per (head, row), 4 waves that take the row's keys in turn; lane
// = dimensions lane + 64e. The waves' states join through LDS.
template <int HD, bool BF>
__global__ __launch_bounds__(256) void paged_attn_kernel(const uint16_t *__restrict__ q, int q_stride, PagedView kv,
                                                         const uint16_t *__restrict__ gate, int gate_stride,
                                                         uint16_t *__restrict__ out, int out_stride,
                                                         int8_t *__restrict__ qx, float *__restrict__ dx, int nh,
                                                         float scale, int win, int sinks) {
  constexpr int E = HD / 64;
  __shared__ float sm[4], sl[4], so[4][HD];
  const int h = blockIdx.y, row = blockIdx.x, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = h / (nh / kv.nkv), kvd = kv.nkv * HD;
  int first, count;
  const int b = paged_seq_of_row(kv, row, first, count);
  if (b < 0) return;
  const int p = kv.kv_len[b] - count + (row - first);
  const int lo = win > 0 && p >= win ? p + 1 - win : 0;
  const int ns = sinks < lo ? sinks : lo;
  float qv[E], o[E], m = -__builtin_inff(), l = 0.0f;
  bool seen = false;
#pragma unroll
  for (int e = 0; e < E; e++) {
    qv[e] = bf2f(q[(size_t)row * q_stride + h * HD + lane + 64 * e]);
    o[e] = 0.0f;
  }
  const int n = p < 0 ? 0 : ns + (p + 1 - lo);
  for (int i = w; i < n; i += 4) {
    const int j = i < ns ? i : lo + (i - ns);
    const long long at = paged_row(kv, b, j, kvd);
    if (at < 0) continue;
    float d = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) d = __builtin_fmaf(qv[e], kv2f<BF>(kv.k[at + g * HD + lane + 64 * e]), d);
    const float s = wave_pairwise_sum(d) * scale;
    const float mn = seen ? fmaxf(m, s) : s;
    const float c = seen ? expf_pq(m - mn) : 0.0f, x = expf_pq(s - mn);
    l = __builtin_fmaf(l, c, x);
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = __builtin_fmaf(x, kv2f<BF>(kv.v[at + g * HD + lane + 64 * e]), o[e] * c);
    m = mn;
    seen = true;
  }
  if (lane == 0) {
    sm[w] = seen ? m : -__builtin_inff();
    sl[w] = seen ? l : -1.0f;   // no key
  }
#pragma unroll
  for (int e = 0; e < E; e++) so[w][lane + 64 * e] = o[e];
  __syncthreads();
  if (w != 0) return;
  float M = -__builtin_inff(), L = 0.0f, O[E];
  bool any = false;
#pragma unroll
  for (int e = 0; e < E; e++) O[e] = 0.0f;
  for (int k = 0; k < 4; k++) {
    if (sl[k] < 0.0f) continue;
    M = any ? fmaxf(M, sm[k]) : sm[k];
    any = true;
  }
  for (int k = 0; k < 4; k++) {
    if (sl[k] < 0.0f) continue;
    const float c = expf_pq(sm[k] - M);
    L = __builtin_fmaf(sl[k], c, L);
#pragma unroll
    for (int e = 0; e < E; e++) O[e] = __builtin_fmaf(so[k][lane + 64 * e], c, O[e]);
  }
  const float gs = gate != nullptr ? 1.0f / (1.0f + expf_pq(-bf2f(gate[(size_t)row * gate_stride + h]))) : 1.0f;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const uint16_t r = any ? f2bf(O[e] / L * gs) : 0;
    const int d = lane + 64 * e;
    if (out != nullptr) out[(size_t)row * out_stride + h * HD + d] = r;
    if (qx != nullptr) {
      const float v = bf2f(r);
      float a = fabsf(v);
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) a = fmaxf(a, __shfl_xor(a, k, 64));
      const float dq = a / 127.0f;
      const size_t K = (size_t)nh * HD;
      qx[(size_t)row * K + h * HD + d] = (int8_t)q8_code(Q8Div(dq).div(v));
      if ((lane & 31) == 0) dx[(size_t)row * (K / 32) + (h * HD + d) / 32] = dq;
    }
  }
}

}  // namespace pq

using namespace pq;

static int paged_attn(const char *who, const uint16_t *q, int q_stride, const pq_paged_kv *kv, const uint16_t *gate,
                      int gate_stride, uint16_t *out, int out_stride, int8_t *qx, float *dx, int nh, int T, float scale,
                      int win, int sinks, int max_kv, void *stream) {
  PagedView v;
  const int rc = paged_attn_check(who, q, q_stride, kv, gate, gate_stride, out, out_stride, qx, dx, nh, win, sinks, max_kv, &v);
  if (rc) return rc;
  PQ_REQUIRE(T > 0 && T <= 1 << 23 && (v.q_start || T == kv->nseq), PQ_ERR_ARG, "%s: %d rows for %d sequences%s", who, T, kv->nseq,
             v.q_start ? "" : " without q_start");
#define PQ_ATT(HH, BB)                                                                                               \
  launch(paged_attn_kernel<HH, BB>, dim3(T, nh), dim3(256), 0, as_stream(stream), q, q_stride, v, gate, gate_stride, \
         out, out_stride, qx, dx, nh, scale, win, sinks)
  const bool bf = kv->dtype == PQ_DTYPE_BF16;
  if (kv->hd == 64) {
    if (bf) PQ_ATT(64, true);
    else PQ_ATT(64, false);
  } else {
    if (bf) PQ_ATT(128, true);
    else PQ_ATT(128, false);
  }
#undef PQ_ATT
  return check_launch(who);
}

extern "C" size_t pq_paged_prefill_workspace_bytes(int nseq, int T, int nh, int nkv, int hd, int max_kv, int win,
                                                   int sinks) {
  return 0;
}

extern "C" int pq_paged_attn_prefill(const uint16_t *q, int q_stride, const pq_paged_kv *kv, const uint16_t *gate,
                                     int gate_stride, uint16_t *out, int out_stride, int8_t *qx, float *dx, int nh,
                                     int T, float scale, int win, int sinks, int max_kv, void *ws, size_t ws_bytes,
                                     void *stream) {
  return paged_attn("pq_paged_attn_prefill", q, q_stride, kv, gate, gate_stride, out, out_stride, qx, dx, nh, T,
                    scale, win, sinks, max_kv, stream);
}
