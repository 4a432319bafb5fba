// paged.h -- what the paged-cache kernels share: the device view of a
// pq_paged_kv, the row -> (sequence, position) map and the visibility rule.
#pragma once
#include "pq_device.h"
#include "pq_host.h"

namespace pq {

// positions that are counted of any table: leaves a tile's end room in an int
constexpr int kPagedCap = 0x7fffff00;

// pq_paged_kv as the kernels take it (by value). cap: positions a table row covers.
struct PagedView {
  uint16_t *k, *v;
  long long page_stride;
  const int32_t *table, *kv_len, *q_start;
  int npages, lg_page, nkv, nseq, table_stride, cap;
};

// Checks the struct's host-side fields; fills the view.
int paged_view(const pq_paged_kv *kv, const char *who, PagedView *out);
// The checks that both attentions share, the view's among them.
int paged_attn_check(const char *who, const uint16_t *q, int q_stride, const pq_paged_kv *kv, const uint16_t *gate,
                     int gate_stride, const uint16_t *out, int out_stride, const int8_t *qx, const float *dx, int nh,
                     int win, int sinks, int max_kv, PagedView *v);

// The sequence that row belongs to (the wave's lanes scan q_start together), or
// -1; first / count: its rows. row must be uniform over the wave.
__device__ __forceinline__ int paged_seq_of_row(const PagedView &kv, int row, int &first, int &count) {
  if (kv.q_start == nullptr) {
    first = row;
    count = 1;
    return row < kv.nseq ? row : -1;
  }
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int i = 0; i < kv.nseq; i += 64)
    b += __popcll(__ballot(i + lane < kv.nseq && kv.q_start[i + lane < kv.nseq ? i + lane + 1 : 0] <= row));
  if (b >= kv.nseq) return -1;
  first = kv.q_start[b];
  const int end = kv.q_start[b + 1];
  count = end - first;
  return row >= first && row < end ? b : -1;
}

// kv_len[b], a length below any call's rows standing for none (so that a row's position does not wrap)
__device__ __forceinline__ int paged_len(const PagedView &kv, int b) {
  const int n = kv.kv_len[b];
  return n < -(1 << 24) ? -(1 << 24) : n;
}

// Element offset of position j's row of kv heads in the pools, or -1 when it
// has none (past the table, or a page outside the pool).
__device__ __forceinline__ long long paged_row(const PagedView &kv, int b, int j, int kvd) {
  if (j < 0 || j >= kv.cap) return -1;
  const int id = kv.table[(size_t)b * kv.table_stride + (j >> kv.lg_page)];
  if (id < 0 || id >= kv.npages) return -1;
  return id * kv.page_stride + (long long)(j & ((1 << kv.lg_page) - 1)) * kvd;
}

// fp16 or bf16 cache element -> f32 and back
template <bool BF>
__device__ __forceinline__ float kv2f(uint16_t v) {
  if constexpr (BF) return bf2f(v);
  else return h2f(v);
}

// Four adjacent dims (d0 a multiple of 4) of one row's head, o unnormalized with
// the sum l: the division, the gate, the one rounding to bf16, and the Q8_0 form
// (a block is 8 adjacent threads' dims). some: the row sees a key.
template <int HD>
__device__ __forceinline__ void paged_store4(const float *o, float l, bool some, int row, int h, int d0, int nh,
                                             const uint16_t *gate, int gate_stride, uint16_t *out, int out_stride,
                                             int8_t *qx, float *dx) {
  float f = 1.0f / l;
  if (gate != nullptr) f = f / (1.0f + expf_pq(-bf2f(gate[(size_t)row * gate_stride + h])));
  uint16_t r[4];
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = some ? f2bf(o[i] * f) : 0;
  if (out != nullptr) {
    uint16_t *dst = out + (size_t)row * out_stride + h * HD + d0;
    if (((uintptr_t)dst & 7) == 0) {
      *reinterpret_cast<uint2 *>(dst) = make_uint2(r[0] | (uint32_t)r[1] << 16, r[2] | (uint32_t)r[3] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) dst[i] = r[i];
    }
  }
  if (qx != nullptr) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) a = fmaxf(a, fabsf(bf2f(r[i])));
    a = fmaxf(a, dpp_f<kDppXor1>(a));
    a = fmaxf(a, dpp_f<kDppXor2>(a));
    a = fmaxf(a, dpp_f<kDppHalfMirror>(a));
    const float d = a / 127.0f;
    const Q8Div dv(d);
    const size_t at = ((size_t)row * nh + h) * HD + d0;
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) q |= (uint32_t)(uint8_t)(int8_t)q8_code(dv.div(bf2f(r[i]))) << (8 * i);
    __builtin_memcpy(qx + at, &q, 4);
    if ((d0 & 31) == 0) dx[at / 32] = d;
  }
}

}  // namespace pq
