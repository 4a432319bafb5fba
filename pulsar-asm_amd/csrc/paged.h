// paged.h -- what the paged-cache kernels share: the device view of a
// pq_paged_kv, the row -> (sequence, position) map, a position's place in the pools
// and the output step.
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

// Of 64 lanes' "the start of my sequence is at most the next one's": those before the first that is not.
__device__ __forceinline__ uint64_t paged_ascending(uint64_t up) { return up & ~(up + 1); }

// The sequence that row of the call belongs to (the wave's lanes scan q_start
// together), or -1; left: the rows from this one to the sequence's end, so that its
// position is kv_len - left. A start above the next one ends the sequences: that
// sequence and those behind it have no rows. row must be uniform over the wave.
__device__ __forceinline__ int paged_seq_of_row(const PagedView &kv, int row, int &left) {
  if (kv.q_start == nullptr) {
    left = 1;
    return row < kv.nseq ? row : -1;
  }
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < kv.nseq; i += 64) {
    const int j = i + lane, jc = j < kv.nseq ? j : kv.nseq - 1;
    const int first = kv.q_start[jc], next = kv.q_start[jc + 1];
    const uint64_t up = __ballot(j < kv.nseq && first <= next);
    const uint64_t hit = __ballot(first <= row && row < next) & paged_ascending(up);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      left = __builtin_amdgcn_readlane(next, l) - row;
      return i + l;
    }
    if (up != ~0ull) break;
  }
  return -1;
}

// Element offset of position j's row of kv heads in the pools, or -1 when it
// has none (past the table, or a page outside the pool).
__device__ __forceinline__ long long paged_row(const PagedView &kv, int b, int j, int kvd) {
  if (j < 0 || j >= kv.cap) return -1;
  const int id = kv.table[(size_t)b * kv.table_stride + (j >> kv.lg_page)];
  if (id < 0 || id >= kv.npages) return -1;
  return id * kv.page_stride + (long long)(j & ((1 << kv.lg_page) - 1)) * kvd;
}

// A finite scale's multiplier of the scores, cut to the finite ones where the queries' exponent takes it past them: a
// score of 0 stays 0.
__device__ __forceinline__ float paged_finite(float sc, float scale) {
  constexpr float most = 0x1.fffffep127f;
  return fabsf(scale) <= most ? fminf(fmaxf(sc, -most), most) : sc;
}

// fp16 or bf16 cache element -> f32
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
