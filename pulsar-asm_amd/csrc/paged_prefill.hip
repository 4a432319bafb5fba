// paged_prefill.hip -- attention of prompt rows over a paged cache (gfx950):
// tiles of 32 NW rows against tiles of 64 keys on the matrix cores, for a ragged
// batch, with a sliding window whose first tokens stay visible.
//
// A row at position p sees keys j <= p with win == 0, or j > p - win, or j < sinks.
// s_j = scale q.k_j; the softmax is online: running maximum m, l = sum 2^(s'_j - m),
// o = sum 2^(s'_j - m) v_j with s' = s log2(e), all fp32.
//
// The rows of a (sequence, kv head) are its queries' G = nh / nkv heads, query by
// query: row r is head r % G of query r / G, so a tile's rows share every key and
// the causal edge costs one or two tiles of keys. A wave holds 32 rows as the
// columns of 32x32x16 products:
//   scores  S^T [key][row] = K Q^T: K from LDS (16 bytes a lane), Q in registers;
//   values  O^T [dim][row] += V^T P^T: V read from LDS through the transposing read.
// Row m of the score product is key swap(m) (bits 2 and 3 of m exchanged), so that
// the 16 scores a lane gets of 32 keys, rows 8 a + 4 h + c of half h, are keys 16 t
// + 8 h + j: the very k index of the value product, and P^T needs no shuffle.
//
// K and V go from memory to LDS without registers, a tile ahead in two buffers;
// a lane's 16 bytes land at 16 lane, so the swizzle that spreads rows over the
// banks is in the address that the lane reads from: chunk c of row r is held at c ^ f(r)
// (no bank conflicts; V's first swizzle had a third of the LDS cycles in them).
//
// What bounds it: the matrix cores and the vector unit by turns. A wave's tile is 32
// products of 32 cycles (head_dim 128; 16 for 64) and 150 to 160 vector instructions (137
// to 145 with a bf16 pool), 32 of them e^x; the two waves of a SIMD are at the same step behind each
// barrier, so the two add up: 47% of the cycles in products, 43% in vector instructions.
// Tiles that some row sees in part cost half as much again. Measured: 16384 queries of 16 q
// and 4 kv heads of 128 1.07 to 1.10 ms (1.0 PFLOP/s; a large library product reaches 1.3),
// 2048 queries behind 14336 in 8 sequences 1.01 PFLOP/s, 8192 queries of 32 and 8 heads of 64
// 344 us (800 TFLOP/s), 16384 in a window of 256 with 4 sinks 99 us, 512 behind 32000 in 8
// splits 155 to 159 us, ragged prompts of up to 2048 of 32 and 8 heads of 64 137 to 145 us.
#include <type_traits>

#include "paged.h"

namespace pq {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;   // keys of a tile

__device__ const uint4 paged_zero[16] = {};   // a row of zeros: what a key that no row sees reads

template <bool BF>
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
  typedef __bf16 v8b __attribute__((ext_vector_type(8)));
  typedef _Float16 v8h __attribute__((ext_vector_type(8)));
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// (a, b) rounded to the cache's type, packed low, high
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) {
    return f2bf2(a, b);
  } else {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const pq_f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, v2h));
  }
}

// c plus both bf16 of w: one dot product with (1, 1), within 1.5 * 2^-23 of the sum
__device__ __forceinline__ float add_bf2(uint32_t w, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pq_bf16x2, w), __builtin_bit_cast(pq_bf16x2, 0x3f803f80u), c, false);
}

// the largest of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) v4u lds_v4u;

// both halves of a dword whose exponent is all ones
template <bool BF>
__device__ __forceinline__ bool odd16(uint32_t v) {
  constexpr uint32_t e = BF ? 0x7f80u : 0x7c00u;
  return (v & e) == e || (v & (e << 16)) == e << 16;
}
template <bool BF>
__device__ __forceinline__ uint32_t finite16(uint32_t v) {
  constexpr uint32_t e = BF ? 0x7f80u : 0x7c00u;
  if ((v & e) == e) v &= 0xffff0000u;
  if ((v & (e << 16)) == e << 16) v &= 0xffffu;
  return v;
}

struct PrefillArgs {
  const uint16_t *q, *gate;
  uint16_t *out;
  int8_t *qx;
  float *dx, *po, *pml;
  int q_stride, gate_stride, out_stride, nh, G, T, win, sinks, nsplit, qvec, ovec;
  float scale;
};

// Grid (row tiles x kv heads, splits). Slot s of the row tiles: sequence b has the
// slots from floor(q_start[b] G / BM) + b on, one more than it can need at most.
// Three waves a SIMD for head_dim 64 (8192 queries 408 -> 392 us), two for 128. Of the fp16 forms 7 and 5 registers are
// spilled for it, outside the inner run.
template <int HD, bool BF, int NW>
__global__ __launch_bounds__(64 * NW, HD == 64 ? 3 : 2) void paged_prefill_kernel(PrefillArgs A, PagedView kv, int slots) {
  constexpr int BM = 32 * NW, S = HD / 16, N = HD / 32, RB = HD * 2;       // rows, score steps, dim tiles, bytes a row
  constexpr int TB = kKeys * RB, RPI = 1024 / RB, LI = TB / 1024 / NW;     // bytes a tile, rows and a wave's loads
  static_assert(LI >= 1, "a wave loads whole pieces");
  __shared__ __align__(1024) char smem[4 * TB];                            // [2][K, V][64][HD]
  __shared__ uint32_t odd_flag[2][NW];
  const int lane = threadIdx.x & 63, m = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % kv.nkv, slot = slots - 1 - blockIdx.x / kv.nkv;
  const int G = A.G, kvd = kv.nkv * HD;
  // the sequence of the slot, its rows and its length: lane j reads sequence i + j's, the last one that starts at the
  // slot or before is taken, of those up to a start that does not ascend (as paged_seq_of_row has them)
  int b = -1, q0 = 0, q1 = 0, len = 0;
  for (int i = 0; i < kv.nseq; i += 64) {
    const int j = i + lane, jc = j < kv.nseq ? j : kv.nseq - 1;
    const int first = kv.q_start != nullptr ? kv.q_start[jc] : jc, next = kv.q_start != nullptr ? kv.q_start[jc + 1] : jc + 1;
    const int n = kv.kv_len[jc];
    const int at = (first > 0 ? (int)((long long)first * G / BM) : 0) + j;
    const uint64_t up = __ballot(j < kv.nseq && first <= next);
    const int before = __popcll(__ballot(at <= slot) & paged_ascending(up));
    if (before == 0) break;
    b = i + before - 1;
    q0 = __builtin_amdgcn_readlane(first, before - 1);
    q1 = __builtin_amdgcn_readlane(next, before - 1);
    len = __builtin_amdgcn_readlane(n, before - 1);
    if (up != ~0ull) break;
  }
  if (b < 0) return;
  // its rows within the call's, and the position of the first: row i of them is at p0 + i. Below -2^24 none of 2^23 rows
  // has one
  if (q0 < 0) q0 = 0;
  const int left = q1 - q0;
  if (q1 > A.T) q1 = A.T;
  if (q1 <= q0) return;
  const int rows = (q1 - q0) * G, r0 = (slot - ((int)((long long)q0 * G / BM) + b)) * BM;
  if (r0 >= rows) return;
  const int p0 = (long long)len - left > -(1 << 24) ? len - left : -(1 << 24);
  const int rlast = r0 + BM < rows ? r0 + BM - 1 : rows - 1;
  const int pmin = p0 + r0 / G, pmax = p0 + rlast / G;
  const int limit = pmax + 1 < kv.cap ? pmax + 1 : kv.cap;                 // keys from here on are no row's
  const int lo = A.win > 0 && pmin >= A.win ? pmin + 1 - A.win : 0;
  const int wt = lo / kKeys;
  int te = limit > 0 ? (limit + kKeys - 1) / kKeys : 0;
  int st = ((A.sinks < limit ? A.sinks : limit) + kKeys - 1) / kKeys;
  st = st < wt ? (st > 0 ? st : 0) : wt;
  const int nt = st + (te > wt ? te - wt : 0);
  const int each = (nt + A.nsplit - 1) / A.nsplit;
  const int t0 = blockIdx.y * each, t1 = t0 + each < nt ? t0 + each : nt;
  const int gap = wt - st;
  auto tile_base = [&](int i) { return (i < st ? i : i + gap) * kKeys; };
  // this lane's row
  const int r = r0 + 32 * w + m, rc = r < rows ? r : rows - 1;
  const int qi = rc / G, head = g * G + (rc - qi * G), row = q0 + qi, pos = p0 + qi;
  const int low = A.win > 0 ? pos - A.win : -1;                            // sees key > low (or a sink)
  const int wr0 = r0 + 32 * w < rows ? r0 + 32 * w : rows - 1, wr1 = wr0 + 31 < rows ? wr0 + 31 : rows - 1;
  const int wmin = p0 + wr0 / G, wmax = p0 + wr1 / G;                      // the wave's positions
  const bool idle = r0 + 32 * w >= rows;                                   // a wave without rows only loads

  // loads of a tile: this wave's pieces of K and V. ids: lane i holds the page of the tile's keys 8 (i % 8) ..
  const int32_t *tb = kv.table + (size_t)b * kv.table_stride;
  const int smask = (1 << kv.lg_page) - 1;
  auto page_ids = [&](int i) {
    const int j = tile_base(i) + 8 * (lane & 7);
    return i < t1 && j < limit ? tb[j >> kv.lg_page] : -1;
  };
  // a piece is RPI rows of one page: its address is the wave's, the lane's part of it the same for every piece
  const int lrow = lane / (64 / RPI), lch = lane % (64 / RPI);   // row of the piece, chunk of the row
  const int prow = w * RPI + lrow;                               // the row's place in the swizzle (pieces are NW apart)
  const int ck = HD == 128 ? lch ^ (prow & 15) : lch ^ ((prow >> 1) & 7);
  const int cv = HD == 128 ? lch ^ 4 * (prow & 3) : lch ^ 4 * ((prow >> 1) & 1);
  const uint32_t offk = (uint32_t)(lrow * kvd + 8 * ck) * 2, offv = (uint32_t)(lrow * kvd + 8 * cv) * 2;
  // Written as asm so that its completion is waited for where the tile is taken up and not at every read of LDS.
  const uint32_t lds0 = (uint32_t)(size_t)(lds_char *)smem;
  auto dma = [&](const char *src, uint32_t off, uint32_t dst) {   // src uniform
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds0 + dst), "v"(off), "s"(src) : "memory", "m0");
  };
  auto dma_each = [&](const char *src, uint32_t dst) {            // src each lane's own
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds0 + dst), "v"(src) : "memory", "m0");
  };
  const char *const kbase = reinterpret_cast<const char *>(kv.k + g * HD), *const vbase = reinterpret_cast<const char *>(kv.v + g * HD);
  const long long pstride = kv.page_stride * 2;
  const int kvd2 = kvd * 2;
  auto load = [&](int i, int buf, int ids) {
    const int base = tile_base(i);
#pragma unroll
    for (int x = 0; x < LI; x++) {
      const int piece = w + x * NW, r0p = base + piece * RPI;
      const int id = __builtin_amdgcn_readlane(ids, piece * RPI / 8);
      const bool page = (unsigned)id < (unsigned)kv.npages;
      const long long at = (page ? id : 0) * pstride + (long long)(r0p & smask) * kvd2;
      const char *ks = kbase + at, *vs = vbase + at;
      const uint32_t dst = buf * 2 * TB + piece * 1024;
      if (page && r0p + RPI <= limit) {
        dma(ks, offk, dst);
        dma(vs, offv, dst + TB);
      } else {   // rows that no row sees read zeros
        const bool ok = page && r0p + lrow < limit;
        dma_each(ok ? ks + offk : reinterpret_cast<const char *>(paged_zero), dst);
        dma_each(ok ? vs + offv : reinterpret_cast<const char *>(paged_zero), dst + TB);
      }
    }
  };
  int ids = page_ids(t0);
  if (t0 < t1) load(t0, 0, ids);
  int ids_next = page_ids(t0 + 1);

  // Q: the operand's column m, dims 16 s + 8 h ..; the scale's sign goes into it. An fp16 cache meets fp16 queries,
  // scaled by the power of two that brings the row's largest value into [1, 2): exact but for what lies 2^-25 below it
  v4u qf[S];
  float sc = fabsf(A.scale) * 1.44269504088896341f;
  {
    const uint16_t *qr = A.q + (size_t)row * A.q_stride + (size_t)head * HD + 8 * h;
    const uint32_t flip = A.scale < 0.0f ? 0x80008000u : 0u;
    float amax = 0.0f;
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (A.qvec) {
        qf[s] = *reinterpret_cast<const v4u *>(qr + 16 * s);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) qf[s][i] = qr[16 * s + 2 * i] | (uint32_t)qr[16 * s + 2 * i + 1] << 16;
      }
    }
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        qf[s][i] ^= flip;
        amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(qf[s][i] << 16)), fabsf(__uint_as_float(qf[s][i] & 0xffff0000u))));
      }
    if constexpr (!BF) {
      amax = max_half_pair(amax);
      const int e = amax > 0.0f && amax < __builtin_inff() ? (int)__builtin_amdgcn_frexp_expf(amax) - 1 : 0;
      sc = __builtin_amdgcn_ldexpf(sc, e);
#pragma unroll
      for (int s = 0; s < S; s++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          qf[s][i] = pack2<false>(__builtin_amdgcn_ldexpf(__uint_as_float(qf[s][i] << 16), -e),
                                  __builtin_amdgcn_ldexpf(__uint_as_float(qf[s][i] & 0xffff0000u), -e));
    }
    // 0 as the scale or what is left of it: the least number, so that a hidden score's product is still -infinity and
    // any finite one's below 2^-21, the weights 1
    if (sc == 0.0f) sc = 0x1p-149f;
    sc = paged_finite(sc, A.scale);
  }

  // LDS addresses: K's row swap(m) of a 32-key half, chunk 2 s + h; V's key and dims of the transposing read
  const int km = (m & ~12) | (m & 4) << 1 | (m & 8) >> 1;
  const int ksw = HD == 128 ? km & 15 : (km >> 1) & 7;
  const int li = lane & 15, g2 = (lane >> 4) & 1;
  lds_char *const lds = (lds_char *)smem;
  auto k_frag = [&](int buf, int u, int s) {
    const int at = km * RB + (((2 * s + h) ^ ksw) * 16);
    return *(const lds_v4u *)(lds + at + buf * 2 * TB + u * 32 * RB);
  };
  auto v_frag = [&](int buf, int nn, int t) {
    v4u f;
#pragma unroll
    for (int x = 0; x < 2; x++) {
      // key 16 t + 8 h + 4 x + li / 4, chunk 4 nn + 2 g2 + (li % 4) / 2 under its swizzle
      const int chunk = 4 * (nn ^ (HD == 128 ? li >> 2 : li >> 3)) + 2 * g2 + ((li & 3) >> 1);
      const int at = (8 * h + (li >> 2)) * RB + chunk * 16 + (li & 1) * 8;
      const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(lds + at + buf * 2 * TB + TB + (16 * t + 4 * x) * RB));
      f[2 * x] = (uint32_t)(uint16_t)y[0] | (uint32_t)(uint16_t)y[1] << 16;
      f[2 * x + 1] = (uint32_t)(uint16_t)y[2] | (uint32_t)(uint16_t)y[3] << 16;
    }
    return f;
  };

  // fp16 weights are held as 2^7 of theirs: what is lost below fp16's range is then 2^-31 of the largest. The maximum
  // that is taken off lags the true one by up to 2^8, so that the sums are rarely rescaled.
  constexpr float kLift = BF ? 0.0f : 7.0f, kLag = 8.0f;
  float mx = -__builtin_inff(), l = 0.0f;
  bool some = false;
  v16f o[N];
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int k = 0; k < 16; k++) o[i][k] = 0.0f;

  auto scores = [&](v16f(&s)[2], int buf) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int k = 0; k < 16; k++) s[u][k] = 0.0f;
#pragma unroll
      for (int k = 0; k < S; k++) s[u] = mfma32<BF>(k_frag(buf, u, k), qf[k], s[u]);
    }
  };
  auto largest = [&](const v16f(&s)[2]) {
    float mt = max3(s[0][0], s[1][0], s[0][1]);
#pragma unroll
    for (int i = 1; i < 15; i++) mt = max3(mt, s[1][i], s[0][i + 1]);
    mt = max3(mt, s[1][15], mt);
    return max_half_pair(mt) * sc;
  };
  // The weights and their sum. A bf16 pool's weights lose up to 2^-8 of themselves before the value product, so what is
  // summed is what is left of them: the roundings then weigh the values and do not scale the output. (A weight as two
  // bf16, as in the decode kernel, takes half as many products again: 16384 queries 1067 -> 1448 us, 512 behind 32000
  // 155 -> 203, for an error of 0.0017 of the outputs' norm where it is 0.0019 to 0.0022; the output's rounding is 0.0017.)
  auto weights = [&](const v16f(&s)[2], v4u(&p)[4]) {
    const float off = (mx == -__builtin_inff() ? 0.0f : mx) - kLift;
    float ls[4] = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], sc, -off));
        const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i + 1], sc, -off));
        if constexpr (!BF) ls[(i >> 1) & 3] += x0 + x1;
        const uint32_t w = pack2<BF>(x0, x1);
        p[2 * u + (i >> 3)][(i & 7) >> 1] = w;
        if constexpr (BF) ls[(i >> 1) & 3] = add_bf2(w, ls[(i >> 1) & 3]);
      }
    l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
  };
  // a tile of which some row sees a part, or whose scores outgrow the maximum. whole: every row sees all of it
  auto edge_tile = [&](int buf, int base, uint32_t pages, bool whole) {
    v16f s[2];
    scores(s, buf);
    // The lane's scores are four runs of 8 adjacent keys, run r at base + 16 r + 8 h (one page group each): what is seen
    // of a run is cut out of its 8 bits by the row's bounds. A score that is not seen becomes -infinity, its weight 0.
    auto first = [](int k) { return (1u << (k < 0 ? 0 : k > 8 ? 8 : k)) - 1u; };   // the run's first k keys
    uint32_t vis = 0;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int at = base + 16 * r + 8 * h, end = pos < limit ? pos + 1 : limit;
      const uint32_t run = first(end - at) & (~first(low + 1 - at) | first(A.sinks - at));
      vis |= (pages >> (2 * r + h) & 1u ? run & 0xffu : 0u) << (8 * r);
    }
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const uint32_t see = (uint32_t)((int)(vis << (31 - 16 * u - i)) >> 31);   // all ones, or none
        s[u][i] = __uint_as_float((__float_as_uint(s[u][i]) & see) | (0xff800000u & ~see));
      }
    if (!__any(vis != 0)) return;
    some = some || vis != 0;
    const float mt = largest(s);
    if (__any(mt > mx + kLag)) {
      const float mn = fmaxf(mx, mt);
      const float f = __builtin_amdgcn_exp2f(mn == mx ? 0.0f : mx - mn);
      l *= f;
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int k = 0; k < 16; k++) o[i][k] *= f;
      mx = mn;
    }
    v4u p[4];
    weights(s, p);
    if (!whole && __any(lane < NW ? odd_flag[buf][lane < NW ? lane : 0] != 0 : false)) {
      // finite values through the products, the others to the rows that see them: they stay what they are under
      // any weight
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int i = 0; i < N; i++) {
          v4u f = v_frag(buf, i, k);
#pragma unroll
          for (int d = 0; d < 4; d++) f[d] = finite16<BF>(f[d]);
          o[i] = mfma32<BF>(f, p[k], o[i]);
        }
      for (int key = 0; key < kKeys; key++) {
        const int j = base + key;
        const bool see = j <= pos && j < limit && (j > low || j < A.sinks) && (pages >> (key >> 3) & 1u);
        const int sw = HD == 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
          for (int a = 0; a < 4; a++) {   // dims 32 i + 8 a + 4 h + c: half of chunk 4 i + a
            const v4s y = *(const lds_v4s *)(lds + buf * 2 * TB + TB + key * RB + ((4 * i + a) ^ sw) * 16 + 8 * h);
#pragma unroll
            for (int c = 0; c < 4; c++) {
              const float v = kv2f<BF>((uint16_t)y[c]);
              o[i][4 * a + c] += see && !(fabsf(v) < __builtin_inff()) ? v : 0.0f;
            }
          }
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int i = 0; i < N; i++) o[i] = mfma32<BF>(v_frag(buf, i, k), p[k], o[i]);
  };
  // the tiles [ta, te_) of the window that every row of the workgroup sees whole, if their pages exist
  const int from = A.win > 0 && pmax >= A.win ? (pmax - A.win) / kKeys + 1 : 0, upto = (pmin + 1 < kv.cap ? pmin + 1 : kv.cap) / kKeys;
  const int ta = from > wt ? from - gap : st, te_ = upto - gap < t1 ? upto - gap : t1;
  // the 8-key groups of a tile whose page exists
  auto pages_of = [&](int x) { return (uint32_t)__ballot((unsigned)x < (unsigned)kv.npages) & 0xffu; };
  // every wave has its pieces of tile t and has left tile t - 1: t + 1 may be loaded into that one's buffer
  auto take_up = [&](int t, int buf) {
    __syncthreads();
    if (t + 1 < t1) load(t + 1, buf ^ 1, ids_next);
    ids = ids_next;
    ids_next = page_ids(t + 2);
  };
  int t = t0;
  bool taken = false;   // tile t is taken up
  while (t < t1) {
    const int buf = (t - t0) & 1, base = tile_base(t);
    uint32_t pages = 0xffu;
    if (!taken) {
      pages = pages_of(ids);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's pieces of the tile are in LDS
      // a value that not every row sees must not meet a zero weight where it is not finite
      bool odd = false;
#pragma unroll
      for (int x = 0; x < LI; x++) {
        const v4u v = *(const lds_v4u *)(lds + buf * 2 * TB + TB + (w + x * NW) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; i++) odd = odd || odd16<BF>(v[i]);
      }
      const bool any = __any(odd);
      if (lane == 0) odd_flag[buf][w] = any ? 1u : 0u;
      take_up(t, buf);
    }
    if (!idle && base <= wmax && (A.win == 0 || base + kKeys > wmin + 1 - A.win || base < A.sinks))
      edge_tile(buf, base, pages, taken);
    taken = false;
    t++;
    // the run of inner tiles, most of a long prompt's: a wave leaves it where its sums have to be rescaled
    while (t >= ta && t < te_ && pages_of(ids) == 0xffu) {
      const int buf = (t - t0) & 1;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      take_up(t, buf);
      v16f s[2];
      scores(s, buf);
      const float mt = largest(s);
      if (__any(mt > mx + kLag)) {
        taken = true;
        break;
      }
      some = true;
      v4u p[4];
      weights(s, p);
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = mfma32<BF>(v_frag(buf, i, k), p[k], o[i]);
      t++;
    }
  }
  l = add_half_pair(l);
  const int other = __shfl_xor((int)some, 32, 64);   // the half that holds the row's other keys
  some = some || other != 0;
  if (r >= rows) return;
  if (A.nsplit > 1) {   // a part: o, m, l (l < 0: no key)
    const size_t pj = ((size_t)row * A.nh + head) * A.nsplit + blockIdx.y;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int a = 0; a < 4; a++)
        *reinterpret_cast<float4 *>(A.po + pj * HD + 32 * i + 8 * a + 4 * h) =
            make_float4(o[i][4 * a], o[i][4 * a + 1], o[i][4 * a + 2], o[i][4 * a + 3]);
    if (h == 0) *reinterpret_cast<float2 *>(A.pml + 2 * pj) = make_float2(mx, some ? l : -1.0f);
    return;
  }
  float f = 1.0f / l;
  if (A.gate != nullptr) f = f / (1.0f + expf_pq(-bf2f(A.gate[(size_t)row * A.gate_stride + head])));
#pragma unroll
  for (int i = 0; i < N; i++) {
    uint16_t y[16];
#pragma unroll
    for (int k = 0; k < 16; k++) y[k] = some ? f2bf(o[i][k] * f) : 0;
    if (A.out != nullptr) {
      uint16_t *dst = A.out + (size_t)row * A.out_stride + head * HD + 32 * i + 4 * h;
#pragma unroll
      for (int a = 0; a < 4; a++) {
        if (A.ovec) {
          *reinterpret_cast<uint2 *>(dst + 8 * a) =
              make_uint2(y[4 * a] | (uint32_t)y[4 * a + 1] << 16, y[4 * a + 2] | (uint32_t)y[4 * a + 3] << 16);
        } else {
#pragma unroll
          for (int c = 0; c < 4; c++) dst[8 * a + c] = y[4 * a + c];
        }
      }
    }
    if (A.qx != nullptr) {   // a Q8_0 block is the 32 dims of the two halves
      float am = 0.0f;
#pragma unroll
      for (int k = 0; k < 16; k++) am = fmaxf(am, fabsf(bf2f(y[k])));
      am = max_half_pair(am);
      const float d = am / 127.0f;
      const Q8Div dv(d);
      const size_t at = ((size_t)row * A.nh + head) * HD + 32 * i;
#pragma unroll
      for (int a = 0; a < 4; a++) {
        uint32_t x = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) x |= (uint32_t)(uint8_t)(int8_t)q8_code(dv.div(bf2f(y[4 * a + c]))) << (8 * c);
        __builtin_memcpy(A.qx + at + 8 * a + 4 * h, &x, 4);
      }
      if (h == 0) A.dx[at / 32] = d;
    }
  }
}

// The parts of each (row, head): HD / 4 threads each, in order of the splits, their
// loads 8 at a time ahead of the sums (512 queries of 16 heads in 8 parts, 34 MB: 9.5 -> 7.8 us,
// 203 queries 18.5 -> 18.0 a call).
template <int HD>
__global__ __launch_bounds__(256) void paged_prefill_join_kernel(PrefillArgs A, PagedView kv) {
  constexpr int TH = HD / 4;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  const int d0 = 4 * (int)(e % TH);
  const long long rh = e / TH;
  const int row = (int)(rh / A.nh), head = (int)(rh % A.nh);
  // whether a sequence has the row, for each of the wave's rows (two or four heads): others have no parts
  bool mine = false;
  for (uint64_t todo = __ballot(row < A.T); todo != 0;) {
    const int r = __builtin_amdgcn_readlane(row, __builtin_ctzll(todo));
    int left;
    const bool has = paged_seq_of_row(kv, r, left) >= 0;
    mine = row == r ? has : mine;
    todo &= ~__ballot(row == r);
  }
  if (!mine) return;
  const size_t p0 = (size_t)rh * A.nsplit;
  const float2 *ml = reinterpret_cast<const float2 *>(A.pml) + p0;
  float M = -__builtin_inff(), L = 0.0f, a[4] = {0, 0, 0, 0};
  bool any = false;
  constexpr int U = 8;   // parts on their way at once
  for (int i0 = 0; i0 < A.nsplit; i0 += U) {
    float2 p[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u < A.nsplit ? i0 + u : i0;
      p[u] = ml[i];
      v[u] = *reinterpret_cast<const float4 *>(A.po + (p0 + i) * HD + d0);
    }
    float mn = M;
#pragma unroll
    for (int u = 0; u < U; u++) mn = fmaxf(mn, p[u].x);
    const float Mz = mn == -__builtin_inff() ? 0.0f : mn, k = M == mn ? 1.0f : __builtin_amdgcn_exp2f(M - Mz);
    M = mn;
    L *= k;
#pragma unroll
    for (int c = 0; c < 4; c++) a[c] *= k;
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (i0 + u >= A.nsplit || p[u].y < 0.0f) continue;
      any = true;
      const float f = __builtin_amdgcn_exp2f(p[u].x - Mz);
      L = __builtin_fmaf(p[u].y, f, L);
      a[0] = __builtin_fmaf(v[u].x, f, a[0]);
      a[1] = __builtin_fmaf(v[u].y, f, a[1]);
      a[2] = __builtin_fmaf(v[u].z, f, a[2]);
      a[3] = __builtin_fmaf(v[u].w, f, a[3]);
    }
  }
  paged_store4<HD>(a, L, any, row, head, d0, A.nh, A.gate, A.gate_stride, A.out, A.out_stride, A.qx, A.dx);
}

// The row tile's waves and the splits of the keys: tiles of 256 rows where they
// fill the chip and see 1024 keys or more (head_dim 128: K and V are then read half as often), else
// of 128; and splits until one workgroup of 256 rows, or two of 128, a CU have
// work, each of at least 2 tiles of keys. Measured, 256 / 128 rows (us): 16384 queries of 16 q
// and 4 kv heads of 128 1070 / 1133 (fp16 1124 / 1180), 16 sequences of 4096 1251 / 1270, 32 of
// 2048 727 / 729, 2048 behind 14336 in 8 sequences 2033 / 2121, 16384 in a window of 256
// 112 / 94; head_dim 64, 32 and 8 heads, 8192 queries 448 / 424 (when it had both); 203 queries
// behind 300 unsplit 25.4 / 21.3, in 3 splits of 128 rows 17.7; 512 behind 32000 unsplit
// 856 / 725, in 8 splits of 128 rows 182. Row tiles are counted as if sequences shared them.
struct PrefillPlan {
  int nw, slots, nsplit;
};
static PrefillPlan prefill_plan(int nseq, int T, int nh, int nkv, int hd, int max_kv, int win, int sinks) {
  PrefillPlan p;
  const long long rows = (long long)T * (nh / nkv);
  p.nw = hd == 128 && (rows + 255) / 256 * nkv >= 256 && (win == 0 || win + (long long)sinks >= 1024) && max_kv >= 1024 ? 8 : 4;
  const int BM = 32 * p.nw;
  p.slots = (int)(rows / BM) + nseq;
  const long long groups = (rows + BM - 1) / BM * nkv, fill = 256 * (8 / p.nw) / groups;
  const long long seen = win > 0 && (long long)win + sinks + BM < max_kv ? (long long)win + sinks + BM : max_kv;
  const long long most = (seen + kKeys - 1) / (2 * kKeys);
  p.nsplit = (int)(fill < most ? fill : most);
  if (p.nsplit < 1) p.nsplit = 1;
  return p;
}
static size_t prefill_ws(const PrefillPlan &p, int T, int nh, int hd) {
  return p.nsplit == 1 ? 0 : (size_t)T * nh * p.nsplit * (hd + 2) * sizeof(float);
}

}  // namespace pq

using namespace pq;

extern "C" size_t pq_paged_prefill_workspace_bytes(int nseq, int T, int nh, int nkv, int hd, int max_kv, int win,
                                                   int sinks) {
  if (nseq <= 0 || T <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || (hd != 64 && hd != 128) || max_kv <= 0 || win < 0 || sinks < 0)
    return 0;
  return prefill_ws(prefill_plan(nseq, T, nh, nkv, hd, max_kv, win, sinks), T, nh, hd);
}

template <int HD, bool BF, int NW>
static void prefill_launch(const PrefillArgs &A, const PagedView &v, const PrefillPlan &p, hipStream_t st) {
  launch(paged_prefill_kernel<HD, BF, NW>, dim3((unsigned)p.slots * v.nkv, p.nsplit), dim3(64 * NW), 0, st, A, v, p.slots);
}

extern "C" int pq_paged_attn_prefill(const uint16_t *q, int q_stride, const pq_paged_kv *kv, const uint16_t *gate,
                                     int gate_stride, uint16_t *out, int out_stride, int8_t *qx, float *dx, int nh,
                                     int T, float scale, int win, int sinks, int max_kv, void *ws, size_t ws_bytes,
                                     void *stream) {
  const char *who = "pq_paged_attn_prefill";
  PagedView v;
  const int rc = paged_attn_check(who, q, q_stride, kv, gate, gate_stride, out, out_stride, qx, dx, nh, win, sinks, max_kv, &v);
  if (rc) return rc;
  PQ_REQUIRE(T > 0 && T <= 1 << 23 && (v.q_start || T == kv->nseq), PQ_ERR_ARG, "%s: %d rows for %d sequences%s", who, T,
             kv->nseq, v.q_start ? "" : " without q_start");
  const int hd = kv->hd;
  const PrefillPlan p = prefill_plan(v.nseq, T, nh, v.nkv, hd, max_kv, win, sinks);
  const size_t need = prefill_ws(p, T, nh, hd);
  PQ_REQUIRE((long long)p.slots * v.nkv <= 1 << 22, PQ_ERR_ARG, "%s: %d rows of %d heads are too many for one call", who, T, nh);
  PQ_REQUIRE(need == 0 || (ws && ws_bytes >= need), PQ_ERR_WORKSPACE, "%s: workspace of %zu bytes needed (got %zu)", who,
             need, ws ? ws_bytes : 0);
  PQ_REQUIRE(need == 0 || aligned(ws, 16), PQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", who);
  PrefillArgs A;
  A.q = q, A.gate = gate, A.out = out, A.qx = qx, A.dx = dx;
  A.po = reinterpret_cast<float *>(ws), A.pml = need ? A.po + (size_t)T * nh * p.nsplit * hd : nullptr;
  A.q_stride = q_stride, A.gate_stride = gate_stride, A.out_stride = out_stride;
  A.nh = nh, A.G = nh / v.nkv, A.T = T, A.win = win, A.sinks = sinks, A.nsplit = p.nsplit, A.scale = scale;
  A.qvec = aligned(q, 16) && q_stride % 8 == 0 ? 1 : 0;
  A.ovec = aligned(out, 8) && out_stride % 4 == 0 ? 1 : 0;
  hipStream_t st = as_stream(stream);
#define PQ_PRE(BB)                                             \
  do {                                                         \
    if (hd == 64) prefill_launch<64, BB, 4>(A, v, p, st);      \
    else if (p.nw == 4) prefill_launch<128, BB, 4>(A, v, p, st); \
    else prefill_launch<128, BB, 8>(A, v, p, st);              \
  } while (0)
  if (kv->dtype == PQ_DTYPE_BF16) PQ_PRE(true);
  else PQ_PRE(false);
#undef PQ_PRE
  const int rl = check_launch(who);
  if (rl || p.nsplit == 1) return rl;
  const dim3 grid((unsigned)(((long long)T * nh * (hd / 4) + 255) / 256));
  if (hd == 64) launch(paged_prefill_join_kernel<64>, grid, dim3(256), 0, st, A, v);
  else launch(paged_prefill_join_kernel<128>, grid, dim3(256), 0, st, A, v);
  return check_launch(who);
}
