// paged_decode.hip -- attention of one new token a sequence over a paged cache
// (gfx950): the keys split over workgroups, the parts joined in order.
//
// A row at position p = kv_len - 1 sees the sinks [0, ns), ns = min(sinks, lo),
// and its window [lo, p], lo = max(0, p + 1 - win). s_j = scale q.k_j; the
// softmax is online: running maximum m, l = sum 2^(s'_j - m), o = sum 2^(s'_j - m) v_j
// with s' = s log2(e), all fp32; parts (m, l, o) join by 2^(m - M).
//
// What bounds it is reading K and V once: 4 nkv hd bytes a key against 4 nh hd
// flop. So a wave takes a tile of 32 keys of one kv head, all G = nh / nkv heads
// of its group against it, straight from memory into the matrix cores'
// registers, with no LDS and no shuffle in between:
//   scores  S^T [key][head] = K q^T, two 16x16x32 tiles: lane (c, Q) = (lane & 15,
//           lane >> 4) loads key 8 (c / 4) + c % 4 + 4u of tile u, dims 32 s + 8 Q ..
//           + 7, and gets the scores of head c at keys 8 Q + r + 4 u, r < 4;
//   values  O^T [dim][head] = V^T P^T: those are the 8 keys 8 Q + j that the lane
//           holds as a column of P^T. It loads V of the same 8 keys, dims HD/16 c ..
//           (a row is read whole by 16 lanes); the 8 x HD/16 block transposed in
//           registers (v_perm) is the operand of HD/16 products, whose row c is
//           dim HD/16 c + n: lane (c, Q) ends with HD/4 adjacent dims of head c.
// Heads past G are zero columns: the matrix cores have 25 times the work's rate.
#include <type_traits>

#include "paged.h"

namespace pq {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;     // keys of a wave's step
constexpr int kWaves = 4;     // waves a workgroup

// The tiles of a sequence of n positions: those of the sinks, then those of the window.
struct PagedTiles {
  int n, lo, ns, sink, first, count;
};
__host__ __device__ inline PagedTiles paged_tiles(int n, int cap, int win, int sinks) {
  PagedTiles t;
  t.lo = win > 0 && n > win ? n - win : 0;
  t.ns = sinks < t.lo ? sinks : t.lo;
  t.n = n < cap ? n : cap;
  t.sink = (t.ns + kTile - 1) / kTile;
  t.first = t.lo / kTile > t.sink ? t.lo / kTile : t.sink;
  const int end = (int)(((long long)t.n + kTile - 1) / kTile);
  if (t.sink > end) t.sink = end > 0 ? end : 0;
  t.count = t.sink + (end > t.first ? end - t.first : 0);
  return t;
}
__device__ __forceinline__ int paged_tile_base(const PagedTiles &t, int i) {
  return (i < t.sink ? i : i - t.sink + t.first) * kTile;
}
// tiles a split takes: the host's share, or more where the sequence is longer than it knew
__host__ __device__ inline int paged_split_tiles(int count, int nsplit, int share) {
  const int even = (count + nsplit - 1) / nsplit;
  return even > share ? even : share;
}

template <bool BF>
__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  typedef __bf16 v8b __attribute__((ext_vector_type(8)));
  typedef _Float16 v8h __attribute__((ext_vector_type(8)));
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t f2h2(float a, float b) { return (uint32_t)f2h(a) | (uint32_t)f2h(b) << 16; }

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

// Grid (kv heads x splits, sequences). A part is HD floats and the pair (m, l) of
// each (sequence, head, split); l < 0: no key. One split: the output itself.
template <int HD, bool BF>
__global__ __launch_bounds__(64 * kWaves) void paged_split_kernel(
    const uint16_t *__restrict__ q, int q_stride, int qvec, PagedView kv, const uint16_t *__restrict__ gate,
    int gate_stride, uint16_t *__restrict__ out, int out_stride, int8_t *__restrict__ qx, float *__restrict__ dx, int nh,
    int G, float scale, int win, int sinks, int nsplit, int share, float *__restrict__ po, float *__restrict__ pml) {
  constexpr int S = HD / 32, N = HD / 16, VW = HD / 32;   // score steps, value products, dwords of V a key and lane
  extern __shared__ __align__(16) float lds[];            // [waves][G][HD + 4]: o, then m, l
  const int g = blockIdx.x % kv.nkv, split = blockIdx.x / kv.nkv, b = blockIdx.y;
  const int lane = threadIdx.x & 63, c = lane & 15, Q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvd = kv.nkv * HD;
  const PagedTiles t = paged_tiles(kv.kv_len[b], kv.cap, win, sinks);
  const int per = paged_split_tiles(t.count, nsplit, share);
  const int t0 = split * per, t1 = t0 + per < t.count ? t0 + per : t.count;
  if (t0 >= t.count && split > 0) return;
  const bool alone = per >= t.count;   // the sequence's only split
  // q: the operand's column c, dims 32 s + 8 Q ..; an fp16 cache meets fp16 queries, scaled by the power of two that
  // brings the row's largest value into [1, 2): exact but for what lies 2^-25 below it
  v4u qf[S];
  float sc = scale * 1.44269504088896341f;
  {
    const uint16_t *qr = q + (size_t)b * q_stride + (size_t)(g * G + (c < G ? c : 0)) * HD + 8 * Q;
    float amax = 0.0f;
#pragma unroll
    for (int s = 0; s < S; s++) {
      v4u v;
      if (qvec) {
        v = *reinterpret_cast<const v4u *>(qr + 32 * s);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = qr[32 * s + 2 * i] | (uint32_t)qr[32 * s + 2 * i + 1] << 16;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (c >= G) v[i] = 0;
        amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(v[i] << 16)), fabsf(__uint_as_float(v[i] & 0xffff0000u))));
      }
      qf[s] = v;
    }
    if constexpr (!BF) {
      amax = max_half_pair(max_row_pair(amax));
      const int e = amax > 0.0f && amax < __builtin_inff() ? (int)__builtin_amdgcn_frexp_expf(amax) - 1 : 0;
      sc = __builtin_amdgcn_ldexpf(sc, e);
#pragma unroll
      for (int s = 0; s < S; s++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          qf[s][i] = f2h2(__builtin_amdgcn_ldexpf(__uint_as_float(qf[s][i] << 16), -e),
                          __builtin_amdgcn_ldexpf(__uint_as_float(qf[s][i] & 0xffff0000u), -e));
    }
  }
  // fp16 weights are held as 2^14 of theirs: what is lost below fp16's range is then 2^-39 of the largest
  constexpr float kLift = BF ? 0.0f : 14.0f;
  float m = -__builtin_inff(), l = 0.0f;
  bool some = false;
  v4f o[N];
#pragma unroll
  for (int n = 0; n < N; n++) o[n] = v4f{0, 0, 0, 0};
  const int32_t *tb = kv.table + (size_t)b * kv.table_stride;
  const int slots = (1 << kv.lg_page) - 1;
  // the page of 8 keys from j: a lane's K keys lie in group c / 4 of the tile, its V keys in group Q
  auto page_of = [&](int j) { return j < t.n ? tb[j >> kv.lg_page] : -1; };
  auto walk = [&](auto two) {
    int idk = -1, idv = -1;
    if (t0 + w < t1) {
      const int base = paged_tile_base(t, t0 + w);
      idk = page_of(base + 8 * (c >> 2));
      idv = page_of(base + 8 * Q);
    }
    for (int i = t0 + w; i < t1; i += kWaves) {
      const int base = paged_tile_base(t, i);
      const int jk = base + 8 * (c >> 2), jv = base + 8 * Q;
      const bool okk = (unsigned)idk < (unsigned)kv.npages, okv = (unsigned)idv < (unsigned)kv.npages;
      const uint16_t *kr = kv.k + (okk ? idk : 0) * kv.page_stride + (long long)((jk & slots) + (c & 3)) * kvd + g * HD + 8 * Q;
      const uint16_t *vr = kv.v + (okv ? idv : 0) * kv.page_stride + (long long)(jv & slots) * kvd + g * HD + (HD / 16) * c;
      v4u kw[2][S];
      uint32_t vw[8][VW];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int s = 0; s < S; s++) kw[u][s] = *reinterpret_cast<const v4u *>(kr + 4 * u * kvd + 32 * s);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if constexpr (VW == 4) {
          const v4u x = *reinterpret_cast<const v4u *>(vr + (size_t)j * kvd);
          vw[j][0] = x[0], vw[j][1] = x[1], vw[j][2] = x[2], vw[j][3] = x[3];
        } else {
          const v2u x = *reinterpret_cast<const v2u *>(vr + (size_t)j * kvd);
          vw[j][0] = x[0], vw[j][1] = x[1];
        }
      }
      if (i + kWaves < t1) {
        const int nb = paged_tile_base(t, i + kWaves);
        idk = page_of(nb + 8 * (c >> 2));
        idv = page_of(nb + 8 * Q);
      }
      v4f s[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        s[u] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < S; k++) s[u] = mfma16<BF>(kw[u][k], qf[k], s[u]);
      }
      // a tile that is not seen whole: hide its other keys, and what their V holds
      const bool whole = base + kTile <= t.n && (base >= t.lo || base + kTile <= t.ns) && __all(okv);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = s[j >> 2][j & 3] * sc;
      if (!whole) {
        bool mine = false;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int key = jv + j;
          const bool see = okv && key < t.n && (key >= t.lo || key < t.ns);
          mine = mine || see;
          if (!see) {
            x[j] = -__builtin_inff();
#pragma unroll
            for (int d = 0; d < VW; d++) vw[j][d] = 0;
          }
        }
        if (!__any(mine)) continue;
      }
      some = true;
      float mt = x[0];
#pragma unroll
      for (int j = 1; j < 8; j++) mt = fmaxf(mt, x[j]);
      mt = max_half_pair(max_row_pair(mt));
      const float mn = fmaxf(m, mt);
      if (__any(mn != m)) {
        // no finite score so far: the weights are 2^-inf whatever is taken off
        const float f = __builtin_amdgcn_exp2f(mn == m ? 0.0f : m - mn);
        l *= f;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
          for (int r = 0; r < 4; r++) o[n][r] *= f;
        m = mn;
      }
      const float off = (m == -__builtin_inff() ? 0.0f : m) - kLift;
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = __builtin_amdgcn_exp2f(x[j] - off);
      l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      v4u ph, pl;
#pragma unroll
      for (int d = 0; d < 4; d++) {
        float a = x[2 * d], e = x[2 * d + 1];
        if constexpr (BF) {
          ph[d] = bfr2(a, e);
          pl[d] = f2bf2(x[2 * d] - a, x[2 * d + 1] - e);
        } else {
          ph[d] = f2h2(a, e);
        }
      }
#pragma unroll
      for (int n = 0; n < N; n++) {
        v4u a;
#pragma unroll
        for (int d = 0; d < 4; d++)
          a[d] = __builtin_amdgcn_perm(vw[2 * d + 1][n >> 1], vw[2 * d][n >> 1], n & 1 ? 0x07060302u : 0x05040100u);
        o[n] = mfma16<BF>(a, ph, o[n]);
        if constexpr (two.value) o[n] = mfma16<BF>(a, pl, o[n]);
      }
    }
  };
  // A bf16 weight goes in as the sum of two bf16 (16 bits of it in all): the second product costs nothing beside the
  // reads. Its factor may be 0 or negative, so an infinite value that the row sees would come out as NaN: a wave that
  // ends with a sum that is not finite walks its keys again with the rounded weight alone.
  walk(std::integral_constant<bool, BF>{});
  if constexpr (BF) {
    bool odd = false;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int r = 0; r < 4; r++) odd = odd || !(fabsf(o[n][r]) < __builtin_inff());
    if (__any(odd)) {
      m = -__builtin_inff();
      l = 0.0f;
#pragma unroll
      for (int n = 0; n < N; n++) o[n] = v4f{0, 0, 0, 0};
      walk(std::false_type{});
    }
  }
  l = add_half_pair(add_row_pair(l));
  // the waves' states, then each thread four dims of a head over them
  constexpr int LD = HD + 4;
  if (c < G) {
    float *dst = lds + (w * G + c) * LD;
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int n = 0; n < N; n += 4)
        *reinterpret_cast<float4 *>(dst + (HD / 16) * (4 * Q + r) + n) = make_float4(o[n][r], o[n + 1][r], o[n + 2][r], o[n + 3][r]);
    if (Q == 0) {
      dst[HD] = m;
      dst[HD + 1] = some ? l : -1.0f;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G * (HD / 4); e += 64 * kWaves) {
    const int h = e / (HD / 4), d0 = 4 * (e % (HD / 4));
    float M = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < kWaves; k++) M = fmaxf(M, lds[(k * G + h) * LD + HD]);
    const float Mz = M == -__builtin_inff() ? 0.0f : M;
    float L = 0.0f, a[4] = {0, 0, 0, 0};
    bool any = false;
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      const float *src = lds + (k * G + h) * LD;
      if (src[HD + 1] < 0.0f) continue;
      any = true;
      const float f = __builtin_amdgcn_exp2f(src[HD] - Mz);
      L = __builtin_fmaf(src[HD + 1], f, L);
      const float4 v = *reinterpret_cast<const float4 *>(src + d0);
      a[0] = __builtin_fmaf(v.x, f, a[0]);
      a[1] = __builtin_fmaf(v.y, f, a[1]);
      a[2] = __builtin_fmaf(v.z, f, a[2]);
      a[3] = __builtin_fmaf(v.w, f, a[3]);
    }
    if (alone) {
      paged_store4<HD>(a, L, any, b, g * G + h, d0, nh, gate, gate_stride, out, out_stride, qx, dx);
    } else {
      const size_t pj = ((size_t)b * nh + g * G + h) * nsplit + split;
      *reinterpret_cast<float4 *>(po + pj * HD + d0) = make_float4(a[0], a[1], a[2], a[3]);
      if (d0 == 0) *reinterpret_cast<float2 *>(pml + 2 * pj) = make_float2(M, any ? L : -1.0f);
    }
  }
}

// The parts of one (head, sequence): HD / 4 threads a split, 256 threads over
// the splits in turn, their sums joined in LDS in a fixed order.
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedView kv, const uint16_t *__restrict__ gate, int gate_stride,
                                                         uint16_t *__restrict__ out, int out_stride,
                                                         int8_t *__restrict__ qx, float *__restrict__ dx, int nh, int win,
                                                         int sinks, int nsplit, int share, const float *__restrict__ po,
                                                         const float *__restrict__ pml) {
  constexpr int TH = HD / 4, R = 256 / TH;   // threads a split, splits a turn
  __shared__ __align__(16) float so[R][HD + 4];
  __shared__ float sm[4];
  const int h = blockIdx.x, b = blockIdx.y, r = threadIdx.x / TH, d0 = 4 * (threadIdx.x % TH);
  const PagedTiles t = paged_tiles(kv.kv_len[b], kv.cap, win, sinks);
  const int per = paged_split_tiles(t.count, nsplit, share);
  if (per >= t.count) return;   // its only split has written the output
  const int ns = (t.count + per - 1) / per;
  const size_t p0 = ((size_t)b * nh + h) * nsplit;
  const float2 *ml = reinterpret_cast<const float2 *>(pml) + p0;
  float M = -__builtin_inff();
  for (int i = threadIdx.x; i < ns; i += 256) M = fmaxf(M, ml[i].x);
  M = wave_max(M);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  if (M == -__builtin_inff()) M = 0.0f;
  float L = 0.0f, a[4] = {0, 0, 0, 0};
  bool any = false;
  for (int i = r; i < ns; i += R) {
    const float2 p = ml[i];
    const float4 v = *reinterpret_cast<const float4 *>(po + (p0 + i) * HD + d0);
    if (p.y < 0.0f) continue;
    any = true;
    const float f = __builtin_amdgcn_exp2f(p.x - M);
    L = __builtin_fmaf(p.y, f, L);
    a[0] = __builtin_fmaf(v.x, f, a[0]);
    a[1] = __builtin_fmaf(v.y, f, a[1]);
    a[2] = __builtin_fmaf(v.z, f, a[2]);
    a[3] = __builtin_fmaf(v.w, f, a[3]);
  }
  *reinterpret_cast<float4 *>(&so[r][d0]) = make_float4(a[0], a[1], a[2], a[3]);
  if (d0 == 0) {
    so[r][HD] = L;
    so[r][HD + 1] = any ? 1.0f : 0.0f;
  }
  __syncthreads();
  if (r != 0) return;
#pragma unroll
  for (int k = 1; k < R; k++) {
    const float4 v = *reinterpret_cast<const float4 *>(&so[k][d0]);
    a[0] += v.x, a[1] += v.y, a[2] += v.z, a[3] += v.w;
    L += so[k][HD];
    any = any || so[k][HD + 1] != 0.0f;
  }
  paged_store4<HD>(a, L, any, b, h, d0, nh, gate, gate_stride, out, out_stride, qx, dx);
}

// How a call is split: nsplit parts a (sequence, kv head), of at least `share` tiles.
struct PagedPlan {
  int nsplit, share;
};
static PagedPlan paged_plan(int nseq, int nkv, int max_kv, int win, int sinks) {
  const int tiles = paged_tiles(max_kv, 0x7fffffff, win, sinks).count;
  const long long want = (1024 + (long long)nseq * nkv - 1) / ((long long)nseq * nkv);
  const long long most = (tiles + 2 * kWaves - 1) / (2 * kWaves);
  PagedPlan p;
  p.nsplit = (int)(want < most ? want : most);
  if (p.nsplit < 1) p.nsplit = 1;
  p.share = (tiles + p.nsplit - 1) / p.nsplit;
  return p;
}

}  // namespace pq

using namespace pq;

extern "C" size_t pq_paged_decode_workspace_bytes(int nseq, int nh, int nkv, int hd, int max_kv, int win, int sinks) {
  if (nseq <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || (hd != 64 && hd != 128) || max_kv <= 0 || win < 0 || sinks < 0) return 0;
  const PagedPlan p = paged_plan(nseq, nkv, max_kv, win, sinks);
  return p.nsplit == 1 ? 0 : (size_t)nseq * nh * p.nsplit * (hd + 2) * sizeof(float);
}

extern "C" int pq_paged_attn_decode(const uint16_t *q, int q_stride, const pq_paged_kv *kv, const uint16_t *gate,
                                    int gate_stride, uint16_t *out, int out_stride, int8_t *qx, float *dx, int nh,
                                    float scale, int win, int sinks, int max_kv, void *ws, size_t ws_bytes,
                                    void *stream) {
  const char *who = "pq_paged_attn_decode";
  PagedView v;
  const int rc = paged_attn_check(who, q, q_stride, kv, gate, gate_stride, out, out_stride, qx, dx, nh, win, sinks, max_kv, &v);
  if (rc) return rc;
  v.q_start = nullptr;
  const int G = nh / v.nkv, hd = kv->hd;
  const PagedPlan p = paged_plan(v.nseq, v.nkv, max_kv, win, sinks);
  const size_t need = pq_paged_decode_workspace_bytes(v.nseq, nh, v.nkv, hd, max_kv, win, sinks);
  PQ_REQUIRE(need == 0 || (ws && ws_bytes >= need), PQ_ERR_WORKSPACE, "%s: workspace of %zu bytes needed (got %zu)", who,
             need, ws ? ws_bytes : 0);
  PQ_REQUIRE(need == 0 || aligned(ws, 16), PQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", who);
  float *po = reinterpret_cast<float *>(ws), *pml = need ? po + (size_t)v.nseq * nh * p.nsplit * hd : nullptr;
  const int qvec = aligned(q, 16) && q_stride % 8 == 0 ? 1 : 0;
  hipStream_t st = as_stream(stream);
  const dim3 grid((unsigned)(v.nkv * p.nsplit), v.nseq);
  const size_t lds = (size_t)kWaves * G * (hd + 4) * sizeof(float);
#define PQ_SPLIT(HH, BB)                                                                                               \
  launch(paged_split_kernel<HH, BB>, grid, dim3(64 * kWaves), lds, st, q, q_stride, qvec, v, gate, gate_stride, out,    \
         out_stride, qx, dx, nh, G, scale, win, sinks, p.nsplit, p.share, po, pml)
  const bool bf = kv->dtype == PQ_DTYPE_BF16;
  if (hd == 64) {
    if (bf) PQ_SPLIT(64, true);
    else PQ_SPLIT(64, false);
  } else {
    if (bf) PQ_SPLIT(128, true);
    else PQ_SPLIT(128, false);
  }
#undef PQ_SPLIT
  const int rl = check_launch(who);
  if (rl || p.nsplit == 1) return rl;
  if (hd == 64)
    launch(paged_join_kernel<64>, dim3(nh, v.nseq), dim3(256), 0, st, v, gate, gate_stride, out, out_stride, qx, dx, nh, win,
           sinks, p.nsplit, p.share, (const float *)po, (const float *)pml);
  else
    launch(paged_join_kernel<128>, dim3(nh, v.nseq), dim3(256), 0, st, v, gate, gate_stride, out, out_stride, qx, dx, nh, win,
           sinks, p.nsplit, p.share, (const float *)po, (const float *)pml);
  return check_launch(who);
}
