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
// Each tile's loads run a tile ahead of its use in the same registers.
//
// Measured: 131072 keys of 4 kv heads of 128, one sequence 56 us (268 MB, 4.8 TB/s with
// the join's 7 us), 64 sequences of up to 8192 keys of 8 heads of 64 102 us (563 MB, 5.5),
// 256 windows of 260 keys of 4 heads of 128 34 us (137 MB, 4.1), 300 keys 9.6 us, the
// call's host time; a plain read of those bytes takes 38, 80 and 20 us.
#include <type_traits>

#include "paged.h"

namespace pq {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;     // keys of a wave's step
constexpr int kWaves = 4;     // waves a workgroup

// The tiles of a sequence of n positions: those of the sinks, then those of the window.
// What the sinks reach is cut to the cap before it is rounded up, so that no length,
// window or sink count wraps (cap <= kPagedCap).
struct PagedTiles {
  int n, lo, ns, sink, first, count;
};
__host__ __device__ inline PagedTiles paged_tiles(int n, int cap, int win, int sinks) {
  PagedTiles t;
  t.n = n < cap ? (n > 0 ? n : 0) : cap;
  t.lo = win > 0 && n > win ? n - win : 0;
  t.ns = sinks < t.lo ? sinks : t.lo;
  if (t.ns > t.n) t.ns = t.n;
  t.sink = (t.ns + kTile - 1) / kTile;
  t.first = t.lo / kTile > t.sink ? t.lo / kTile : t.sink;
  const int end = (t.n + kTile - 1) / kTile;
  t.count = t.sink + (end > t.first ? end - t.first : 0);
  return t;
}
__device__ __forceinline__ int paged_tile_base(const PagedTiles &t, int i) {
  return (i < t.sink ? i : i - t.sink + t.first) * kTile;
}
// tiles of sequence b, at least one: a sequence without keys is a tile that sees nothing
__device__ __forceinline__ int paged_count(const PagedView &kv, int b, int win, int sinks) {
  const int c = paged_tiles(kv.kv_len[b], kv.cap, win, sinks).count;
  return c > 0 ? c : 1;
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

// a piece of K or V; NT: not to be kept in the caches
template <bool NT, typename T>
__device__ __forceinline__ T read_kv(const uint16_t *p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const T *>(p));
  else return *reinterpret_cast<const T *>(p);
}

// A workgroup's 4 waves are HW kv heads (a group) by KW = 4 / HW ways through the
// keys. A segment is a group of one sequence, its work the sequence's tiles.
//
// share == 0: a workgroup a segment, which writes the output. share > 0: the
// segments' tiles lie end to end in order of (sequence, group) and workgroup x
// takes the tiles [x per, (x + 1) per), per = max(total / gridDim + 1, share), so that all
// carry the same work whatever the lengths. A segment that lies whole in one
// workgroup's tiles is output at once; of one cut in pieces, a workgroup holds at
// most two (its first, which began in the workgroup before, and its last): part
// 2 x + (the piece begins the segment). A part is (m, l) and hd floats of each head;
// l < 0: no key. seg[]: where the segments are cut: by_wg, entry x is the segment whose
// first piece is part 2 x + 1 (-1: none) and its last workgroup; else entry
// (sequence, group) is the segment's first and last workgroup.
template <int HD, bool BF, bool NT>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_split_kernel(
    const uint16_t *__restrict__ q, int q_stride, int qvec, PagedView kv, const uint16_t *__restrict__ gate,
    int gate_stride, uint16_t *__restrict__ out, int out_stride, int8_t *__restrict__ qx, float *__restrict__ dx, int nh,
    int G, float scale, int win, int sinks, int HW, int share, int by_wg, float *__restrict__ po,
    float *__restrict__ pml, int2 *__restrict__ seg) {
  constexpr int S = HD / 32, N = HD / 16, VW = HD / 32;   // score steps, value products, dwords of V a key and lane
  extern __shared__ __align__(16) float lds[];            // [waves][G][HD + 4]: o, then m, l
  __shared__ long long scan[64 * kWaves + 1];
  const int ng = kv.nkv / HW, KW = kWaves / HW;
  const int lane = threadIdx.x & 63, c = lane & 15, Q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = wave / HW;
  const int kvd = kv.nkv * HD;
  // the workgroup's tiles [at, end); b, gg, begin: the segment that holds `at`, and where it begins
  int b, gg;
  long long at, end, begin, per = 0;
  if (share == 0) {
    b = blockIdx.x / ng;
    gg = blockIdx.x % ng;
    at = begin = 0;
    end = 1;
  } else {
    // thread i sums the tiles of sequences [i per_t, (i + 1) per_t), then the workgroup's running sums
    const int per_t = (kv.nseq + 64 * kWaves - 1) / (64 * kWaves);
    long long sum = 0;
    for (int i = threadIdx.x * per_t; i < (int)(threadIdx.x + 1) * per_t && i < kv.nseq; i++)
      sum += paged_count(kv, i, win, sinks);
    long long run = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const long long y = __shfl_up(run, d, 64);
      if (lane >= d) run += y;
    }
    if (threadIdx.x == 0) scan[0] = 0;
    scan[threadIdx.x + 1] = run;
    __syncthreads();
    long long pre = 0;
    for (int i = 1; i <= wave; i++) pre += scan[64 * i];
    __syncthreads();
    scan[threadIdx.x + 1] = run + pre;
    __syncthreads();
    const long long total = scan[64 * kWaves] * ng;
    per = (long long)((double)total / gridDim.x) + 1;
    if (per < share) per = share;
    at = per * blockIdx.x;
    end = at + per < total ? at + per : total;
    if (by_wg && threadIdx.x == 0) seg[blockIdx.x].x = -1;
    if (at >= end) return;
    int lo = 0, hi = 64 * kWaves;   // the last i with scan[i] ng <= at
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (scan[mid] * ng <= at) lo = mid;
      else hi = mid;
    }
    begin = scan[lo] * ng;
    b = lo * per_t;
    long long n = paged_count(kv, b, win, sinks);
    while (begin + n * ng <= at) {
      begin += n * ng;
      b++;
      n = paged_count(kv, b, win, sinks);
    }
    gg = (int)((double)(at - begin) / (double)n);   // below 2^52: the quotient's floor is exact
    begin += gg * n;
  }
  while (at < end) {
    const int g0 = gg * HW, g = g0 + wave % HW;
    const PagedTiles t = paged_tiles(kv.kv_len[b], kv.cap, win, sinks);
    const int count = t.count > 0 ? t.count : 1;
    const int t0 = (int)(at - begin);
    const int t1 = share == 0 || end - begin > count ? count : (int)(end - begin);
    const bool alone = t0 == 0 && t1 == count;
    const int32_t *tb = kv.table + (size_t)b * kv.table_stride;
    const int slots = (1 << kv.lg_page) - 1;
    // the page of 8 keys from j: a lane's K keys lie in group c / 4 of the tile, its V keys in group Q
    auto page_of = [&](int j) { return j < t.n ? tb[j >> kv.lg_page] : -1; };
    // the tile's loads run a tile ahead: K's as soon as the scores have read the registers, V's after the value
    // products, the page ids two tiles ahead
    v4u kw[2][S];
    uint32_t vw[8][VW];
    int idk = -1, idv = -1, pgk = -1, pgv = -1;
    auto ids = [&](int i) {
      if (i >= t1) return;
      const int base = paged_tile_base(t, i);
      idk = page_of(base + 8 * (c >> 2));
      idv = page_of(base + 8 * Q);
    };
    auto load_k = [&](int i) {
      const int jk = paged_tile_base(t, i) + 8 * (c >> 2);
      const bool ok = (unsigned)pgk < (unsigned)kv.npages;
      const uint16_t *kr = kv.k + (ok ? pgk : 0) * kv.page_stride + (long long)((jk & slots) + (c & 3)) * kvd + g * HD + 8 * Q;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int s = 0; s < S; s++) kw[u][s] = read_kv<NT, v4u>(kr + 4 * u * kvd + 32 * s);
    };
    auto load_v = [&](int i) {
      const int jv = paged_tile_base(t, i) + 8 * Q;
      const bool ok = (unsigned)pgv < (unsigned)kv.npages;
      const uint16_t *vr = kv.v + (ok ? pgv : 0) * kv.page_stride + (long long)(jv & slots) * kvd + g * HD + (HD / 16) * c;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if constexpr (VW == 4) {
          const v4u x = read_kv<NT, v4u>(vr + (size_t)j * kvd);
          vw[j][0] = x[0], vw[j][1] = x[1], vw[j][2] = x[2], vw[j][3] = x[3];
        } else {
          const v2u x = read_kv<NT, v2u>(vr + (size_t)j * kvd);
          vw[j][0] = x[0], vw[j][1] = x[1];
        }
      }
    };
    auto start = [&]() {
      ids(t0 + w);
      pgk = idk;
      pgv = idv;
      if (t0 + w < t1) {
        load_k(t0 + w);
        load_v(t0 + w);
      }
      ids(t0 + w + KW);
    };
    // q: the operand's column c, dims 32 s + 8 Q ..; its loads and the first tile's are on their way together
    v4u qf[S];
    const uint16_t *qr = q + (size_t)b * q_stride + (size_t)(g * G + (c < G ? c : 0)) * HD + 8 * Q;
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (qvec) {
        qf[s] = *reinterpret_cast<const v4u *>(qr + 32 * s);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) qf[s][i] = qr[32 * s + 2 * i] | (uint32_t)qr[32 * s + 2 * i + 1] << 16;
      }
    }
    start();
    float sc = scale * 1.44269504088896341f;
    if (c >= G) {
#pragma unroll
      for (int s = 0; s < S; s++) qf[s] = v4u{0, 0, 0, 0};
    }
    // an fp16 cache meets fp16 queries, scaled by the power of two that brings the row's largest value into [1, 2):
    // exact but for what lies 2^-25 below it
    if constexpr (!BF) {
      float amax = 0.0f;
#pragma unroll
      for (int s = 0; s < S; s++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(qf[s][i] << 16)), fabsf(__uint_as_float(qf[s][i] & 0xffff0000u))));
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
    sc = paged_finite(sc, scale);
    // fp16 weights are held as 2^14 of theirs: what is lost below fp16's range is then 2^-39 of the largest
    constexpr float kLift = BF ? 0.0f : 14.0f;
    float m = -__builtin_inff(), l = 0.0f;
    bool some = false;
    v4f o[N];
#pragma unroll
    for (int n = 0; n < N; n++) o[n] = v4f{0, 0, 0, 0};
    auto walk = [&](auto two) {
      for (int i = t0 + w; i < t1; i += KW) {
        const int base = paged_tile_base(t, i), jv = base + 8 * Q;
        const bool okv = (unsigned)pgv < (unsigned)kv.npages, more = i + KW < t1;
        v4f s[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          s[u] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < S; k++) s[u] = mfma16<BF>(kw[u][k], qf[k], s[u]);
        }
        pgk = idk;
        pgv = idv;
        if (more) {
          load_k(i + KW);
          ids(i + 2 * KW);
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
          if (!__any(mine)) {
            if (more) load_v(i + KW);
            continue;
          }
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
        if (more) load_v(i + KW);
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
        start();
        walk(std::false_type{});
      }
    }
    l = add_half_pair(add_row_pair(l));
    // the waves' states, then each thread four dims of a head over them
    constexpr int LD = HD + 4;
    if (c < G) {
      float *dst = lds + (wave * G + c) * LD;
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
    for (int e = threadIdx.x; e < HW * G * (HD / 4); e += 64 * kWaves) {
      const int hh = e / (HD / 4), d0 = 4 * (e % (HD / 4));   // head hh of the workgroup's HW G
      const int x = hh / G, h = hh % G;
      float M = -__builtin_inff();
      for (int k = 0; k < KW; k++) M = fmaxf(M, lds[((k * HW + x) * G + h) * LD + HD]);
      const float Mz = M == -__builtin_inff() ? 0.0f : M;
      float L = 0.0f, a[4] = {0, 0, 0, 0};
      bool any = false;
      for (int k = 0; k < KW; k++) {
        const float *src = lds + ((k * HW + x) * G + h) * LD;
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
        paged_store4<HD>(a, L, any, b, g0 * G + hh, d0, nh, gate, gate_stride, out, out_stride, qx, dx);
      } else {
        const size_t pj = ((size_t)blockIdx.x * 2 + (t0 == 0 ? 1 : 0)) * HW * G + hh;
        *reinterpret_cast<float4 *>(po + pj * HD + d0) = make_float4(a[0], a[1], a[2], a[3]);
        if (d0 == 0) *reinterpret_cast<float2 *>(pml + 2 * pj) = make_float2(M, any ? L : -1.0f);
      }
    }
    if (share == 0) return;
    if (t0 == 0 && threadIdx.x == 0) {
      const int last = (int)((double)(begin + count - 1) / (double)per);
      if (!by_wg) seg[(size_t)b * ng + gg] = make_int2(blockIdx.x, last);
      else if (!alone) seg[blockIdx.x] = make_int2((int)((size_t)b * ng + gg), last);
    }
    at = begin + t1;
    begin += count;
    if (++gg == ng) {
      gg = 0;
      b++;
    }
    __syncthreads();   // the states in LDS are read
  }
}

// The parts of a cut segment's heads: TH = HD / 4 threads a part. by_wg (many
// segments, cut in few pieces): a workgroup for each of the split's, its threads over
// the heads, each over the parts in turn. Else (few, cut in many) a workgroup for
// each (head, sequence), its threads over the parts, their sums joined in LDS in a
// fixed order.
template <int HD>
__global__ __launch_bounds__(256) void paged_join_few_kernel(const uint16_t *__restrict__ gate, int gate_stride,
                                                             uint16_t *__restrict__ out, int out_stride,
                                                             int8_t *__restrict__ qx, float *__restrict__ dx, int nh,
                                                             int G, int HW, const float *__restrict__ po,
                                                             const float *__restrict__ pml, const int2 *__restrict__ seg) {
  constexpr int TH = HD / 4;
  const int rows = HW * G, ng = nh / rows;
  const int2 x = seg[blockIdx.x];
  if (x.x < 0) return;
  const int b = x.x / ng, h0 = x.x % ng * rows, ns = x.y - (int)blockIdx.x + 1;
  const float2 *ml = reinterpret_cast<const float2 *>(pml);
  for (int e = threadIdx.x; e < rows * TH; e += 256) {
    const int h = e / TH, d0 = 4 * (e % TH);
    float M = -__builtin_inff(), L = 0.0f, a[4] = {0, 0, 0, 0};
    bool any = false;
    constexpr int U = 4;   // parts on their way at once
    for (int i0 = 0; i0 < ns; i0 += U) {
      float2 p[U];
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + u < ns ? i0 + u : i0;
        const size_t pj = ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * rows + h;
        p[u] = ml[pj];
        v[u] = *reinterpret_cast<const float4 *>(po + pj * HD + d0);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i0 + u >= ns || p[u].y < 0.0f) continue;
        any = true;
        const float mn = fmaxf(M, p[u].x), Mz = mn == -__builtin_inff() ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(p[u].x - Mz), k = M == mn ? 1.0f : __builtin_amdgcn_exp2f(M - Mz);
        L = __builtin_fmaf(p[u].y, f, L * k);
        a[0] = __builtin_fmaf(v[u].x, f, a[0] * k);
        a[1] = __builtin_fmaf(v[u].y, f, a[1] * k);
        a[2] = __builtin_fmaf(v[u].z, f, a[2] * k);
        a[3] = __builtin_fmaf(v[u].w, f, a[3] * k);
        M = mn;
      }
    }
    paged_store4<HD>(a, L, any, b, h0 + h, d0, nh, gate, gate_stride, out, out_stride, qx, dx);
  }
}

constexpr int kJoin = 512;

template <int HD>
__global__ __launch_bounds__(kJoin) void paged_join_kernel(const uint16_t *__restrict__ gate, int gate_stride,
                                                           uint16_t *__restrict__ out, int out_stride,
                                                           int8_t *__restrict__ qx, float *__restrict__ dx, int nh, int G,
                                                           int HW, const float *__restrict__ po,
                                                           const float *__restrict__ pml, const int2 *__restrict__ seg) {
  constexpr int TH = HD / 4, R = kJoin / TH;   // threads a part, parts a turn
  __shared__ __align__(16) float so[R][HD + 4];
  __shared__ float sm[kJoin / 64];
  const int h = blockIdx.x, b = blockIdx.y, r = threadIdx.x / TH, d0 = 4 * (threadIdx.x % TH);
  const int rows = HW * G;                   // heads of a group
  const int2 x = seg[(size_t)b * (nh / rows) + h / rows];
  const int ns = x.y - x.x + 1;
  if (ns == 1) return;                       // its workgroup has written the output
  // part i: the first workgroup's last piece, then the others' first ones
  auto part = [&](int i) { return ((size_t)(x.x + i) * 2 + (i == 0 ? 1 : 0)) * rows + h % rows; };
  const float2 *ml = reinterpret_cast<const float2 *>(pml);
  float M = -__builtin_inff();
  for (int i = threadIdx.x; i < ns; i += kJoin) M = fmaxf(M, ml[part(i)].x);
  M = wave_max(M);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoin / 64; i++) M = fmaxf(M, sm[i]);
  if (M == -__builtin_inff()) M = 0.0f;
  float L = 0.0f, a[4] = {0, 0, 0, 0};
  bool any = false;
  constexpr int U = 4;   // parts on their way at once
  for (int i0 = r; i0 < ns; i0 += U * R) {
    float2 p[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * R < ns ? i0 + u * R : i0;
      const size_t pj = part(i);
      p[u] = ml[pj];
      v[u] = *reinterpret_cast<const float4 *>(po + pj * HD + d0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (i0 + u * R >= ns || p[u].y < 0.0f) continue;
      any = true;
      const float f = __builtin_amdgcn_exp2f(p[u].x - M);
      L = __builtin_fmaf(p[u].y, f, L);
      a[0] = __builtin_fmaf(v[u].x, f, a[0]);
      a[1] = __builtin_fmaf(v[u].y, f, a[1]);
      a[2] = __builtin_fmaf(v[u].z, f, a[2]);
      a[3] = __builtin_fmaf(v[u].w, f, a[3]);
    }
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

// How a call is laid out: HW heads a workgroup, `grid` workgroups, of at least
// `share` tiles each (0: one a segment, no join).
//
// One workgroup a segment where it has at most 40 tiles (10 a wave): the even split
// costs a scan of the lengths and a second launch, about 6 us. Measured, a workgroup
// a segment / split evenly (us; lengths spread from a quarter to the whole): 32 q and 8 kv
// heads of 64, 1 sequence of 600 keys 12.4 / 16.9, 1200 13.2 / 16.9, 2400 20.0 / 17.0, 32 of
// 1200 16.1 / 22.5, 2400 31.0 / 33.4, 128 of 1200 46.5 / 50.0, 2400 86.0 / 82.7; 16 and 4 of
// 128, 8 of 1200 19.3 / 18.5, 2400 31.0 / 19.4, 128 of 1200 46.7 / 51.4, 2400 85.7 / 82.3.
// There four waves share a head's keys until 1024 heads fill the chip, then two heads'
// rows, which lie side by side, are read together: 256 sequences of 260 keys of 4 heads of
// 128 39.5 -> 33.8, 128 of 600 of 8 of 64 26.6 -> 24.9, 32 of 600 12.4 / 15.4.
//
// The even split takes 4 heads a workgroup and few workgroups: the fewer streams of
// keys, the longer each and the better memory answers (64 sequences of 8192 keys of 8
// heads of 64: 8 workgroups a CU in pieces of 256 keys 4.8 TB/s, one a CU 5.7). One a CU for
// head_dim 128 (131072 keys of 4 heads 58.4 us, two a CU 63.5), two for 64 (64
// sequences of up to 8192 112.4, one a CU 113.2, 128 of up to 600 32.5 / 36.1; all of
// these before the reads past the caches below).
//
// K and V are read past the caches (once) where they fill the last-level cache of 256
// MiB: 563 MB 112 -> 102 us, 128 sequences of up to 4800 keys of 8 heads of 64 151 -> 139. Through
// the caches / past them (us), 16 sequences of 8 heads of 64, one pool read again and
// again: 64 MiB 24.3 / 26.0, 128 33.2 / 36.6, 192 41.9 / 47.4, 256 52.4 / 57.4, 320 70.7 / 69.0,
// 512 112 / 101; six such pools in turn, as a model's layers are: 64 27.7 / 27.2, 128 38.9 /
// 37.2, 192 49.7 / 46.9, 256 60.9 / 56.5, 512 110 / 100. A call does not know which it is; the
// border keeps a pool that fits its place in the cache. Shorter ones lose more: 32 sequences
// of 1200, 50 MB, 15.8 / 21.8.
//
// by_wg, join by head / by workgroup (us), 32 q and 8 kv heads of 64, 4096 keys: 1 sequence 14.9 /
// 21.9, 8 22.9 / 27.5, 16 33.2 / 33.4, 32 61 / 56, 64 109 / 98; 16 and 4 of 128: 1 14.5 / 33.5, 16 31.8 / 37.9,
// 32 55 / 57.6, 64 97 / 96, 128 of 2048 102 / 95.
struct PagedPlan {
  int HW, grid, share, by_wg;
  bool once;
};
static PagedPlan paged_plan(int nseq, int nkv, int hd, int max_kv, int win, int sinks) {
  const int tiles = paged_tiles(max_kv, kPagedCap, win, sinks).count;
  const bool even = tiles > 40;
  PagedPlan p = {1, 1, 0, 0, false};
  p.once = (long long)nseq * nkv * tiles * (kTile * 4LL) * hd >= 256LL << 20;
  p.HW = even ? 4 : (long long)nseq * nkv >= 1024 ? 2 : 1;
  while (nkv % p.HW) p.HW >>= 1;
  const long long segs = (long long)nseq * (nkv / p.HW);
  if (!even) {
    p.grid = (int)segs;
    return p;
  }
  p.share = 2 * kWaves / p.HW;
  const int most = hd == 64 ? 512 : 256;
  const long long want = (segs * tiles + p.share - 1) / p.share;
  p.grid = (int)(want < most ? want : most);
  p.by_wg = segs * 8 >= p.grid ? 1 : 0;
  return p;
}
static size_t paged_ws(const PagedPlan &p, int nseq, int nh, int nkv, int hd) {
  if (p.share == 0) return 0;
  return (size_t)p.grid * 2 * p.HW * (nh / nkv) * (hd + 2) * sizeof(float) +
         (p.by_wg ? (size_t)p.grid : (size_t)nseq * (nkv / p.HW)) * sizeof(int2);
}

}  // namespace pq

using namespace pq;

extern "C" size_t pq_paged_decode_workspace_bytes(int nseq, int nh, int nkv, int hd, int max_kv, int win, int sinks) {
  if (nseq <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || (hd != 64 && hd != 128) || max_kv <= 0 || win < 0 || sinks < 0) return 0;
  return paged_ws(paged_plan(nseq, nkv, hd, max_kv, win, sinks), nseq, nh, nkv, hd);
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
  const PagedPlan p = paged_plan(v.nseq, v.nkv, hd, max_kv, win, sinks);
  const size_t need = paged_ws(p, v.nseq, nh, v.nkv, hd);
  PQ_REQUIRE(need == 0 || (ws && ws_bytes >= need), PQ_ERR_WORKSPACE, "%s: workspace of %zu bytes needed (got %zu)", who,
             need, ws ? ws_bytes : 0);
  PQ_REQUIRE(need == 0 || aligned(ws, 16), PQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", who);
  // the workspace: o of every part, their (m, l), the segments
  float *po = reinterpret_cast<float *>(ws), *pml = nullptr;
  int2 *seg = nullptr;
  if (need) {
    const size_t parts = (size_t)p.grid * 2 * p.HW * G;
    pml = po + parts * hd;
    seg = reinterpret_cast<int2 *>(pml + parts * 2);
  }
  const int qvec = aligned(q, 16) && q_stride % 8 == 0 ? 1 : 0;
  hipStream_t st = as_stream(stream);
  const size_t lds = (size_t)kWaves * G * (hd + 4) * sizeof(float);
#define PQ_SPLIT(HH, BB)                                                                                           \
  do {                                                                                                             \
    if (p.once)                                                                                                    \
      launch(paged_split_kernel<HH, BB, true>, dim3(p.grid), dim3(64 * kWaves), lds, st, q, q_stride, qvec, v, gate, \
             gate_stride, out, out_stride, qx, dx, nh, G, scale, win, sinks, p.HW, p.share, p.by_wg, po, pml, seg);  \
    else                                                                                                           \
      launch(paged_split_kernel<HH, BB, false>, dim3(p.grid), dim3(64 * kWaves), lds, st, q, q_stride, qvec, v, gate, \
             gate_stride, out, out_stride, qx, dx, nh, G, scale, win, sinks, p.HW, p.share, p.by_wg, po, pml, seg);  \
  } while (0)
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
  if (rl || p.share == 0) return rl;
#define PQ_JOIN(KERN, GRID, BLOCK)                                                                                    \
  launch(KERN, GRID, dim3(BLOCK), 0, st, gate, gate_stride, out, out_stride, qx, dx, nh, G, p.HW, (const float *)po, \
         (const float *)pml, (const int2 *)seg)
  if (p.by_wg) {
    if (hd == 64) PQ_JOIN(paged_join_few_kernel<64>, dim3(p.grid), 256);
    else PQ_JOIN(paged_join_few_kernel<128>, dim3(p.grid), 256);
  } else {
    if (hd == 64) PQ_JOIN(paged_join_kernel<64>, dim3(nh, v.nseq), kJoin);
    else PQ_JOIN(paged_join_kernel<128>, dim3(nh, v.nseq), kJoin);
  }
#undef PQ_JOIN
  return check_launch(who);
}
