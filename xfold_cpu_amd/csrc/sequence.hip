// Sequence attention for any head dim up to 128, in fp32 and for the bf16 layouts that
// sequence_bf16_forward.hip and sequence_bf16_backward.hip do not take (rows that are not whole 16-byte pieces):
// forward, dq, dk and dv.
//
// A workgroup owns 64 tokens (16 per wavefront, one per lane column): queries in the forward pass and
// for dq, keys for dk and dv. It walks the other side in tiles of 64, held row-major in LDS. With the
// owned tokens as the columns of every product,
//   forward  S^T = K Q^T                     O^T  += V^T P^T
//   dq       S^T = K Q^T, dP^T = V dO^T      dQ^T += K^T dS^T
//   dk, dv   S = Q K^T, dP = dO V^T          dV^T += dO^T P, dK^T += Q^T dS
// a lane holds four rows of one column after the first products, which is the B operand of the
// second ones up to a permutation of the 32 rows of a step; the A operand read applies the same. So no
// score leaves its lane but for the sums over the four lanes of a column.
//
// Tiles that no owned token sees are skipped: a wavefront tests 64 tiles at a time, one per lane. The next
// tile's loads are issued before the work on the one in LDS.
//
// What a masked place holds does not matter: its score is replaced and its weight is 0, but in the
// second products 0 times an infinity or a NaN of the other side is NaN. Such a sum cannot become
// finite again, so one test of the results finds it, and the tile loop runs once more in a form that
// takes these elements out of the operand (as 0) and adds them to the rows that see them.
//
// fp32, D = 128: 57 to 65 TFLOP/s forward, 45 backward, of the 136 of a large product, with one wavefront per SIMD
// (its registers hold the sums). 384 tokens in 3 chains, 16 heads of 24: 30 us forward, the tiles one after the other
// on 96 workgroups.
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "sequence.h"

namespace xfh {
namespace {

using namespace seq;

// Range of each tile of 64 keys: one wavefront per tile (3 us, a launch's own time).
__global__ __launch_bounds__(256) void ranges_kernel(SequenceArgs a, Range *out) {
  const int64_t item = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> 6;
  if (item >= int64_t(a.B) * a.tiles) return;
  const int b = int(item / a.tiles), tile = int(item % a.tiles), lane = threadIdx.x & 63;
  const int key = tile * kTile + lane;
  const int n = place_of(a, b).n;
  const int id = key < n ? a.documents[int64_t(b) * a.documents_stride + key] : -1;
  int lo = id < 0 ? 0x7fffffff : id, hi = id < 0 ? -1 : id;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o, 64));
    hi = max(hi, __shfl_xor(hi, o, 64));
  }
  const bool full = __ballot(id < 0) == 0;
  if (lane == 0) out[item] = Range{lo, hi, full, 0};
}

template <typename T> constexpr int pitch_pad() { return 16 / int(sizeof(T)); }

// Rows [row0, row0 + 64) of a [rows][D] matrix to LDS, zero beyond its end and beyond D, in two steps: `fetch` issues
// the loads of the next tile before the work on this one, `put` stores them after it. Rows that are not
// whole 16-byte pieces are read element by element by `put`.
template <typename T, int DP> struct TileLoad {
  typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
  static constexpr int P = DP + pitch_pad<T>(), E = 16 / int(sizeof(T)), N = kTile * DP / E / 256;
  static_assert(N * 256 * E == kTile * DP, "whole pieces for each thread");
  u32x4 v[N];
  __device__ __forceinline__ void fetch(const T *src, int64_t stride, int row0, int rows, int D, bool vec) {
    if (!vec) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = j * 256 + threadIdx.x, r = i / (DP / E), c = (i % (DP / E)) * E;
      v[j] = u32x4{0, 0, 0, 0};
      if (row0 + r < rows && c < D) v[j] = *reinterpret_cast<const u32x4 *>(src + int64_t(row0 + r) * stride + c);
    }
  }
  __device__ __forceinline__ void put(T *dst, const T *src, int64_t stride, int row0, int rows, int D, bool vec) const {
    if (vec) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = j * 256 + threadIdx.x;
        *reinterpret_cast<u32x4 *>(dst + i / (DP / E) * P + (i % (DP / E)) * E) = v[j];
      }
    } else {
#pragma unroll 8
      for (int i = threadIdx.x; i < kTile * DP; i += 256) {
        const int r = i / DP, c = i % DP;
        dst[r * P + c] = row0 + r < rows && c < D ? src[int64_t(row0 + r) * stride + c] : T(0.f);
      }
    }
  }
};
// The owned token's row as B fragments: d = 32 step + 8 grp + 0..7.
template <typename T, int DP>
__device__ __forceinline__ void load_own(typename Frag<T>::type (&f)[DP / 32], const T *row, int D, bool valid, int grp,
                                         bool vec) {
#pragma unroll
  for (int st = 0; st < DP / 32; ++st) {
    __attribute__((aligned(16))) T t[8];
    if (vec) {
      typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
      constexpr int E = 16 / int(sizeof(T));
#pragma unroll
      for (int e = 0; e < 8; e += E) {
        const int d = st * 32 + grp * 8 + e;
        u32x4 v = {0, 0, 0, 0};
        if (valid && d < D) v = *reinterpret_cast<const u32x4 *>(row + d);
        __builtin_memcpy(t + e, &v, 16);
      }
      __builtin_memcpy(&f[st], t, sizeof(t));
      continue;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = st * 32 + grp * 8 + e;
      t[e] = valid && d < D ? row[d] : T(0.f);
    }
    __builtin_memcpy(&f[st], t, sizeof(t));
  }
}
// Product of the tile's 64 rows with the owned columns: acc[kt][e] is row 16 kt + 4 grp + e.
template <typename T, int DP>
__device__ __forceinline__ void tile_product(const T *tile, const typename Frag<T>::type (&own)[DP / 32], f32x4 (&acc)[4]) {
  constexpr int P = DP + pitch_pad<T>();
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    acc[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < DP / 32; ++st) {
      typename Frag<T>::type f;
      __builtin_memcpy(&f, tile + (kt * 16 + col) * P + st * 32 + grp * 8, sizeof(f));
      acc[kt] = mfma16(f, own[st], acc[kt]);
    }
  }
}

template <typename T> __device__ __forceinline__ bool finite(T x) { return fabsf(to_f32(x)) < INFINITY; }

// acc[t] (rows 16 t + 4 grp + e of the result) += tile^T w, w the 64 rows' weights of this column.
// strict: elements that are not finite count as 0 here and are then added where `seen` (bit 4 kt + e)
// says so: an infinity as itself when `weights` says that w >= 0, else as NaN.
template <typename T, int DP>
__device__ __forceinline__ void add_transposed(const T *tile, const float (&w)[4][4], uint32_t seen, bool strict,
                                               bool weights, f32x4 (&acc)[DP / 16]) {
  constexpr int P = DP + pitch_pad<T>();
  typedef typename Frag<T>::type F;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    T wt[8], st[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      wt[e] = from_f32<T>(w[2 * c][e]);
      wt[4 + e] = from_f32<T>(w[2 * c + 1][e]);
      st[e] = T((seen >> (8 * c + e)) & 1 ? 1.f : 0.f);
      st[4 + e] = T((seen >> (8 * c + 4 + e)) & 1 ? 1.f : 0.f);
    }
    F wf, sf;
    __builtin_memcpy(&wf, wt, sizeof(wt));
    __builtin_memcpy(&sf, st, sizeof(st));
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      T at[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        at[e] = tile[(c * 32 + grp * 4 + e) * P + t * 16 + col];
        at[4 + e] = tile[(c * 32 + 16 + grp * 4 + e) * P + t * 16 + col];
      }
      F af;
      if (strict) {
        T up[8], down[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool bad = !finite(at[e]);
          const float x = to_f32(at[e]);
          up[e] = T(bad && !(weights && x < 0.f) ? 1.f : 0.f);
          down[e] = T(bad && !(weights && x > 0.f) ? 1.f : 0.f);
          if (bad) at[e] = T(0.f);
        }
        F uf, df;
        __builtin_memcpy(&uf, up, sizeof(up));
        __builtin_memcpy(&df, down, sizeof(down));
        const f32x4 ups = mfma16(uf, sf, f32x4{0.f, 0.f, 0.f, 0.f}), downs = mfma16(df, sf, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (ups[e] > 0.f) acc[t][e] += INFINITY;
          if (downs[e] > 0.f) acc[t][e] -= INFINITY;
        }
      }
      __builtin_memcpy(&af, at, sizeof(at));
      acc[t] = mfma16(af, wf, acc[t]);
    }
  }
}

__device__ __forceinline__ float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// Score of a pair, and d(score)/d(dot) up to `scale`. bf16: in log 2 units. fp32: as it is, and its difference to
// the row's maximum is taken before the change of base (a score of 10 changed first is off by 1e-6).
template <typename T> __device__ __forceinline__ constexpr float score_unit() { return sizeof(T) == 4 ? 1.0f : kLog2e; }
template <typename T> __device__ __forceinline__ float weight_of(float x, float m) {
  return __builtin_amdgcn_exp2f(sizeof(T) == 4 ? (x - m) * kLog2e : x - m);
}
template <typename T> struct Scorer {
  float scale, cap, inv_cap, slope;
  __device__ __forceinline__ Scorer(const SequenceArgs &a, int h)
      : scale(a.scale), cap(a.cap), inv_cap(a.cap > 0.f ? 1.0f / a.cap : 0.f), slope(a.slopes ? a.slopes[h] * score_unit<T>() : 0.f) {}
  __device__ __forceinline__ float operator()(const SequenceArgs &a, float dot, int pos, int key, float &factor) const {
    float x = dot * scale;
    factor = 1.f;
    if (a.cap > 0.f) {
      const float t = bend<T>(x * inv_cap);
      factor = 1.f - t * t;
      x = cap * t;
    }
    x *= score_unit<T>();
    if (a.slopes) x -= slope * fabsf(float(pos - key));
    return x;
  }
};

// A row's statistics for the backward pass. bf16: a = its log 2 sum, P = exp2(score - a). fp32: a = its maximum, b =
// 1 / sum, P = exp(score - a) b, in two planes of a.lse. No visible key: P is 0.
struct Stat { float a, b; };
template <typename T> __device__ __forceinline__ void put_stat(const SequenceArgs &a, int64_t at, float m, float l) {
  if (sizeof(T) == 4) {
    a.lse[at] = l == 0.f ? 0.f : m;
    a.lse[int64_t(a.B) * a.H * a.Nq + at] = l == 0.f ? 0.f : 1.0f / l;
  } else {
    a.lse[at] = l == 0.f ? INFINITY : m + log2f(l);
  }
}
template <typename T> __device__ __forceinline__ Stat get_stat(const SequenceArgs &a, int64_t at, bool valid) {
  if (!valid) return {INFINITY, 0.f};
  return {a.lse[at], sizeof(T) == 4 ? a.lse[int64_t(a.B) * a.H * a.Nq + at] : 1.f};
}
template <typename T> __device__ __forceinline__ float probability(float x, const Stat &s) {
  return sizeof(T) == 4 ? weight_of<T>(x, s.a) * s.b : weight_of<T>(x, s.a);
}

// What a workgroup with 64 columns of queries works on: columns and work items are as in the bf16 kernels
// (sequence_bf16_forward.hip), query by query over the heads that share a key head.
struct Columns {
  int b, h, hk, i, c;
  bool valid;
  Place place;
  Row row;
  Span span;
  __device__ __forceinline__ Columns(const SequenceArgs &a, const Part &part) {
    const int group = a.H / a.Hk, columns = group * a.Nq, blk = part.blk;
    hk = part.hk;
    b = part.b;
    const int c0 = blk * kTile, c1 = min(c0 + kTile, columns) - 1;
    c = c0 + (threadIdx.x >> 6) * 16 + (threadIdx.x & 15);
    valid = c < columns;
    i = valid ? c / group : a.Nq;
    h = hk * group + (valid ? c % group : 0);
    place = place_of(a, b);
    row = row_of(a, place, b, i);
    span = span_of(a, place, b, c0 / group, c1 / group);
  }
};

template <typename T, int DP>
__global__ __launch_bounds__(256) void forward_kernel(SequenceArgs a, int blocks, Parts parts, bool vec) {
  constexpr int P = DP + pitch_pad<T>();
  __shared__ __attribute__((aligned(16))) T ks[kTile * P], vs[kTile * P];
  __shared__ int ids[kTile];
  const Part part(a, parts, blocks, blockIdx.x);
  if (part.count == 0) return;
  const Columns own(a, part);
  const int b = own.b, h = own.h, hk = own.hk, i = own.i;
  const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4;
  const Place &place = own.place;
  const bool valid = own.valid;
  const Row &row = own.row;
  const T *kp = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1];
  const T *vp = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1];
  typename Frag<T>::type qf[DP / 32];
  load_own<T, DP>(qf, static_cast<const T *>(a.q) + b * a.qs[0] + h * a.qs[1] + i * a.qs[2], a.D, valid, grp, vec);
  const auto test = [&](int tile) { return key_tile_needs(a, b, tile, own.span, own.span); };
  const Scorer<T> score(a, h);
  int end = (own.span.high + kTile - 1) / kTile, begin = 0;
  if (several(parts)) part.take(begin, end);

  f32x4 o[DP / 16];
  float m, l;
  for (int strict = 0; strict < 2; ++strict) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    Walk walk(begin, end);
    Step now = walk.next(test);
    TileLoad<T, DP> kt, vt;
    int id = -1;
    const auto fetch = [&](int k0) {
      kt.fetch(kp, a.ks[2], k0, place.n, a.D, vec);
      vt.fetch(vp, a.vs[2], k0, place.n, a.Dv, vec);
      if (a.documents && tid < kTile) id = k0 + tid < place.n ? a.documents[int64_t(b) * a.documents_stride + k0 + tid] : -1;
    };
    if (now.tile >= 0) fetch(now.tile * kTile);
    {
      while (now.tile >= 0) {
        const int k0 = now.tile * kTile;
        const bool whole = now.whole;
        __syncthreads();
        kt.put(ks, kp, a.ks[2], k0, place.n, a.D, vec);
        vt.put(vs, vp, a.vs[2], k0, place.n, a.Dv, vec);
        if (tid < kTile) ids[tid] = id;
        __syncthreads();
        now = walk.next(test);
        if (now.tile >= 0) fetch(now.tile * kTile);
        f32x4 s[4];
        tile_product<T, DP>(ks, qf, s);
        float w[4][4];
        uint32_t seen = 0;
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = kt * 16 + grp * 4 + e, key = k0 + r;
            const bool see = whole || (key < row.limit && (!a.documents || ids[r] == row.document));
            float factor;
            const float x = score(a, s[kt][e], row.pos, key, factor);
            w[kt][e] = x;
            if (see) {
              seen |= 1u << (4 * kt + e);
              top = fmaxf(top, x);
            }
          }
        const float m_new = fmaxf(m, column_max(top)), base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = weight_of<T>(m, base);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) o[t] *= alpha;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[kt][e] = (seen >> (4 * kt + e)) & 1 ? weight_of<T>(w[kt][e], base) : 0.f;
            l += w[kt][e];
          }
        add_transposed<T, DP>(vs, w, seen, strict != 0, true, o);
      }
    }
    bool bad = false;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[t][e]) < INFINITY);
    if (!__syncthreads_or(valid && bad)) break;
  }
  l = column_sum(l);
  if (!valid) return;
  if (several(parts)) {
    const int64_t at = (int64_t(part.slot) * a.Hk + hk) * (a.H / a.Hk * a.Nq) + own.c;
    if (grp == 0) parts.ml[at] = make_float2(m, l);
    if (l == 0.f) return;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = t * 16 + grp * 4 + e;
        if (d < a.Dv) parts.o[at * a.Dv + d] = o[t][e];
      }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  T *op = static_cast<T *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2];
#pragma unroll
  for (int t = 0; t < DP / 16; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = t * 16 + grp * 4 + e;
      if (d < a.Dv) {
        const float x = o[t][e] * inv;
        const T r = from_f32<T>(x);
        op[d] = r;
        if (a.low) static_cast<bf16 *>(a.low)[((int64_t(b) * a.H + h) * a.Nq + i) * a.Dv + d] = bf16(x - to_f32(r));
      }
    }
  if (a.lse && grp == 0) put_stat<T>(a, (int64_t(b) * a.H + h) * a.Nq + i, m, l);
}

// Joins the parts of split keys, in their order: a thread per element, or per 4 where Dv is a multiple of 4. Bound by
// reading the parts: 30 MB of 4 x 200 queries in 10 us.
template <typename T, int N> __global__ __launch_bounds__(256) void join_kernel(SequenceArgs a, Parts parts) {
  const int group = a.H / a.Hk, columns = group * a.Nq, pieces = a.Dv / N;
  const int64_t total = int64_t(a.B) * a.Hk * columns, at = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= total * pieces) return;
  const int64_t column = at / pieces;
  const int d = int(at - column * pieces) * N;
  const int c = int(column % columns), bk = int(column / columns), hk = bk % a.Hk, b = bk / a.Hk;
  int slot = b, step = a.B, count = parts.splits;
  if (parts.table) {
    const int2 t = parts.table[b];
    slot = t.x;
    step = 1;
    count = t.y;
  }
  const int64_t from = (int64_t(slot) * a.Hk + hk) * columns + c, stride = int64_t(step) * a.Hk * columns;
  // Four parts at a time, whose loads do not wait for each other (for tokens of 16 sequences of up to 8192 keys forward pass
  // and join take 62.5 us, 64.3 with one part at a time; eight take more registers: 75 us for 72 in the case at seq::Part).
  constexpr int kBatch = 4;
  float top = kLowest;
  for (int s = 0; s < count; s += kBatch) {
    float m[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch; ++e) m[e] = s + e < count ? parts.ml[from + (s + e) * stride].x : kLowest;
#pragma unroll
    for (int e = 0; e < kBatch; ++e) top = fmaxf(top, m[e]);
  }
  float sum = 0.f, v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = 0.f;
  for (int s = 0; s < count; s += kBatch) {
    float2 p[kBatch];
    float o[kBatch][N];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (s + j >= count) break;
      const int64_t row = from + (s + j) * stride;
      p[j] = parts.ml[row];
      __builtin_memcpy(o[j], __builtin_assume_aligned(parts.o + row * a.Dv + d, 4 * N), 4 * N);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (s + j >= count || p[j].y == 0.f) continue;     // (a part whose sum is 0 has no o)
      const float f = weight_of<T>(p[j].x, top);
      sum += f * p[j].y;
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] += f * o[j][e];
    }
  }
  const int i = c / group, h = hk * group + c % group;
  const int64_t row = (int64_t(b) * a.H + h) * a.Nq + i;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  T r[N];
  bf16 low[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float x = v[e] * inv;
    r[e] = from_f32<T>(x);
    low[e] = bf16(x - to_f32(r[e]));
  }
  T *out = static_cast<T *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2] + d;
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = r[e];
  if (a.low) {
#pragma unroll
    for (int e = 0; e < N; ++e) static_cast<bf16 *>(a.low)[row * a.Dv + d + e] = low[e];
  }
  if (a.lse && d == 0) put_stat<T>(a, row, top, sum);
}

// delta = dout . out of each query, four lanes a row.
template <typename T> __global__ __launch_bounds__(256) void delta_kernel(SequenceArgs a) {
  const int64_t at = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> 2;
  if (at >= int64_t(a.B) * a.H * a.Nq) return;           // (all lanes of a row)
  const int i = int(at % a.Nq), h = int(at / a.Nq % a.H), b = int(at / a.Nq / a.H);
  const T *gp = static_cast<const T *>(a.dout) + b * a.gs[0] + h * a.gs[1] + i * a.gs[2];
  const T *op = static_cast<const T *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2];
  const bf16 *low = a.low ? static_cast<const bf16 *>(a.low) + at * a.Dv : nullptr;
  float delta = 0.f;
  for (int d = threadIdx.x & 3; d < a.Dv; d += 4) delta += to_f32(gp[d]) * (to_f32(op[d]) + (low ? to_f32(low[d]) : 0.f));
  delta += __shfl_xor(delta, 1, 64);
  delta += __shfl_xor(delta, 2, 64);
  if (threadIdx.x % 4 == 0) a.delta[at] = delta;
}

// dq of 64 queries, and the slopes' part of each query,
//   - sum_j P (dP - sum P dP) |gap| = - (sum_j P (dP - delta) |gap| - (sum_j P (dP - delta)) (sum_j P |gap|)),
// in fp32 from unrounded values: delta, which has the output's rounding in it, drops out, and so does
// what the row's P are off by together, since each sum is divided by theirs.
template <typename T, int DP>
__device__ __forceinline__ void dq_block(const SequenceArgs &a, int blocks, bool vec, unsigned item, T *ks, T *vs, int *ids) {
  const Columns own(a, Part(a, Parts{nullptr, nullptr, nullptr, 1, a.B}, blocks, item));
  const int b = own.b, h = own.h, hk = own.hk, i = own.i;
  const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4;
  const Place &place = own.place;
  const bool valid = own.valid;
  const Row &row = own.row;
  const T *kp = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1];
  const T *vp = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1];
  typename Frag<T>::type qf[DP / 32], gf[DP / 32];
  load_own<T, DP>(qf, static_cast<const T *>(a.q) + b * a.qs[0] + h * a.qs[1] + i * a.qs[2], a.D, valid, grp, vec);
  const T *gp = static_cast<const T *>(a.dout) + b * a.gs[0] + h * a.gs[1] + i * a.gs[2];
  load_own<T, DP>(gf, gp, a.Dv, valid, grp, vec);
  const int64_t at = (int64_t(b) * a.H + h) * a.Nq + i;
  const float delta = valid ? a.delta[at] : 0.f;
  const Stat stat = get_stat<T>(a, at, valid);
  const auto test = [&](int tile) { return key_tile_needs(a, b, tile, own.span, own.span); };
  const Scorer<T> score(a, h);

  f32x4 dq[DP / 16];
  float all, far, error, far_error;
  for (int strict = 0; strict < 2; ++strict) {
    all = far = error = far_error = 0.f;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) dq[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    Walk walk(0, (own.span.high + kTile - 1) / kTile);
    Step now = walk.next(test);
    TileLoad<T, DP> kt, vt;
    int id = -1;
    const auto fetch = [&](int k0) {
      kt.fetch(kp, a.ks[2], k0, place.n, a.D, vec);
      vt.fetch(vp, a.vs[2], k0, place.n, a.Dv, vec);
      if (a.documents && tid < kTile) id = k0 + tid < place.n ? a.documents[int64_t(b) * a.documents_stride + k0 + tid] : -1;
    };
    if (now.tile >= 0) fetch(now.tile * kTile);
    {
      while (now.tile >= 0) {
        const int k0 = now.tile * kTile;
        const bool whole = now.whole;
        __syncthreads();
        kt.put(ks, kp, a.ks[2], k0, place.n, a.D, vec);
        vt.put(vs, vp, a.vs[2], k0, place.n, a.Dv, vec);
        if (tid < kTile) ids[tid] = id;
        __syncthreads();
        now = walk.next(test);
        if (now.tile >= 0) fetch(now.tile * kTile);
        f32x4 s[4], dp[4];
        tile_product<T, DP>(ks, qf, s);
        tile_product<T, DP>(vs, gf, dp);
        float w[4][4];
        uint32_t seen = 0;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = kt * 16 + grp * 4 + e, key = k0 + r;
            const bool see = valid && (whole || (key < row.limit && (!a.documents || ids[r] == row.document)));
            float factor;
            const float x = score(a, s[kt][e], row.pos, key, factor);
            const float p = see ? probability<T>(x, stat) : 0.f;
            const float ds = see ? p * (dp[kt][e] - delta) : 0.f;
            w[kt][e] = ds * factor;
            seen |= see ? 1u << (4 * kt + e) : 0u;
            if (a.slope_part && see) {
              const float gap = fabsf(float(row.pos - key));
              all += p;
              far += p * gap;
              error += ds;
              far_error += ds * gap;
            }
          }
        add_transposed<T, DP>(ks, w, seen, strict != 0, false, dq);
      }
    }
    bool bad = false;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !(fabsf(dq[t][e]) < INFINITY);
    if (!__syncthreads_or(valid && bad)) break;
  }
  if (valid) {
    T *out = static_cast<T *>(a.dq) + b * a.dqs[0] + h * a.dqs[1] + i * a.dqs[2];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = t * 16 + grp * 4 + e;
        if (d < a.D) out[d] = from_f32<T>(dq[t][e] * a.scale);
      }
  }
  if (a.slope_part) {
    all = column_sum(all);
    far = column_sum(far);
    error = column_sum(error);
    far_error = column_sum(far_error);
    if (valid && grp == 0) a.slope_part[(int64_t(h) * a.B + b) * a.Nq + i] = slope_gradient(all, far, error, far_error);
  }
}

// dk and dv of 64 keys: over the heads that share them and the queries that see them (of a work item's share).
template <typename T, int DP>
__device__ __forceinline__ void dkv_block(const SequenceArgs &a, const Splits &splits, float *parts, bool vec, unsigned number,
                                          T *qs, T *gs, Row *rows, Stat *stats, float *deltas) {
  const KeyItem item(a, splits, number);
  const int hk = item.hk, b = item.b, block = item.block, group = a.H / a.Hk;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
  const Place place = place_of(a, b);
  const int k0 = block * kTile, key = k0 + wave * 16 + col;
  const bool valid = key < place.n;
  typename Frag<T>::type kf[DP / 32], vf[DP / 32];
  load_own<T, DP>(kf, static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1] + key * a.ks[2], a.D, valid, grp, vec);
  load_own<T, DP>(vf, static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1] + key * a.vs[2], a.Dv, valid, grp, vec);
  int id = 0;
  Range mine{};
  if (a.documents) {
    id = valid ? a.documents[int64_t(b) * a.documents_stride + key] : -1;
    mine = static_cast<const Range *>(a.ranges)[int64_t(b) * a.tiles + block];
  }

  f32x4 dk[DP / 16], dv[DP / 16];
  for (int strict = 0; strict < 2; ++strict) {
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) dk[t] = dv[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int g = item.share.head0; g < item.share.head1; ++g) {
      const int h = hk * group + g;
      const T *qp = static_cast<const T *>(a.q) + b * a.qs[0] + h * a.qs[1];
      const T *gp = static_cast<const T *>(a.dout) + b * a.gs[0] + h * a.gs[1];
      const Scorer<T> score(a, h);
      const int64_t at = (int64_t(b) * a.H + h) * a.Nq;
      const auto test = [&](int tile) {
        const int r0 = tile * kTile, r1 = min(r0 + kTile, a.Nq) - 1;
        Needs n{limit_of(a, place, r1) > k0, true, r0 + kTile <= a.Nq && limit_of(a, place, r0) >= k0 + kTile};
        if (a.documents && n.block) {
          const Range r = query_range(a, place, b, r0, r1);
          n.block = overlap(r, mine);
          n.whole = n.whole && same_document(r, mine);
        }
        return n;
      };
      Walk walk(item.share.tile0, item.share.tile1);
      Step now = walk.next(test);
      TileLoad<T, DP> qt, gt;
      Row next_row{};
      Stat next_stat{INFINITY, 0.f};
      float next_delta = 0.f;
      const auto fetch = [&](int i0) {
        qt.fetch(qp, a.qs[2], i0, a.Nq, a.D, vec);
        gt.fetch(gp, a.gs[2], i0, a.Nq, a.Dv, vec);
        if (tid < kTile) {
          const int i = i0 + tid;
          next_row = row_of(a, place, b, i);
          next_stat = get_stat<T>(a, at + i, i < a.Nq);
          next_delta = i < a.Nq ? a.delta[at + i] : 0.f;
        }
      };
      if (now.tile >= 0) fetch(now.tile * kTile);
      {
        while (now.tile >= 0) {
          const int i0 = now.tile * kTile;
          const bool all = now.whole;
          __syncthreads();
          qt.put(qs, qp, a.qs[2], i0, a.Nq, a.D, vec);
          gt.put(gs, gp, a.gs[2], i0, a.Nq, a.Dv, vec);
          if (tid < kTile) {
            rows[tid] = next_row;
            stats[tid] = next_stat;
            deltas[tid] = next_delta;
          }
          __syncthreads();
          now = walk.next(test);
          if (now.tile >= 0) fetch(now.tile * kTile);
          f32x4 s[4], dp[4];
          tile_product<T, DP>(qs, kf, s);
          tile_product<T, DP>(gs, vf, dp);
          float pw[4][4], w[4][4];
          uint32_t seen = 0;
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = kt * 16 + grp * 4 + e;
              const Row row = rows[r];
              const bool see = valid && (all || (key < row.limit && (!a.documents || id == row.document)));
              float factor;
              const float x = score(a, s[kt][e], row.pos, key, factor);
              pw[kt][e] = see ? probability<T>(x, stats[r]) : 0.f;
              w[kt][e] = see ? pw[kt][e] * (dp[kt][e] - deltas[r]) * factor : 0.f;
              seen |= see ? 1u << (4 * kt + e) : 0u;
            }
          add_transposed<T, DP>(gs, pw, seen, strict != 0, false, dv);
          add_transposed<T, DP>(qs, w, seen, strict != 0, false, dk);
        }
      }
    }
    bool bad = false;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !(fabsf(dk[t][e]) < INFINITY) || !(fabsf(dv[t][e]) < INFINITY);
    if (!__syncthreads_or(valid && bad)) break;
  }
  if (key >= a.Nk) return;                                 // (keys beyond a length: zeros)
  if (splits.heads * splits.tiles > 1) {
    float *to = parts + ((int64_t(item.split) * a.B * a.Hk + int64_t(b) * a.Hk + hk) * a.Nk + key) * (a.D + a.Dv);
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = t * 16 + grp * 4 + e;
        if (d < a.D) to[d] = valid ? dk[t][e] : 0.f;
        if (d < a.Dv) to[a.D + d] = valid ? dv[t][e] : 0.f;
      }
    return;
  }
  T *kout = static_cast<T *>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2];
  T *vout = static_cast<T *>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2];
#pragma unroll
  for (int t = 0; t < DP / 16; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = t * 16 + grp * 4 + e;
      if (d < a.D) kout[d] = from_f32<T>(valid ? dk[t][e] * a.scale : 0.f);
      if (d < a.Dv) vout[d] = from_f32<T>(valid ? dv[t][e] : 0.f);
    }
}

// Both in one launch, dq's work items first, with dout . out from delta_kernel: each alone leaves CUs idle, at its
// end at least. In fp32, one launch and two: 384 tokens in 3 chains, 16 heads of 24, 40 and 62 us; the backward pass of
// 2 x 1111, 8 heads on 2, D = 64, 222 and 256 us; where there is work for all CUs 684 and 660 (2 x 1024, 16 heads of
// 96), 812 and 778 (4 x 2048, 8 of 32). Up to 32 dims two workgroups fit a CU's registers, if the compiler is held to
// it (1161 us in the last case if not).
template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 32 ? 2 : 1) void backward_kernel(SequenceArgs a, int blocks, int dq_items, Splits splits, float *parts, bool vec) {
  constexpr int P = DP + pitch_pad<T>();
  __shared__ __attribute__((aligned(16))) T tile0[kTile * P], tile1[kTile * P];
  __shared__ Row rows[kTile];
  __shared__ Stat stats[kTile];
  __shared__ float deltas[kTile];
  __shared__ int ids[kTile];
  if (int(blockIdx.x) < dq_items) dq_block<T, DP>(a, blocks, vec, blockIdx.x, tile0, tile1, ids);
  else dkv_block<T, DP>(a, splits, parts, vec, blockIdx.x - dq_items, tile0, tile1, rows, stats, deltas);
}

// dk and dv from the parts of their work items, in order: a thread per element, or per 4 (2 x 4096 tokens, 4 key heads of
// 128 in two parts: 67 MB in 16 us).
template <typename T, int N> __global__ __launch_bounds__(256) void dkv_join_kernel(SequenceArgs a, int splits, const float *parts) {
  const int width = a.D + a.Dv, pieces = width / N;
  const int64_t rows = int64_t(a.B) * a.Hk * a.Nk, at = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= rows * pieces) return;
  const int64_t row = at / pieces;
  const int d = int(at - row * pieces) * N;
  float sum[N];
#pragma unroll
  for (int e = 0; e < N; ++e) sum[e] = 0.f;
  for (int s = 0; s < splits; ++s) {
    float p[N];
    __builtin_memcpy(p, __builtin_assume_aligned(parts + (s * rows + row) * width + d, 4 * N), 4 * N);
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] += p[e];
  }
  const int key = int(row % a.Nk), bk = int(row / a.Nk), hk = bk % a.Hk, b = bk / a.Hk;
  T *out = d < a.D ? static_cast<T *>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2] + d
                   : static_cast<T *>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2] + d - a.D;
  const float scale = d < a.D ? a.scale : 1.f;
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = from_f32<T>(sum[e] * scale);
}

// dslopes[h]: the sum of its parts, in their order.
__global__ __launch_bounds__(256) void dslopes_kernel(const float *part, int64_t count, float *out) {
  __shared__ double sums[256];
  double t = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 256) t += double(part[blockIdx.x * count + i]);
  sums[threadIdx.x] = t;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (int(threadIdx.x) < o) sums[threadIdx.x] += sums[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[blockIdx.x] = float(sums[0]);
}

// Rows that can be read 16 bytes at a time.
template <typename T> bool vector_rows(std::initializer_list<std::pair<const void *, const int64_t *>> tensors, int64_t D) {
  constexpr int64_t E = 16 / sizeof(T);
  if (D % E) return false;
  for (const auto &t : tensors)
    if (reinterpret_cast<uintptr_t>(t.first) % 16 || t.second[0] % E || t.second[1] % E || t.second[2] % E) return false;
  return true;
}

template <typename T, int DP> int launch_forward(const SequenceArgs &a, const Parts &parts, hipStream_t s) {
  const int64_t blocks = ceil_div(int64_t(a.H / a.Hk) * a.Nq, int64_t(kTile));
  const bool vec = vector_rows<T>({{a.q, a.qs}, {a.k, a.ks}}, a.D) && vector_rows<T>({{a.v, a.vs}}, a.Dv);
  forward_kernel<T, DP><<<dim3(unsigned(blocks * a.Hk * parts.slots)), 256, 0, s>>>(a, int(blocks), parts, vec);
  return check_launch("sequence_attention");
}

template <typename T, int DP> int launch_backward(const SequenceArgs &a, const Splits &splits, float *parts, hipStream_t s) {
  const int64_t qblocks = ceil_div(int64_t(a.H / a.Hk) * a.Nq, int64_t(kTile)), kblocks = ceil_div(a.Nk, int64_t(kTile));
  const bool vec = vector_rows<T>({{a.k, a.ks}, {a.q, a.qs}}, a.D) && vector_rows<T>({{a.v, a.vs}, {a.dout, a.gs}}, a.Dv);
  const int64_t dq_items = qblocks * a.Hk * a.B, dkv_items = a.dk || a.dv ? kblocks * a.Hk * a.B * splits.heads * splits.tiles : 0;
  if (dq_items > 0) delta_kernel<T><<<dim3(unsigned(ceil_div(int64_t(a.B) * a.H * a.Nq, int64_t(64)))), 256, 0, s>>>(a);
  XFH_TRY(check_launch("sequence_attention_backward"));
  return sequence_launch_both(dq_items, dkv_items, [&](int64_t items, int64_t first) {
    backward_kernel<T, DP><<<dim3(unsigned(items)), 256, 0, s>>>(a, int(qblocks), int(first), splits, parts, vec);
  });
}

int check_grid(const SequenceArgs &a) {
  // At most 64 splits of a work item's keys, and those only of few work items.
  const int64_t most = std::max((ceil_div(int64_t(a.Nq), int64_t(kTile)) + 1) * a.H, ceil_div(int64_t(a.Nk), int64_t(kTile)) * a.Hk) * a.B;
  if (most > kMostItems || int64_t(a.H / std::max(a.Hk, 1)) * a.Nq > (int64_t(1) << 31) - 256)
    return fail(XFH_EUNSUPPORTED, "sequence_attention: problem too large");
  return XFH_OK;
}

}  // namespace

int64_t sequence_ranges_bytes(int64_t B, int64_t Nk) { return B * ceil_div(Nk, int64_t(kTile)) * int64_t(sizeof(Range)); }

int sequence_ranges(const SequenceArgs &a, hipStream_t s) {
  const int64_t items = int64_t(a.B) * a.tiles;
  if (!a.documents || items == 0) return XFH_OK;
  if (ceil_div(items, int64_t(4)) > (int64_t(1) << 31) - 1) return fail(XFH_EUNSUPPORTED, "sequence_attention: problem too large");
  ranges_kernel<<<dim3(unsigned(ceil_div(items, int64_t(4)))), 256, 0, s>>>(a, static_cast<Range *>(const_cast<void *>(a.ranges)));
  return check_launch("sequence_attention");
}

// Whether the parts are distributed by the sequences' lengths, which only the device has (seq::Part).
static bool shares_slots(const SequenceArgs &a) { return a.lengths && a.B > 1 && int64_t(a.H / a.Hk) * a.Nq > 32; }

SequenceSplits sequence_splits(const SequenceArgs &a, int dtype) {
  SequenceSplits n{1, a.B, {1, 1}};
  if (a.B == 0 || a.H == 0 || a.Hk == 0) return n;
  const bool bf = dtype == XFH_BF16 && sequence_bf16_forward_fits(a);
  const int64_t columns = int64_t(a.H / a.Hk) * a.Nq, single = int64_t(a.B) * a.Hk;
  if (columns > 0 && a.Nk > 0) {
    // Keys are split until there are about 512 work items (two workgroups per CU), down to 8 tiles each: 4 x 200
    // queries of up to 5000 keys in bf16 (224 work items) take 124 us in one part each. Sequences with lengths of
    // their own share the parts by need (seq::Part). Up to 32 columns (single tokens): down to 4 tiles, in equal
    // parts. Their workgroups fill a CU's LDS at D = 128: 256 parts, all at once, take 97 us for 16 tokens of 8192 keys (8 key
    // heads) and 101 for one of 100000, 512 take 106 and 134. With lengths 512, so that a CU with a short part takes
    // another: 16 of 700 to 8192 keys 63 us against 70 with 256, and 66 to 71 with parts by need.
    const bool tokens = columns <= 32;
    const int64_t items = tokens ? single : single * ceil_div(columns, int64_t(bf ? 128 : kTile));
    const int64_t most = std::min(ceil_div(int64_t(a.Nk), int64_t(tokens ? 256 : 512)), int64_t(64));
    const int64_t want = tokens && !a.lengths ? 256 : 512;
    n.keys = int(std::max(int64_t(1), std::min(most, want / items)));
    n.slots = n.keys * a.B;
    if (shares_slots(a)) n.slots = int(std::max(int64_t(a.B), std::min(most * a.B, want * a.B / items)));
  }
  if (a.Nk > 0 && a.Nq > 0) {
    // dk and dv are summed in parts (heads first, then runs of queries of at least 4 tiles) until there are about 1024
    // work items, so that long and short ones even out. Packed training 2 x 4096: 175 + 16 us in two parts, 275 in one.
    const int64_t items = ceil_div(int64_t(a.Nk), int64_t(kTile)) * single, want = std::max(int64_t(1), 1024 / items);
    const int64_t heads = std::min(int64_t(a.H / a.Hk), want);
    const int64_t tiles = std::min(want / heads, ceil_div(int64_t(a.Nq), int64_t(4 * kTile)));
    n.queries = {int(heads), int(std::max(int64_t(1), std::min(tiles, int64_t(16))))};
  }
  return n;
}
int64_t sequence_forward_parts(const SequenceArgs &a, const SequenceSplits &n) {
  const int64_t rows = int64_t(n.slots) * a.H * a.Nq;
  return n.slots <= a.B ? 0 : align_up(rows, 2) * 8 + align_up(rows * a.Dv, 2) * 4 + (shares_slots(a) ? int64_t(a.B) * 8 : 0);
}
int64_t sequence_backward_parts(const SequenceArgs &a, const SequenceSplits &n) {
  const int64_t count = int64_t(n.queries.heads) * n.queries.tiles;
  return count <= 1 ? 0 : count * a.B * a.Hk * a.Nk * (a.D + a.Dv) * 4;
}

int sequence_forward(const SequenceArgs &a, int dtype, void *memory, hipStream_t s) {
  if (a.B == 0 || a.H == 0 || a.Nq == 0) return XFH_OK;
  XFH_TRY(check_grid(a));
  XFH_TRY(sequence_ranges(a, s));
  const SequenceSplits n = sequence_splits(a, dtype);
  Parts parts{static_cast<float2 *>(memory), nullptr, nullptr, 1, a.B};
  if (n.slots > a.B) {
    const int64_t rows = int64_t(n.slots) * a.H * a.Nq;
    parts.o = reinterpret_cast<float *>(parts.ml + align_up(rows, 2));   // (on 16 bytes)
    if (shares_slots(a)) parts.table = reinterpret_cast<int2 *>(parts.o + align_up(rows * a.Dv, 2));
    else parts.splits = n.keys;
    parts.slots = n.slots;
  }
  if (dtype == XFH_BF16 && sequence_bf16_forward_fits(a)) {
    XFH_TRY(sequence_bf16_forward(a, parts, s));
  } else {
    const int d = std::max(a.D, a.Dv);
    int status = XFH_OK;
#define XFH_SEQ_FORWARD(DP) status = dtype == XFH_BF16 ? launch_forward<bf16, DP>(a, parts, s) : launch_forward<float, DP>(a, parts, s)
    if (d <= 32) XFH_SEQ_FORWARD(32);
    else if (d <= 64) XFH_SEQ_FORWARD(64);
    else if (d <= 96) XFH_SEQ_FORWARD(96);
    else XFH_SEQ_FORWARD(128);
#undef XFH_SEQ_FORWARD
    if (status != XFH_OK) return status;
  }
  if (n.slots <= a.B) return XFH_OK;
  const bool quads = a.Dv % 4 == 0;
  const dim3 grid(unsigned(ceil_div(int64_t(a.B) * a.H * a.Nq * (quads ? a.Dv / 4 : a.Dv), int64_t(256))));
  if (dtype == XFH_BF16) {
    if (quads) join_kernel<bf16, 4><<<grid, 256, 0, s>>>(a, parts);
    else join_kernel<bf16, 1><<<grid, 256, 0, s>>>(a, parts);
  } else {
    if (quads) join_kernel<float, 4><<<grid, 256, 0, s>>>(a, parts);
    else join_kernel<float, 1><<<grid, 256, 0, s>>>(a, parts);
  }
  return check_launch("sequence_attention");
}

int64_t sequence_slope_part(int64_t B, int64_t H, int64_t Nq) { return H * B * Nq; }

int sequence_backward(const SequenceArgs &a, int dtype, void *memory, float *dslopes, hipStream_t s) {
  float *parts = static_cast<float *>(memory);
  if (a.B > 0 && a.Hk > 0) {
    XFH_TRY(check_grid(a));
    XFH_TRY(sequence_ranges(a, s));
    const Splits splits = sequence_splits(a, dtype).queries;
    const int d = std::max(a.D, a.Dv), count = splits.heads * splits.tiles;
    int status = XFH_OK;
#define XFH_SEQ_BACKWARD(DP) \
  status = dtype == XFH_BF16 ? launch_backward<bf16, DP>(a, splits, parts, s) : launch_backward<float, DP>(a, splits, parts, s)
    if (dtype == XFH_BF16 && sequence_bf16_backward_fits(a)) status = sequence_bf16_backward(a, splits, parts, s);
    else if (d <= 32) XFH_SEQ_BACKWARD(32);
    else if (d <= 64) XFH_SEQ_BACKWARD(64);
    else if (d <= 96) XFH_SEQ_BACKWARD(96);
    else XFH_SEQ_BACKWARD(128);
#undef XFH_SEQ_BACKWARD
    if (status != XFH_OK) return status;
    if (count > 1 && (a.dk || a.dv)) {
      const bool quads = a.D % 4 == 0 && a.Dv % 4 == 0;
      const dim3 grid(unsigned(ceil_div(int64_t(a.B) * a.Hk * a.Nk * ((a.D + a.Dv) / (quads ? 4 : 1)), int64_t(256))));
      if (dtype == XFH_BF16) {
        if (quads) dkv_join_kernel<bf16, 4><<<grid, 256, 0, s>>>(a, count, parts);
        else dkv_join_kernel<bf16, 1><<<grid, 256, 0, s>>>(a, count, parts);
      } else {
        if (quads) dkv_join_kernel<float, 4><<<grid, 256, 0, s>>>(a, count, parts);
        else dkv_join_kernel<float, 1><<<grid, 256, 0, s>>>(a, count, parts);
      }
      XFH_TRY(check_launch("sequence_attention_backward"));
    }
  }
  if (!dslopes || a.H == 0) return XFH_OK;
  dslopes_kernel<<<dim3(unsigned(a.H)), 256, 0, s>>>(a.slope_part, int64_t(a.B) * a.Nq, dslopes);
  return check_launch("sequence_attention_backward");
}

}  // namespace xfh
