// Sequence attention in bf16 on 32x32x16 MFMAs (sequence_bf16.h): forward, dq, dk and dv.
//
// Forward and dq: the columns of a workgroup are 128 queries of the heads that share a key head, query by
// query (column c = query c / G, head c % G of the group of G): the heads of one query read the same
// keys, and a few queries fill a tile. A wavefront owns 32 of them, with K and V tiles shared.
// dk and dv: the columns are 64 keys, each 32 of them with two wavefronts that take turns at the queries (half
// a tile each); the loop goes over the heads of the group and their queries.
//
// Tiles are brought to LDS by direct loads, one ahead of the one in use (two stages, one barrier a tile).
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "sequence_bf16.h"

namespace xfh {
namespace {

using namespace seq;

constexpr int kColumns = 128;                            // columns of a workgroup (32 per wavefront)
constexpr float kSlack = 8.0f;                           // log 2 units that a score may exceed the maximum in use
constexpr float kLowest = -3.402823466e38f;              // running maximum before the first key

// One wavefront's 64 keys of a tile: scores, running maximum and sum, o += P V. The maximum in use is
// raised (and o and l scaled) only when a score exceeds it by kSlack, so weights are at most 2^kSlack.
template <class D, int MODE, bool STRICT, int ROWS>
__device__ __forceinline__ void forward_tile(const SequenceArgs &a, const Lane<D> &ln, const bf16 *kt, const bf16 *vt,
                                             const bf16x8 (&qf)[D::KS], const Score<MODE> &score, int b, int k0, int n,
                                             bool whole, const Row &row, Marks &marks, float &m, float &l,
                                             f32x16 (&o)[D::DT]) {
  constexpr int RT = ROWS / 32;
  f32x16 w[RT];
  uint32_t seen[RT];
  float top = kLowest;
  if (!whole) mark_keys(a, b, k0, n, marks);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) w[rt] = ln.product(kt, rt, qf);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if constexpr (MODE != 0) {
      const float gap = float(row.pos - k0 - rt * 32 - 4 * ln.half);
#pragma unroll
      for (int r = 0; r < 16; ++r) w[rt][r] = score(w[rt][r], gap - float(row_of_register(r)));
    }
    seen[rt] = 0xffff;
    if (!whole) seen[rt] = hide_keys(a, marks, rt, k0, ln.half, row, w[rt]);
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, w[rt][r]);
  }
  top = score.in_log2(top);
  if (__ballot(top > m + kSlack)) {
    top = fmaxf(top, other_half(top));
    const float next = top > m + kSlack ? top : m;       // (of this column alone: another's scores change no bit of it)
    const float alpha = __builtin_amdgcn_exp2f(m - next);
    m = next;
    l *= alpha;
#pragma unroll
    for (int t = 0; t < D::DT; ++t) o[t] *= alpha;
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      w[rt][r] = score.weight(w[rt][r], m);
      l += w[rt][r];
    }
#pragma unroll
  for (int kk = 0; kk < 2 * RT; ++kk)
    ln.template accumulate<STRICT, true>(vt, kk, weights(w[kk / 2], 8 * (kk & 1)), weights_seen(seen[kk / 2], 8 * (kk & 1)), o);
}

template <class D> __device__ __forceinline__ bool any_bad(const f32x16 (&o)[D::DT]) {
  bool bad = false;
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad |= !(fabsf(o[t][r]) < INFINITY);
  return bad;
}

// A column's result: dims 32 t + 8 j + 4 half .. + 3, four at a time.
template <class D>
__device__ __forceinline__ void store_column(bf16 *out, int dim, const f32x16 (&o)[D::DT], float scale, int half) {
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = t * 32 + 8 * j + 4 * half;
      if (d < dim) {
        bf16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<bf16>(o[t][4 * j + e] * scale);
        *reinterpret_cast<bf16x4 *>(out + d) = v;
      }
    }
}

// Where the parts of a forward pass whose keys are split go: o [splits][B Hk][columns][Dv], (m, l) beside it.
struct Parts {
  float *o;
  float2 *ml;
  int splits;
};

template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void forward_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *lds, const Loader<D, 4> &kl,
                                             const Loader<D, 4> &vl, const bf16x8 (&qf)[D::KS], const Score<MODE> &score,
                                             int b, int first, int end, int n, const Span &block, const Span &wave,
                                             const Row &row, Marks &marks, float &m, float &l, f32x16 (&o)[D::DT]) {
  constexpr int TILE = kTile * D::DL;
  m = kLowest;
  l = 0.f;
#pragma unroll
  for (int t = 0; t < D::DT; ++t) o[t] = zeros16();
  const auto test = [&](int tile) { return key_tile_needs(a, b, tile, block, wave); };
  Walk walk(first, end);
  Step now = walk.next(test);
  if (now.tile >= 0) {
    kl.load(lds, now.tile * kTile);
    vl.load(lds + TILE, now.tile * kTile);
  }
  int stage = 0;
  while (now.tile >= 0) {
    wait_loads();
    ring_barrier();                                      // the tile has landed; the other stage is no longer read
    const Step then = walk.next(test);
    bf16 *spare = lds + (stage ^ 1) * 2 * TILE;
    if (then.tile >= 0) {
      kl.load(spare, then.tile * kTile);
      vl.load(spare + TILE, then.tile * kTile);
    }
    if (now.mine) {
      const bf16 *kt = lds + stage * 2 * TILE;
      forward_tile<D, MODE, STRICT, kTile>(a, ln, kt, kt + TILE, qf, score, b, now.tile * kTile, n, now.whole, row, marks, m, l, o);
    }
    now = then;
    stage ^= 1;
  }
}

template <class D, int MODE>
__global__ __launch_bounds__(256, 2) void forward_bf16_kernel(SequenceArgs a, int blocks, Parts parts) {
  constexpr int TILE = kTile * D::DL;
  __shared__ __attribute__((aligned(1024))) bf16 lds[4 * TILE];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  const int group = a.H / a.Hk, columns = group * a.Nq;
  const int hk = blockIdx.x % a.Hk;
  int rest = blockIdx.x / a.Hk;
  const int split = rest % parts.splits;
  rest /= parts.splits;
  const int blk = blocks - 1 - rest % blocks, b = rest / blocks;   // the last queries, which see most under a causal mask, first
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane<D> ln;
  const int c0 = blk * kColumns, c1 = min(c0 + kColumns, columns) - 1;
  const int w0 = c0 + wave * 32, w1 = min(w0 + 31, c1);
  const int c = w0 + ln.col;
  const bool valid = c < columns;
  const int i = valid ? c / group : a.Nq, h = hk * group + (valid ? c % group : 0);
  const Place place = place_of(a, b);
  const Span block = span_of(a, place, b, c0 / group, c1 / group);
  const Span mine = w0 <= w1 ? span_of(a, place, b, w0 / group, w1 / group) : span_of(a, place, b, 0, -1);
  const Row row = row_of(a, place, b, i);
  const Score<MODE> score(a, h);
  bf16x8 qf[D::KS];
  own_row<D>(qf, static_cast<const bf16 *>(a.q) + b * a.qs[0] + h * a.qs[1] + i * a.qs[2], a.D, valid, ln.half);
  const Loader<D, 4> kl(static_cast<const bf16 *>(a.k) + b * a.ks[0] + hk * a.ks[1], a.ks[2], place.n, a.D, wave);
  const Loader<D, 4> vl(static_cast<const bf16 *>(a.v) + b * a.vs[0] + hk * a.vs[1], a.vs[2], place.n, a.Dv, wave);
  int end = (block.high + kTile - 1) / kTile, first = 0;
  if (parts.splits > 1) {
    const int per = (end + parts.splits - 1) / parts.splits;
    first = min(split * per, end);
    end = min(first + per, end);
  }
  f32x16 o[D::DT];
  float m, l;
  forward_walk<D, MODE, false>(a, ln, lds, kl, vl, qf, score, b, first, end, place.n, block, mine, row, marks[wave], m, l, o);
  if (__syncthreads_or(valid && any_bad<D>(o)))
    forward_walk<D, MODE, true>(a, ln, lds, kl, vl, qf, score, b, first, end, place.n, block, mine, row, marks[wave], m, l, o);
  l += other_half(l);
  if (!valid) return;
  if (parts.splits > 1) {
    const int64_t at = (int64_t(split) * a.B * a.Hk + int64_t(b) * a.Hk + hk) * columns + c;
    if (ln.half == 0) parts.ml[at] = make_float2(m, l);
    float *out = parts.o + at * a.Dv;
#pragma unroll
    for (int t = 0; t < D::DT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = t * 32 + 8 * j + 4 * ln.half;
        if (d < a.Dv)
          *reinterpret_cast<float4 *>(out + d) = make_float4(o[t][4 * j], o[t][4 * j + 1], o[t][4 * j + 2], o[t][4 * j + 3]);
      }
    return;
  }
  store_column<D>(static_cast<bf16 *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2], a.Dv, o, l == 0.f ? 0.f : 1.0f / l, ln.half);
  if (a.lse && ln.half == 0) a.lse[(int64_t(b) * a.H + h) * a.Nq + i] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// At most 32 columns (single tokens): the four wavefronts of a workgroup share the columns and take tiles of
// 32 keys each, in LDS of their own (no barrier until their results are joined).
template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void token_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *lds, const Loader<D, 1, 32> &kl,
                                           const Loader<D, 1, 32> &vl, const bf16x8 (&qf)[D::KS], const Score<MODE> &score,
                                           int b, int first, int end, int n, const Span &span, const Row &row, Marks &marks,
                                           float &m, float &l, f32x16 (&o)[D::DT]) {
  constexpr int TILE = 32 * D::DL;
  m = kLowest;
  l = 0.f;
#pragma unroll
  for (int t = 0; t < D::DT; ++t) o[t] = zeros16();
  if (first < end) {
    kl.load(lds, first * 32);
    vl.load(lds + TILE, first * 32);
  }
  int stage = 0;
  for (int tile = first; tile < end; tile += 4) {
    wait_loads();
    bf16 *spare = lds + (stage ^ 1) * 2 * TILE;
    if (tile + 4 < end) {
      kl.load(spare, (tile + 4) * 32);
      vl.load(spare + TILE, (tile + 4) * 32);
    }
    bool need = true, whole = tile * 32 + 32 <= span.low;
    if (a.documents) {
      const Range r = static_cast<const Range *>(a.ranges)[int64_t(b) * a.tiles + tile / 2];
      need = overlap(r, span.range);
      whole = whole && same_document(r, span.range);
    }
    const bf16 *kt = lds + stage * 2 * TILE;
    if (need) forward_tile<D, MODE, STRICT, 32>(a, ln, kt, kt + TILE, qf, score, b, tile * 32, n, whole, row, marks, m, l, o);
    // The loads of the step after next go to this stage: every read of it has to be done.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stage ^= 1;
  }
}

template <class D, int MODE>
__global__ __launch_bounds__(256, 1) void token_bf16_kernel(SequenceArgs a, int blocks, Parts parts) {
  constexpr int TILE = 32 * D::DL, PITCH = D::DT * 32 + 4;
  __shared__ __attribute__((aligned(1024))) bf16 lds[4][4 * TILE];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  __shared__ float2 ml[4][32];
  static_assert(sizeof(lds) >= 4 * 32 * PITCH * 4 || D::DL < 128, "joined in the tiles' memory");
  __shared__ float joined[D::DL < 128 ? 4 * 32 * PITCH : 1];
  float *parts_o = D::DL < 128 ? joined : reinterpret_cast<float *>(&lds[0][0]);
  const int group = a.H / a.Hk, columns = group * a.Nq;
  const int hk = blockIdx.x % a.Hk;
  int rest = blockIdx.x / a.Hk;
  const int split = rest % parts.splits, b = rest / parts.splits;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane<D> ln;
  const int c = ln.col;
  const bool valid = c < columns;
  const int i = valid ? c / group : a.Nq, h = hk * group + (valid ? c % group : 0);
  const Place place = place_of(a, b);
  const Span span = span_of(a, place, b, 0, a.Nq - 1);
  const Row row = row_of(a, place, b, i);
  const Score<MODE> score(a, h);
  bf16x8 qf[D::KS];
  own_row<D>(qf, static_cast<const bf16 *>(a.q) + b * a.qs[0] + h * a.qs[1] + i * a.qs[2], a.D, valid, ln.half);
  const Loader<D, 1, 32> kl(static_cast<const bf16 *>(a.k) + b * a.ks[0] + hk * a.ks[1], a.ks[2], place.n, a.D, 0);
  const Loader<D, 1, 32> vl(static_cast<const bf16 *>(a.v) + b * a.vs[0] + hk * a.vs[1], a.vs[2], place.n, a.Dv, 0);
  const int tiles = (span.high + 31) / 32, per = (tiles + parts.splits - 1) / parts.splits;
  const int first = min(split * per, tiles), end = min(first + per, tiles);
  f32x16 o[D::DT];
  float m, l;
  token_walk<D, MODE, false>(a, ln, lds[wave], kl, vl, qf, score, b, first + wave, end, place.n, span, row, marks[wave], m, l, o);
  if (__syncthreads_or(valid && any_bad<D>(o)))
    token_walk<D, MODE, true>(a, ln, lds[wave], kl, vl, qf, score, b, first + wave, end, place.n, span, row, marks[wave], m, l, o);
  l += other_half(l);
  __syncthreads();
  if (ln.half == 0) ml[wave][c] = make_float2(m, l);
  float *mine = parts_o + (wave * 32 + c) * PITCH;
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) mine[t * 32 + row_of_register(r) + 4 * ln.half] = o[t][r];
  __syncthreads();
  for (int at = threadIdx.x; at < columns * a.Dv; at += 256) {
    const int col = at / a.Dv, d = at % a.Dv;
    float top = ml[0][col].x;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[w][col].x);
    float sum = 0.f, value = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[w][col].x - top);
      sum += f * ml[w][col].y;
      value += f * parts_o[(w * 32 + col) * PITCH + d];
    }
    const int query = col / group, head = hk * group + col % group;
    if (parts.splits > 1) {
      const int64_t p = (int64_t(split) * a.B * a.Hk + int64_t(b) * a.Hk + hk) * columns + col;
      parts.o[p * a.Dv + d] = value;
      if (d == 0) parts.ml[p] = make_float2(top, sum);
    } else {
      static_cast<bf16 *>(a.out)[b * a.os[0] + head * a.os[1] + query * a.os[2] + d] = bf16(sum == 0.f ? 0.f : value / sum);
      if (a.lse && d == 0)
        a.lse[(int64_t(b) * a.H + head) * a.Nq + query] = sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
    }
  }
}

// Joins the parts of split keys, in their order: a thread per 4 elements (Dv is a multiple of 8 here).
__global__ __launch_bounds__(256) void join_kernel(SequenceArgs a, Parts parts) {
  const int group = a.H / a.Hk, columns = group * a.Nq, quads = a.Dv / 4;
  const int64_t total = int64_t(a.B) * a.Hk * columns, at = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= total * quads) return;
  const int64_t column = at / quads;
  const int d = int(at - column * quads) * 4;
  float top = kLowest;
  for (int s = 0; s < parts.splits; ++s) top = fmaxf(top, parts.ml[s * total + column].x);
  float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < parts.splits; ++s) {
    const float2 p = parts.ml[s * total + column];
    const float4 o = *reinterpret_cast<const float4 *>(parts.o + (s * total + column) * a.Dv + d);
    const float f = __builtin_amdgcn_exp2f(p.x - top);
    sum += f * p.y;
    v[0] += f * o.x; v[1] += f * o.y; v[2] += f * o.z; v[3] += f * o.w;
  }
  const int c = int(column % columns), bk = int(column / columns), hk = bk % a.Hk, b = bk / a.Hk;
  const int i = c / group, h = hk * group + c % group;
  bf16 *out = static_cast<bf16 *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2] + d;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  bf16x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = static_cast<bf16>(v[e] * inv);
  *reinterpret_cast<bf16x4 *>(out) = r;
  if (a.lse && d == 0) a.lse[(int64_t(b) * a.H + h) * a.Nq + i] = sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
}

// ------------------------------------------------------------------------------ dq

struct SlopeSums { float far, error, far_error; };       // sum P |gap|, sum P (dP - delta), sum P (dP - delta) |gap|

template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void dq_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *lds, const Loader<D, 4> &kl,
                                        const Loader<D, 4> &vl, const bf16x8 (&qf)[D::KS], const bf16x8 (&gf)[D::KS],
                                        const Score<MODE> &score, int b, int end, int n, const Span &block,
                                        const Span &wave, const Row &row, Marks &marks, float lse, float delta,
                                        f32x16 (&dq)[D::DT], SlopeSums &sums) {
  constexpr int TILE = kTile * D::DL;
  sums = SlopeSums{0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < D::DT; ++t) dq[t] = zeros16();
  const auto test = [&](int tile) { return key_tile_needs(a, b, tile, block, wave); };
  Walk walk(0, end);
  Step now = walk.next(test);
  if (now.tile >= 0) {
    kl.load(lds, now.tile * kTile);
    vl.load(lds + TILE, now.tile * kTile);
  }
  int stage = 0;
  while (now.tile >= 0) {
    wait_loads();
    ring_barrier();
    const Step then = walk.next(test);
    bf16 *spare = lds + (stage ^ 1) * 2 * TILE;
    if (then.tile >= 0) {
      kl.load(spare, then.tile * kTile);
      vl.load(spare + TILE, then.tile * kTile);
    }
    if (now.mine) {
      const bf16 *kt = lds + stage * 2 * TILE, *vt = kt + TILE;
      if (!now.whole) mark_keys(a, b, now.tile * kTile, n, marks);
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const int k0 = now.tile * kTile + rt * 32;
        f32x16 w = ln.product(kt, rt, qf), dp = ln.product(vt, rt, gf), bent;
        const float gap = float(row.pos - k0 - 4 * ln.half);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float f = 1.f;
          w[r] = score(w[r], gap - float(row_of_register(r)), &f);
          if constexpr (Score<MODE>::CAP) bent[r] = f;
        }
        uint32_t seen = 0xffff;
        if (!now.whole) seen = hide_keys(a, marks, rt, now.tile * kTile, ln.half, row, w);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = score.weight(w[r], lse), error = dp[r] - delta;
          // A hidden pair's dP may be anything: its product is not taken.
          float ds = now.whole || p != 0.f ? p * error : 0.f;
          if constexpr (STRICT) ds = (seen >> r) & 1 ? ds : 0.f;
          if constexpr (Score<MODE>::SLOPE) {
            const float away = fabsf(gap - float(row_of_register(r)));
            if (a.slope_part) {
              sums.far = __builtin_fmaf(p, away, sums.far);
              sums.error += ds;
              sums.far_error = __builtin_fmaf(ds, away, sums.far_error);
            }
          }
          w[r] = Score<MODE>::CAP ? ds * bent[r] : ds;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
          ln.template accumulate<STRICT, false>(kt, 2 * rt + s, weights(w, 8 * s), weights_seen(seen, 8 * s), dq);
      }
    }
    now = then;
    stage ^= 1;
  }
}

template <class D, int MODE>
__global__ __launch_bounds__(256, 2) void dq_bf16_kernel(SequenceArgs a, int blocks) {
  constexpr int TILE = kTile * D::DL;
  __shared__ __attribute__((aligned(1024))) bf16 lds[4 * TILE];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  const int group = a.H / a.Hk, columns = group * a.Nq;
  const int hk = blockIdx.x % a.Hk, rest = blockIdx.x / a.Hk, blk = blocks - 1 - rest % blocks, b = rest / blocks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane<D> ln;
  const int c0 = blk * kColumns, c1 = min(c0 + kColumns, columns) - 1;
  const int w0 = c0 + wave * 32, w1 = min(w0 + 31, c1);
  const int c = w0 + ln.col;
  const bool valid = c < columns;
  const int i = valid ? c / group : a.Nq, h = hk * group + (valid ? c % group : 0);
  const Place place = place_of(a, b);
  const Span block = span_of(a, place, b, c0 / group, c1 / group);
  const Span mine = w0 <= w1 ? span_of(a, place, b, w0 / group, w1 / group) : span_of(a, place, b, 0, -1);
  const Row row = row_of(a, place, b, i);
  const Score<MODE> score(a, h);
  bf16x8 qf[D::KS], gf[D::KS];
  own_row<D>(qf, static_cast<const bf16 *>(a.q) + b * a.qs[0] + h * a.qs[1] + i * a.qs[2], a.D, valid, ln.half);
  own_row<D>(gf, static_cast<const bf16 *>(a.dout) + b * a.gs[0] + h * a.gs[1] + i * a.gs[2], a.Dv, valid, ln.half);
  const int64_t at = (int64_t(b) * a.H + h) * a.Nq + i;
  float delta = 0.f;
  {
    bf16x8 of[D::KS];
    own_row<D>(of, static_cast<const bf16 *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2], a.Dv, valid, ln.half);
#pragma unroll
    for (int ks = 0; ks < D::KS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(static_cast<float>(of[ks][e]), static_cast<float>(gf[ks][e]), delta);
  }
  delta += other_half(delta);
  const float lse = valid ? a.lse[at] : INFINITY;
  if (valid && ln.half == 0) a.delta[at] = delta;
  const Loader<D, 4> kl(static_cast<const bf16 *>(a.k) + b * a.ks[0] + hk * a.ks[1], a.ks[2], place.n, a.D, wave);
  const Loader<D, 4> vl(static_cast<const bf16 *>(a.v) + b * a.vs[0] + hk * a.vs[1], a.vs[2], place.n, a.Dv, wave);
  const int end = (block.high + kTile - 1) / kTile;
  f32x16 dq[D::DT];
  SlopeSums sums;
  dq_walk<D, MODE, false>(a, ln, lds, kl, vl, qf, gf, score, b, end, place.n, block, mine, row, marks[wave], lse, delta, dq, sums);
  if (__syncthreads_or(valid && any_bad<D>(dq)))
    dq_walk<D, MODE, true>(a, ln, lds, kl, vl, qf, gf, score, b, end, place.n, block, mine, row, marks[wave], lse, delta, dq, sums);
  if (valid)
    store_column<D>(static_cast<bf16 *>(a.dq) + b * a.dqs[0] + h * a.dqs[1] + i * a.dqs[2], a.D, dq, a.scale, ln.half);
  if constexpr (Score<MODE>::SLOPE) {
    if (!a.slope_part) return;
    sums.far += other_half(sums.far);
    sums.error += other_half(sums.error);
    sums.far_error += other_half(sums.far_error);
    // One part per query and head: slope_part [H][B][Nq].
    if (valid && ln.half == 0) a.slope_part[(int64_t(h) * a.B + b) * a.Nq + i] = -(sums.far_error - sums.error * sums.far);
  }
}

// ------------------------------------------------------------------------------ dk, dv

// Bounds and documents of 32 queries (i0 ..), a lane each.
__device__ __forceinline__ void mark_queries(const SequenceArgs &a, const Place &place, int b, int i0, Marks &marks) {
  const int at = threadIdx.x & 31;
  const Row row = row_of(a, place, b, i0 + at);
  marks_written();                                       // (the tile before is done with them)
  marks.limit[at] = row.limit;
  marks.document[at] = row.document;
  marks_written();
}
// Scores of hidden pairs of one key column become -infinity.
__device__ __forceinline__ uint32_t hide_queries(const Marks &marks, int half, int key, int document, f32x16 &w) {
  uint32_t seen = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int4 limits = *reinterpret_cast<const int4 *>(marks.limit + 8 * j + 4 * half);
    const int4 ids = *reinterpret_cast<const int4 *>(marks.document + 8 * j + 4 * half);
    const int limit[4] = {limits.x, limits.y, limits.z, limits.w}, id[4] = {ids.x, ids.y, ids.z, ids.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool see = (key < limit[e]) & (id[e] == document);
      w[4 * j + e] = see ? w[4 * j + e] : -INFINITY;
      seen |= see ? 1u << (4 * j + e) : 0u;
    }
  }
  return seen;
}

constexpr int kKeys = 64;                                // keys of a workgroup: 2 groups of 32, each with 2 wavefronts

// One wavefront: 32 keys from kw on, and of each tile of 64 queries the 32 from 32 rt on.
template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void dkv_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *lds, float *stats, Marks &marks,
                                         const bf16x8 (&kf)[D::KS], const bf16x8 (&vf)[D::KS], int b, int hk, int wave, int kb,
                                         int kw, int rt, int key, int document, const Place &place, f32x16 (&dk)[D::DT],
                                         f32x16 (&dv)[D::DT]) {
  constexpr int TILE = kTile * D::DL;
  const int group = a.H / a.Hk, qtiles = (a.Nq + kTile - 1) / kTile;
#pragma unroll
  for (int t = 0; t < D::DT; ++t) {
    dk[t] = zeros16();
    dv[t] = zeros16();
  }
  Range range{0x7fffffff, -1, 0, 0};
  if (a.documents) range = static_cast<const Range *>(a.ranges)[int64_t(b) * a.tiles + kb / kTile];
  const auto test = [&](int tile) {
    const int i0 = tile * kTile + rt * 32, i1 = min(i0 + 32, a.Nq) - 1, last = min(tile * kTile + kTile, a.Nq) - 1;
    Needs n{limit_of(a, place, last) > kb, i0 <= i1 && limit_of(a, place, max(i1, 0)) > kw,
            i0 + 32 <= a.Nq && limit_of(a, place, i0) >= kw + 32};
    if (a.documents && n.block) {
      const Range r = query_range(a, place, b, tile * kTile, last);
      n.block = overlap(r, range);
      n.whole = n.whole && same_document(r, range);
    }
    return n;
  };
  for (int g = 0; g < group; ++g) {
    const int h = hk * group + g;
    const Score<MODE> score(a, h);
    const Loader<D, 4> ql(static_cast<const bf16 *>(a.q) + b * a.qs[0] + h * a.qs[1], a.qs[2], a.Nq, a.D, wave);
    const Loader<D, 4> gl(static_cast<const bf16 *>(a.dout) + b * a.gs[0] + h * a.gs[1], a.gs[2], a.Nq, a.Dv, wave);
    const int64_t at = (int64_t(b) * a.H + h) * a.Nq;
    const auto load = [&](int tile, int stage) {
      bf16 *to = lds + stage * 2 * TILE;
      ql.load(to, tile * kTile);
      gl.load(to + TILE, tile * kTile);
      if (wave < 2) {                                    // 64 lse, 64 delta (beyond the end: the last one's)
        const float *from = (wave ? a.delta : a.lse) + at + min(tile * kTile + int(threadIdx.x & 63), a.Nq - 1);
        __builtin_amdgcn_global_load_lds((global_void *)from, (lds_void *)(stats + (stage * 2 + wave) * kTile), 4, 0, 0);
      }
    };
    Walk walk(0, qtiles);
    Step now = walk.next(test);
    ring_barrier();                                      // (the last head's tiles are no longer read)
    if (now.tile >= 0) load(now.tile, 0);
    int stage = 0;
    while (now.tile >= 0) {
      wait_loads();
      ring_barrier();
      const Step then = walk.next(test);
      if (then.tile >= 0) load(then.tile, stage ^ 1);
      if (now.mine) {
        const bf16 *qt = lds + stage * 2 * TILE, *gt = qt + TILE;
        const float *lses = stats + stage * 2 * kTile + rt * 32, *deltas = lses + kTile;
        const int i0 = now.tile * kTile + rt * 32;
        if (!now.whole) mark_queries(a, place, b, i0, marks);
        f32x16 w = ln.product(qt, rt, kf), dp = ln.product(gt, rt, vf), bent;
        const float gap = float(i0 + place.shift + 4 * ln.half - key);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float f = 1.f;
          w[r] = score(w[r], gap + float(row_of_register(r)), &f);
          if constexpr (Score<MODE>::CAP) bent[r] = f;
        }
        uint32_t seen = 0xffff;
        if (!now.whole) seen = hide_queries(marks, ln.half, key, document, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 lse = *reinterpret_cast<const f32x4 *>(lses + 8 * j + 4 * ln.half);
          const f32x4 delta = *reinterpret_cast<const f32x4 *>(deltas + 8 * j + 4 * ln.half);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * j + e;
            const bool see = now.whole || ((seen >> r) & 1);
            const float p = see ? score.weight(w[r], lse[e]) : 0.f;
            float ds = see ? p * (dp[r] - delta[e]) : 0.f;
            if constexpr (Score<MODE>::CAP) ds *= bent[r];
            w[r] = p;
            dp[r] = ds;
          }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const bf16x8 sf = weights_seen(seen, 8 * s);
          ln.template accumulate<STRICT, false>(gt, 2 * rt + s, weights(w, 8 * s), sf, dv);
          ln.template accumulate<STRICT, false>(qt, 2 * rt + s, weights(dp, 8 * s), sf, dk);
        }
      }
      now = then;
      stage ^= 1;
    }
  }
}

template <class D, int MODE>
__global__ __launch_bounds__(256, 2) void dkv_bf16_kernel(SequenceArgs a, int blocks) {
  constexpr int TILE = kTile * D::DL, JOIN = 2 * 2 * D::DT * 16 * 64;   // floats: 2 key groups, dk and dv
  __shared__ __attribute__((aligned(1024))) unsigned char memory[JOIN * 4 > 8 * TILE ? JOIN * 4 : 8 * TILE];
  __shared__ __attribute__((aligned(1024))) float stats[4 * kTile];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  bf16 *lds = reinterpret_cast<bf16 *>(memory);
  const int hk = blockIdx.x % a.Hk, rest = blockIdx.x / a.Hk, blk = rest % blocks, b = rest / blocks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rt = wave >> 1;
  const Lane<D> ln;
  const Place place = place_of(a, b);
  const int kb = blk * kKeys, kw = kb + (wave & 1) * 32, key = kw + ln.col;
  const bool valid = key < place.n;
  bf16x8 kf[D::KS], vf[D::KS];
  own_row<D>(kf, static_cast<const bf16 *>(a.k) + b * a.ks[0] + hk * a.ks[1] + key * a.ks[2], a.D, valid, ln.half);
  own_row<D>(vf, static_cast<const bf16 *>(a.v) + b * a.vs[0] + hk * a.vs[1] + key * a.vs[2], a.Dv, valid, ln.half);
  int document = 0;                                      // (as row_of has it without documents)
  if (a.documents) document = valid ? a.documents[int64_t(b) * a.documents_stride + key] : -1;
  f32x16 dk[D::DT], dv[D::DT];
  dkv_walk<D, MODE, false>(a, ln, lds, stats, marks[wave], kf, vf, b, hk, wave, kb, kw, rt, key, document, place, dk, dv);
  if (__syncthreads_or(valid && (any_bad<D>(dk) || any_bad<D>(dv))))
    dkv_walk<D, MODE, true>(a, ln, lds, stats, marks[wave], kf, vf, b, hk, wave, kb, kw, rt, key, document, place, dk, dv);
  __syncthreads();
  // The wavefront of the tiles' second halves hands its sums to that of the first.
  float *join = reinterpret_cast<float *>(memory) + (wave & 1) * (JOIN / 2) + (threadIdx.x & 63);
  if (rt) {
#pragma unroll
    for (int t = 0; t < D::DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        join[(t * 16 + r) * 64] = dk[t][r];
        join[((D::DT + t) * 16 + r) * 64] = dv[t][r];
      }
  }
  __syncthreads();
  if (rt || key >= a.Nk) return;
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {                       // beyond the length: zeros
      dk[t][r] = valid ? dk[t][r] + join[(t * 16 + r) * 64] : 0.f;
      dv[t][r] = valid ? dv[t][r] + join[((D::DT + t) * 16 + r) * 64] : 0.f;
    }
  store_column<D>(static_cast<bf16 *>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2], a.D, dk, a.scale, ln.half);
  store_column<D>(static_cast<bf16 *>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2], a.Dv, dv, 1.f, ln.half);
}

// ------------------------------------------------------------------------------ launches

int mode_of(const SequenceArgs &a) { return (a.cap > 0.f ? 1 : 0) | (a.slopes || (a.cap <= 0.f && a.scale <= 0.f) ? 2 : 0); }

// f(Dim, MODE) for the call's head dims and scores.
template <class D, class F> int with_mode(int mode, F f) {
  switch (mode) {
    case 0: return f(D(), std::integral_constant<int, 0>());
    case 1: return f(D(), std::integral_constant<int, 1>());
    case 2: return f(D(), std::integral_constant<int, 2>());
    default: return f(D(), std::integral_constant<int, 3>());
  }
}
template <class F> int with_dims(const SequenceArgs &a, F f) {
  const int d = std::max(a.D, a.Dv), mode = mode_of(a);
  if (d <= 32) return with_mode<Dim<32, 2, 1>>(mode, f);
  if (d <= 48) return with_mode<Dim<64, 3, 2>>(mode, f);
  if (d <= 64) return with_mode<Dim<64, 4, 2>>(mode, f);
  if (d <= 96) return with_mode<Dim<128, 6, 3>>(mode, f);
  return with_mode<Dim<128, 8, 4>>(mode, f);
}

bool rows_fit(const void *p, const int64_t *strides, int64_t dim, int64_t unit) {
  if (reinterpret_cast<uintptr_t>(p) % (2 * unit) || dim % unit) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] % unit || strides[i] < 0) return false;
  return strides[2] < (int64_t(1) << 24);                // 64 rows of a tile within 32-bit offsets
}

}  // namespace

bool sequence_bf16_forward_fits(const SequenceArgs &a) {
  return rows_fit(a.q, a.qs, a.D, 8) && rows_fit(a.k, a.ks, a.D, 8) && rows_fit(a.v, a.vs, a.Dv, 8) && rows_fit(a.out, a.os, a.Dv, 4) &&
         int64_t(a.H / a.Hk) * a.Nq < (int64_t(1) << 31) - 256;
}
bool sequence_bf16_backward_fits(const SequenceArgs &a) {
  return sequence_bf16_forward_fits(a) && rows_fit(a.out, a.os, a.Dv, 8) && rows_fit(a.dout, a.gs, a.Dv, 8) &&
         rows_fit(a.dq, a.dqs, a.D, 4) && rows_fit(a.dk, a.dks, a.D, 4) && rows_fit(a.dv, a.dvs, a.Dv, 4);
}

int sequence_splits(int64_t B, int64_t H, int64_t Hk, int64_t Nq, int64_t Nk) {
  if (H == 0 || Hk == 0 || B == 0) return 1;
  const int64_t columns = H / Hk * Nq;
  const int64_t items = columns <= 32 ? B * Hk : B * Hk * ceil_div(columns, int64_t(kColumns));
  const int64_t most = columns <= 32 ? ceil_div(Nk, int64_t(256)) : ceil_div(Nk, int64_t(512));
  return int(std::max(int64_t(1), std::min(std::min(most, 512 / items), int64_t(64))));
}

int64_t sequence_parts_bytes(int64_t B, int64_t H, int64_t Nq, int64_t Dv, int splits) {
  return splits <= 1 ? 0 : splits * B * H * Nq * (Dv * 4 + 8);
}

int sequence_bf16_forward(const SequenceArgs &a, void *parts_memory, int splits, hipStream_t s) {
  const int64_t columns = int64_t(a.H / a.Hk) * a.Nq;
  Parts parts{static_cast<float *>(parts_memory), nullptr, splits};
  if (splits > 1) parts.ml = reinterpret_cast<float2 *>(parts.o + splits * int64_t(a.B) * a.H * a.Nq * a.Dv);
  const int64_t blocks = columns <= 32 ? 1 : ceil_div(columns, int64_t(kColumns));
  const dim3 grid(unsigned(blocks * a.Hk * a.B * splits));
  XFH_TRY(with_dims(a, [&](auto dim, auto mode) {
    typedef decltype(dim) D;
    constexpr int MODE = decltype(mode)::value;
    if (columns <= 32) token_bf16_kernel<D, MODE><<<grid, 256, 0, s>>>(a, 1, parts);
    else forward_bf16_kernel<D, MODE><<<grid, 256, 0, s>>>(a, int(blocks), parts);
    return check_launch("sequence_attention");
  }));
  if (splits <= 1) return XFH_OK;
  join_kernel<<<dim3(unsigned(ceil_div(int64_t(a.B) * a.H * a.Nq * (a.Dv / 4), int64_t(256)))), 256, 0, s>>>(a, parts);
  return check_launch("sequence_attention");
}

int sequence_bf16_backward(const SequenceArgs &a, hipStream_t s) {
  const int64_t blocks = ceil_div(int64_t(a.H / a.Hk) * a.Nq, int64_t(kColumns)), kblocks = ceil_div(int64_t(a.Nk), int64_t(kKeys));
  return with_dims(a, [&](auto dim, auto mode) {
    typedef decltype(dim) D;
    constexpr int MODE = decltype(mode)::value;
    if (blocks > 0) dq_bf16_kernel<D, MODE><<<dim3(unsigned(blocks * a.Hk * a.B)), 256, 0, s>>>(a, int(blocks));
    XFH_TRY(check_launch("sequence_attention_backward"));
    if (kblocks > 0) dkv_bf16_kernel<D, MODE><<<dim3(unsigned(kblocks * a.Hk * a.B)), 256, 0, s>>>(a, int(kblocks));
    return check_launch("sequence_attention_backward");
  });
}

}  // namespace xfh
