// Sequence attention in bf16 on 32x32x16 MFMAs (sequence_bf16.h), forward.
//
// The columns of a workgroup are 128 queries of the heads that share a key head, query by query (column c =
// query c / G, head c % G of the group of G): the heads of one query read the same keys, and a few queries
// fill a tile. A wavefront owns 32 of them, with K and V tiles shared. Tiles are brought to LDS by
// direct loads, one ahead of the one in use (two stages, one barrier a tile).
//
// With D = 128 the products are the larger part: 784 TFLOP/s at 2 x 16 heads of 4096 tokens (all pairs), 913 under a causal
// mask at 8192 tokens. With less D the softmax is: 740 TFLOP/s at D = 64, and 5 x 768 tokens of 16 heads of 48 with
// documents and slopes take 42 us, 21 in a form without the exponentials. A cap adds an exponential and a reciprocal
// per score: 8192 tokens, 16 heads on 8, D = 128 take 376 us.
#include "sequence_bf16.h"

namespace xfh {
namespace {

using namespace seq;

constexpr float kSlack = 8.0f;                           // log 2 units that a score may exceed the maximum in use

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
  for (int kk = 0; kk < 2 * RT; ++kk) {
    bf16x8 vf[D::DT];
    ln.transposed_fragments(vt, kk, vf);
    add_product<STRICT, true>(vf, weights(w[kk / 2], 8 * (kk & 1)), weights_seen(seen[kk / 2], 8 * (kk & 1)), o);
  }
}

// The stages are arrays of their own, which the code takes in turns: reads of one are then known not to
// depend on the direct loads in flight to the other (else the compiler waits for these before every read).
template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void forward_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *stage0, bf16 *stage1,
                                             const Loader<D, 4> &kl, const Loader<D, 4> &vl, const bf16x8 (&qf)[D::KS],
                                             const Score<MODE> &score, int b, int first, int end, int n, const Span &block,
                                             const Span &wave, const Row &row, Marks &marks, float &m, float &l,
                                             f32x16 (&o)[D::DT]) {
  constexpr int TILE = kTile * D::DL;
  m = kLowest;
  l = 0.f;
#pragma unroll
  for (int t = 0; t < D::DT; ++t) o[t] = zeros16();
  const auto test = [&](int tile) { return key_tile_needs(a, b, tile, block, wave); };
  Walk walk(first, end);
  Step now = walk.next(test);
  const auto load = [&](bf16 *to, int tile) {
    kl.load(to, tile * kTile);
    vl.load(to + TILE, tile * kTile);
  };
  const auto compute = [&](const bf16 *kt) {
    if (now.mine)
      forward_tile<D, MODE, STRICT, kTile>(a, ln, kt, kt + TILE, qf, score, b, now.tile * kTile, n, now.whole, row, marks, m, l, o);
  };
  if constexpr (STRICT) {                                // rare: one stage will do
    while (now.tile >= 0) {
      ring_barrier();
      load(stage0, now.tile);
      wait_loads();
      ring_barrier();
      compute(stage0);
      now = walk.next(test);
    }
  } else {
    const auto step = [&](bf16 *use, bf16 *spare) {
      wait_loads();
      ring_barrier();                                    // the tile has landed; the other stage is no longer read
      const Step then = walk.next(test);
      if (then.tile >= 0) load(spare, then.tile);
      compute(use);
      now = then;
    };
    if (now.tile >= 0) load(stage0, now.tile);
    while (now.tile >= 0) {
      step(stage0, stage1);
      if (now.tile < 0) break;
      step(stage1, stage0);
    }
  }
}

template <class D, int MODE>
__global__ __launch_bounds__(256, 2) void forward_bf16_kernel(SequenceArgs a, int blocks, Parts parts) {
  constexpr int TILE = kTile * D::DL;
  __shared__ __attribute__((aligned(1024))) bf16 stage0[2 * TILE], stage1[2 * TILE];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  const int group = a.H / a.Hk, columns = group * a.Nq;
  const Part part(a, parts, blocks, blockIdx.x);
  if (part.count == 0) return;
  const int b = part.b, hk = part.hk, blk = part.blk;
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
  if (several(parts)) part.take(first, end);
  f32x16 o[D::DT];
  float m, l;
  forward_walk<D, MODE, false>(a, ln, stage0, stage1, kl, vl, qf, score, b, first, end, place.n, block, mine, row, marks[wave], m, l, o);
  if (__syncthreads_or(valid && any_bad(o)))
    forward_walk<D, MODE, true>(a, ln, stage0, stage1, kl, vl, qf, score, b, first, end, place.n, block, mine, row, marks[wave], m, l, o);
  l += other_half(l);
  if (!valid) return;
  if (several(parts)) {
    const int64_t at = (int64_t(part.slot) * a.Hk + hk) * columns + c;
    if (ln.half == 0) parts.ml[at] = make_float2(m, l);
    if (l == 0.f) return;
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
  store_column(static_cast<bf16 *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2], a.Dv, o, l == 0.f ? 0.f : 1.0f / l, ln.half,
               a.low ? static_cast<bf16 *>(a.low) + ((int64_t(b) * a.H + h) * a.Nq + i) * a.Dv : nullptr);
  if (a.lse && ln.half == 0) a.lse[(int64_t(b) * a.H + h) * a.Nq + i] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// At most 32 columns (single tokens): the four wavefronts of a workgroup share the columns and take tiles of
// 32 keys each, in LDS of their own (no barrier until their results are joined). Bound by reading the cache: 16 sequences
// of 700 to 8192 keys, 32 heads on 8, D = 128, 291 MB in 57 us (5.1 TB/s) and 5 for the join.
template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void token_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *stage0, bf16 *stage1,
                                           const Loader<D, 1, 32> &kl, const Loader<D, 1, 32> &vl, const bf16x8 (&qf)[D::KS],
                                           const Score<MODE> &score, int b, int first, int end, int n, const Span &span,
                                           const Row &row, Marks &marks, float &m, float &l, f32x16 (&o)[D::DT]) {
  constexpr int TILE = 32 * D::DL;
  m = kLowest;
  l = 0.f;
#pragma unroll
  for (int t = 0; t < D::DT; ++t) o[t] = zeros16();
  const auto load = [&](bf16 *to, int tile) {
    kl.load(to, tile * 32);
    vl.load(to + TILE, tile * 32);
  };
  const auto compute = [&](const bf16 *kt, int tile) {
    bool need = true, whole = tile * 32 + 32 <= span.low;
    if (a.documents) {
      const Range r = static_cast<const Range *>(a.ranges)[int64_t(b) * a.tiles + tile / 2];
      need = overlap(r, span.range);
      whole = whole && same_document(r, span.range);
    }
    if (need) forward_tile<D, MODE, STRICT, 32>(a, ln, kt, kt + TILE, qf, score, b, tile * 32, n, whole, row, marks, m, l, o);
    // The next loads go to this stage: every read of it has to be done.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  if constexpr (STRICT) {
    for (int tile = first; tile < end; tile += 4) {
      load(stage0, tile);
      wait_loads();
      compute(stage0, tile);
    }
  } else {
    int tile = first;
    const auto step = [&](bf16 *use, bf16 *spare) {
      wait_loads();
      if (tile + 4 < end) load(spare, tile + 4);
      compute(use, tile);
      tile += 4;
    };
    if (first < end) load(stage0, first);
    while (tile < end) {
      step(stage0, stage1);
      if (tile >= end) break;
      step(stage1, stage0);
    }
  }
}

template <class D, int MODE>
__global__ __launch_bounds__(256, 1) void token_bf16_kernel(SequenceArgs a, Parts parts) {
  constexpr int TILE = 32 * D::DL, PITCH = D::DT * 32 + 4;
  __shared__ __attribute__((aligned(1024))) bf16 stage0[4][2 * TILE], stage1[4][2 * TILE];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  __shared__ float2 ml[4][32];
  static_assert(sizeof(stage0) >= 2 * 32 * PITCH * 4, "two wavefronts' results are joined in a stage");
  const auto joined = [&](int w) { return reinterpret_cast<float *>(w < 2 ? stage0 : stage1) + (w & 1) * 32 * PITCH; };
  const int group = a.H / a.Hk, columns = group * a.Nq;
  const Part part(a, parts, 1, blockIdx.x);
  const int b = part.b, hk = part.hk;
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
  int first, end = (span.high + 31) / 32;
  part.take(first, end);
  f32x16 o[D::DT];
  float m, l;
  token_walk<D, MODE, false>(a, ln, stage0[wave], stage1[wave], kl, vl, qf, score, b, first + wave, end, place.n, span, row, marks[wave], m, l, o);
  if (__syncthreads_or(valid && any_bad(o)))
    token_walk<D, MODE, true>(a, ln, stage0[wave], stage1[wave], kl, vl, qf, score, b, first + wave, end, place.n, span, row, marks[wave], m, l, o);
  l += other_half(l);
  __syncthreads();
  if (ln.half == 0) ml[wave][c] = make_float2(m, l);
  float *mine = joined(wave) + c * PITCH;
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
      value += f * joined(w)[col * PITCH + d];
    }
    const int query = col / group, head = hk * group + col % group;
    if (several(parts)) {
      const int64_t p = (int64_t(part.slot) * a.Hk + hk) * columns + col;
      if (sum != 0.f) parts.o[p * a.Dv + d] = value;
      if (d == 0) parts.ml[p] = make_float2(top, sum);
    } else {
      const float x = sum == 0.f ? 0.f : value / sum;
      const bf16 r = bf16(x);
      static_cast<bf16 *>(a.out)[b * a.os[0] + head * a.os[1] + query * a.os[2] + d] = r;
      if (a.low) static_cast<bf16 *>(a.low)[((int64_t(b) * a.H + head) * a.Nq + query) * a.Dv + d] = bf16(x - static_cast<float>(r));
      if (a.lse && d == 0)
        a.lse[(int64_t(b) * a.H + head) * a.Nq + query] = sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
    }
  }
}

}  // namespace

bool sequence_bf16_forward_fits(const SequenceArgs &a) {
  return rows_fit(a.q, a.qs, a.D, 8) && rows_fit(a.k, a.ks, a.D, 8) && rows_fit(a.v, a.vs, a.Dv, 8) && rows_fit(a.out, a.os, a.Dv, 4) &&
         reinterpret_cast<uintptr_t>(a.low) % 8 == 0 && int64_t(a.H / a.Hk) * a.Nq < (int64_t(1) << 31) - 256;
}

int sequence_bf16_forward(const SequenceArgs &a, const Parts &parts, hipStream_t s) {
  const int64_t columns = int64_t(a.H / a.Hk) * a.Nq;
  const int64_t blocks = columns <= 32 ? 1 : ceil_div(columns, int64_t(kColumns));
  const dim3 grid(unsigned(blocks * a.Hk * parts.slots));
  return with_dims(a, [&](auto dim, auto mode) {
    typedef decltype(dim) D;
    constexpr int MODE = decltype(mode)::value;
    if (columns <= 32) token_bf16_kernel<D, MODE><<<grid, 256, 0, s>>>(a, parts);
    else forward_bf16_kernel<D, MODE><<<grid, 256, 0, s>>>(a, int(blocks), parts);
    return check_launch("sequence_attention");
  });
}

}  // namespace xfh
