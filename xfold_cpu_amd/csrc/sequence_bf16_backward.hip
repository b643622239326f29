// Sequence attention in bf16 on 32x32x16 MFMAs (sequence_bf16.h), backward: dq, dk and dv.
//
// dq: the columns are queries, as in the forward pass. dk and dv: the columns are 64 keys, the loop goes
// over the heads of the group and their queries. Work items of their own with 3 and 4 products, of which 2 are the same,
// in place of one kind with 5: the sums of dq need no atomics, and a call gives the same bits every time.
#include "sequence_bf16.h"

namespace xfh {
namespace {

using namespace seq;

// ------------------------------------------------------------------------------ dq

struct SlopeSums { float all, far, error, far_error; };  // as slope_gradient takes them

template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void dq_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *stage0, bf16 *stage1,
                                        const Loader<D, 4> &kl, const Loader<D, 4> &vl, const bf16x8 (&qf)[D::KS],
                                        const bf16x8 (&gf)[D::KS], const Score<MODE> &score, int b, int end, int n,
                                        const Span &block, const Span &wave, const Row &row, Marks &marks, float lse,
                                        float delta, f32x16 (&dq)[D::DT], SlopeSums &sums) {
  constexpr int TILE = kTile * D::DL;
  sums = SlopeSums{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < D::DT; ++t) dq[t] = zeros16();
  const auto test = [&](int tile) { return key_tile_needs(a, b, tile, block, wave); };
  Walk walk(0, end);
  Step now = walk.next(test);
  const auto load = [&](bf16 *to, int tile) {
    kl.load(to, tile * kTile);
    vl.load(to + TILE, tile * kTile);
  };
  const auto compute = [&](const bf16 *kt) {
    if (!now.mine) return;
    const bf16 *vt = kt + TILE;
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
            sums.all += p;
            sums.far = __builtin_fmaf(p, away, sums.far);
            sums.error += ds;
            sums.far_error = __builtin_fmaf(ds, away, sums.far_error);
          }
        }
        w[r] = Score<MODE>::CAP ? ds * bent[r] : ds;
      }
      // dS in two bf16 pieces: in one, its rounding (relative rms 2^-9, no less than the output's own, and more where
      // the sum over the keys cancels) is most of dq's error: 2.4e-3 to 2.9e-3 of its norm, 1.7e-3 to 2.2e-3 in two. With
      // slopes 5 x 768 tokens take 158 us in place of 154, long runs 4 x 4096 1508 in place of 1350. At D = 128
      // there are no registers for it (error 2.4e-3 to 2.6e-3).
      f32x16 rest;
#pragma unroll
      for (int r = 0; r < 16; ++r) rest[r] = w[r] - static_cast<float>(bf16(w[r]));
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 tf[D::DT];
        ln.transposed_fragments(kt, 2 * rt + s, tf);
        add_product<STRICT, false>(tf, weights(w, 8 * s), weights_seen(seen, 8 * s), dq);
        if constexpr (D::DL <= 64) add_product<STRICT, false>(tf, weights(rest, 8 * s), bf16x8{}, dq);
      }
    }
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
      ring_barrier();
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

// DELTA: dout . out is worked out here and kept for dk and dv; else it is there.
template <class D, int MODE, bool DELTA>
__device__ __forceinline__ void dq_block(const SequenceArgs &a, int blocks, int item, bf16 *stage0, bf16 *stage1, Marks *marks) {
  const int group = a.H / a.Hk, columns = group * a.Nq;
  const int hk = item % a.Hk, rest = item / a.Hk, blk = blocks - 1 - rest % blocks, b = rest / blocks;
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
  if constexpr (DELTA) {
    bf16x8 of[D::KS], lf[D::KS] = {};
    own_row<D>(of, static_cast<const bf16 *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2], a.Dv, valid, ln.half);
    if (a.low) own_row<D>(lf, static_cast<const bf16 *>(a.low) + at * a.Dv, a.Dv, valid, ln.half);
#pragma unroll
    for (int ks = 0; ks < D::KS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        delta = __builtin_fmaf(static_cast<float>(of[ks][e]) + static_cast<float>(lf[ks][e]), static_cast<float>(gf[ks][e]), delta);
    delta += other_half(delta);
    if (valid && ln.half == 0) a.delta[at] = delta;
  } else if (valid) {
    delta = a.delta[at];
  }
  const float lse = valid ? a.lse[at] : INFINITY;
  const Loader<D, 4> kl(static_cast<const bf16 *>(a.k) + b * a.ks[0] + hk * a.ks[1], a.ks[2], place.n, a.D, wave);
  const Loader<D, 4> vl(static_cast<const bf16 *>(a.v) + b * a.vs[0] + hk * a.vs[1], a.vs[2], place.n, a.Dv, wave);
  const int end = (block.high + kTile - 1) / kTile;
  f32x16 dq[D::DT];
  SlopeSums sums;
  dq_walk<D, MODE, false>(a, ln, stage0, stage1, kl, vl, qf, gf, score, b, end, place.n, block, mine, row, marks[wave], lse, delta, dq, sums);
  if (__syncthreads_or(valid && any_bad(dq)))
    dq_walk<D, MODE, true>(a, ln, stage0, stage1, kl, vl, qf, gf, score, b, end, place.n, block, mine, row, marks[wave], lse, delta, dq, sums);
  if (valid)
    store_column(static_cast<bf16 *>(a.dq) + b * a.dqs[0] + h * a.dqs[1] + i * a.dqs[2], a.D, dq, a.scale, ln.half);
  if constexpr (Score<MODE>::SLOPE) {
    if (!a.slope_part) return;
    sums.all += other_half(sums.all);
    sums.far += other_half(sums.far);
    sums.error += other_half(sums.error);
    sums.far_error += other_half(sums.far_error);
    // One part per query and head: slope_part [H][B][Nq].
    if (valid && ln.half == 0) a.slope_part[(int64_t(h) * a.B + b) * a.Nq + i] = slope_gradient(sums.all, sums.far, sums.error, sums.far_error);
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

// Tiles of LDS in use: with two, the next one is on its way during a step. At DL = 128 two would leave room for
// one workgroup per CU; two workgroups with one stage each hide each other's loads.
template <class D> constexpr int kDkvStages = D::DL == 128 ? 1 : 2;

// What the two wavefronts of a key group hand each other: P and dS of 32 queries as B fragments, and, in
// the rare form, the bits of the pairs that are seen.
struct Exchange { bf16x8 p[2][64], ds[2][64]; uint32_t seen[64]; };

// Wavefront (key group kg, part): keys kw .. + 31. Of a tile of 64 queries it works out P and dS of the 32
// from 32 part on, and it owns dims 16 DT part .. of dk and dv (half of them: the sums of a whole
// head dim of 128 take 128 registers, and with the keys' own 64 leave room for one wavefront per SIMD
// only). So it adds its own 32 queries' products, then, behind a barrier, its partner's. 2 x 4096 tokens in 5
// documents, 16 heads on 4, D = 128, causal: 175 us, dq 135. The four dependent products, and the softmax between them,
// leave the matrix cores waiting with two wavefronts per SIMD: 550 to 620 TFLOP/s over the backward pass of 4096 tokens.
template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void dkv_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *stage0, bf16 *stage1, float *stats0,
                                         float *stats1, Exchange *exchange, Marks &marks, const bf16x8 (&kf)[D::KS],
                                         const bf16x8 (&vf)[D::KS], int b, int hk, int wave, int kb, int kw, int part, int key,
                                         int document, const Place &place, const Share &share, f32x16 (&dk)[D::DT / 2],
                                         f32x16 (&dv)[D::DT / 2]) {
  constexpr int TILE = kTile * D::DL, T = D::DT / 2;
  const int group = a.H / a.Hk, lane = threadIdx.x & 63;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    dk[t] = zeros16();
    dv[t] = zeros16();
  }
  Range range{0x7fffffff, -1, 0, 0};
  if (a.documents) range = static_cast<const Range *>(a.ranges)[int64_t(b) * a.tiles + kb / kTile];
  const auto test = [&](int tile) {
    const int i0 = tile * kTile + part * 32, i1 = min(i0 + 32, a.Nq) - 1, last = min(tile * kTile + kTile, a.Nq) - 1;
    Needs n{limit_of(a, place, last) > kb, i0 <= i1 && limit_of(a, place, max(i1, 0)) > kw,
            i0 + 32 <= a.Nq && limit_of(a, place, i0) >= kw + 32};
    if (a.documents && n.block) {
      const Range r = query_range(a, place, b, tile * kTile, last);
      n.block = overlap(r, range);
      n.whole = n.whole && same_document(r, range);
    }
    return n;
  };
  for (int g = share.head0; g < share.head1; ++g) {
    const int h = hk * group + g;
    const Score<MODE> score(a, h);
    const Loader<D, 4> ql(static_cast<const bf16 *>(a.q) + b * a.qs[0] + h * a.qs[1], a.qs[2], a.Nq, a.D, wave);
    const Loader<D, 4> gl(static_cast<const bf16 *>(a.dout) + b * a.gs[0] + h * a.gs[1], a.gs[2], a.Nq, a.Dv, wave);
    const int64_t at = (int64_t(b) * a.H + h) * a.Nq;
    Walk walk(share.tile0, share.tile1);
    Step now = walk.next(test);
    const auto load = [&](bf16 *stage, float *stats, int tile) {
      ql.load(stage, tile * kTile);
      gl.load(stage + TILE, tile * kTile);
      if (wave < 2) {                                    // 64 lse, 64 delta (beyond the end: the last one's)
        const float *from = (wave ? a.delta : a.lse) + at + min(tile * kTile + lane, a.Nq - 1);
        __builtin_amdgcn_global_load_lds((global_void *)from, (lds_void *)(stats + wave * kTile), 4, 0, 0);
      }
    };
    const auto compute = [&](const bf16 *qt, const float *stats) {
      const bf16 *gt = qt + TILE;
      // acc += transposed rows (steps of 16 from 2 half on) times the fragments of P and dS.
      const auto add = [&](int half, const bf16x8 (&p)[2], const bf16x8 (&ds)[2], uint32_t seen) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const bf16x8 sf = weights_seen(seen, 8 * s);
          bf16x8 f[T];
#pragma unroll
          for (int t = 0; t < T; ++t) f[t] = ln.transposed(gt, part * T + t, 2 * half + s);
          add_product<STRICT, false>(f, p[s], sf, dv);
#pragma unroll
          for (int t = 0; t < T; ++t) f[t] = ln.transposed(qt, part * T + t, 2 * half + s);
          add_product<STRICT, false>(f, ds[s], sf, dk);
        }
      };
      uint32_t seen = 0;
      bf16x8 pf[2] = {}, dsf[2] = {};
      if (now.mine) {
        if (!now.whole) mark_queries(a, place, b, now.tile * kTile + part * 32, marks);
        const float *lses = stats + part * 32, *deltas = lses + kTile;
        f32x16 w = ln.product(qt, part, kf), dp = ln.product(gt, part, vf), bent;
        const float gap = float(now.tile * kTile + part * 32 + place.shift + 4 * ln.half - key);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float f = 1.f;
          w[r] = score(w[r], gap + float(row_of_register(r)), &f);
          if constexpr (Score<MODE>::CAP) bent[r] = f;
        }
        seen = now.whole ? 0xffff : hide_queries(marks, ln.half, key, document, w);
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
          pf[s] = weights(w, 8 * s);
          dsf[s] = weights(dp, 8 * s);
        }
      }
      Exchange &mine = exchange[wave];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        mine.p[s][lane] = pf[s];
        mine.ds[s][lane] = dsf[s];
      }
      if constexpr (STRICT) mine.seen[lane] = seen;
      add(part, pf, dsf, seen);
      ring_barrier();
      const Exchange &other = exchange[wave ^ 2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        pf[s] = other.p[s][lane];
        dsf[s] = other.ds[s][lane];
      }
      add(part ^ 1, pf, dsf, STRICT ? other.seen[lane] : 0);
    };
    if constexpr (STRICT || kDkvStages<D> == 1) {
      for (; now.tile >= 0; now = walk.next(test)) {
        ring_barrier();                                  // the tile before is no longer read
        load(stage0, stats0, now.tile);
        wait_loads();
        ring_barrier();
        compute(stage0, stats0);
      }
    } else {
      const auto step = [&](bf16 *use, float *use_stats, bf16 *spare, float *spare_stats) {
        wait_loads();
        ring_barrier();
        const Step then = walk.next(test);
        if (then.tile >= 0) load(spare, spare_stats, then.tile);
        compute(use, use_stats);
        now = then;
      };
      ring_barrier();                                    // (the last head's tiles are no longer read)
      if (now.tile >= 0) load(stage0, stats0, now.tile);
      while (now.tile >= 0) {
        step(stage0, stats0, stage1, stats1);
        if (now.tile < 0) break;
        step(stage1, stats1, stage0, stats0);
      }
    }
  }
}

// Work item = (split, key block, batch entry, key head); the sums of split s go to parts [s][B Hk][Nk][D + Dv] in
// fp32 when there are several.
template <class D, int MODE>
__device__ __forceinline__ void dkv_block(const SequenceArgs &a, const Splits &splits, float *parts, int at, bf16 *stage0,
                                          bf16 *stage1, float *stats0, float *stats1, Exchange *exchange, Marks *marks) {
  constexpr int T = D::DT / 2;
  static_assert(D::DT % 2 == 0, "two wavefronts share the head dim");
  const KeyItem item(a, splits, at);
  const int hk = item.hk, b = item.b;
  const Share &share = item.share;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave >> 1;
  const Lane<D> ln;
  const Place place = place_of(a, b);
  const int kb = item.block * kTile, kw = kb + (wave & 1) * 32, key = kw + ln.col;
  const bool valid = key < place.n;
  bf16x8 kf[D::KS], vf[D::KS];
  own_row<D>(kf, static_cast<const bf16 *>(a.k) + b * a.ks[0] + hk * a.ks[1] + key * a.ks[2], a.D, valid, ln.half);
  own_row<D>(vf, static_cast<const bf16 *>(a.v) + b * a.vs[0] + hk * a.vs[1] + key * a.vs[2], a.Dv, valid, ln.half);
  int document = 0;                                      // (as row_of has it without documents)
  if (a.documents) document = valid ? a.documents[int64_t(b) * a.documents_stride + key] : -1;
  f32x16 dk[T], dv[T];
  dkv_walk<D, MODE, false>(a, ln, stage0, stage1, stats0, stats1, exchange, marks[wave], kf, vf, b, hk, wave, kb, kw, part, key,
                           document, place, share, dk, dv);
  if (__syncthreads_or(valid && (any_bad(dk) || any_bad(dv))))
    dkv_walk<D, MODE, true>(a, ln, stage0, stage1, stats0, stats1, exchange, marks[wave], kf, vf, b, hk, wave, kb, kw, part, key,
                            document, place, share, dk, dv);
  if (key >= a.Nk) return;
  if (!valid) {                                          // beyond the length: zeros
#pragma unroll
    for (int t = 0; t < T; ++t) {
      dk[t] = zeros16();
      dv[t] = zeros16();
    }
  }
  const int d0 = part * T * 32;
  if (splits.heads * splits.tiles > 1) {
    float *to = parts + ((int64_t(item.split) * a.B * a.Hk + int64_t(b) * a.Hk + hk) * a.Nk + key) * (a.D + a.Dv);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = d0 + t * 32 + 8 * j + 4 * ln.half;
        if (d < a.D) *reinterpret_cast<f32x4 *>(to + d) = f32x4{dk[t][4 * j], dk[t][4 * j + 1], dk[t][4 * j + 2], dk[t][4 * j + 3]};
        if (d < a.Dv)
          *reinterpret_cast<f32x4 *>(to + a.D + d) = f32x4{dv[t][4 * j], dv[t][4 * j + 1], dv[t][4 * j + 2], dv[t][4 * j + 3]};
      }
    return;
  }
  store_column(static_cast<bf16 *>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2] + d0, a.D - d0, dk, a.scale, ln.half);
  store_column(static_cast<bf16 *>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2] + d0, a.Dv - d0, dv, 1.f, ln.half);
}

// ------------------------------------------------------------------------------ launches

template <class D, int MODE> __global__ __launch_bounds__(256, 2) void dq_bf16_kernel(SequenceArgs a, int blocks) {
  constexpr int TILE = kTile * D::DL;
  __shared__ __attribute__((aligned(1024))) bf16 stage0[2 * TILE], stage1[2 * TILE];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  dq_block<D, MODE, true>(a, blocks, blockIdx.x, stage0, stage1, marks);
}

template <class D, int MODE>
__global__ __launch_bounds__(256, 2) void dkv_bf16_kernel(SequenceArgs a, Splits splits, float *parts) {
  constexpr int TILE = kTile * D::DL, STAGES = kDkvStages<D>;
  __shared__ __attribute__((aligned(1024))) bf16 stage0[2 * TILE], stage1[STAGES == 2 ? 2 * TILE : 8];
  __shared__ __attribute__((aligned(1024))) float stats0[2 * kTile], stats1[STAGES == 2 ? 2 * kTile : 4];
  __shared__ __attribute__((aligned(16))) Exchange exchange[4];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  dkv_block<D, MODE>(a, splits, parts, blockIdx.x, stage0, stage1, stats0, stats1, exchange, marks);
}

// Both in one launch, dq's work items first, with dout . out from delta_bf16_kernel (6 us at 5 x 768 tokens of 16
// heads of 48): each alone leaves CUs idle at its end, and with few work items all along. Forward and backward of
// 3 x 1111 tokens, 8 heads on 2, D = 64: 116 us in two launches, 97 in one; 5 x 768, 16 heads of 48, with slopes: 163 and
// 154; the backward pass of 2 x 2048, 16 heads on 4, D = 64: 154 and 128, of 4 x 4096 1359 in both (before dS was in
// two pieces). Head dims over 64 stay in two launches: with the stages of both a CU would hold one workgroup.
template <class E> constexpr bool kOneLaunch = kDkvStages<E> == 2;
static_assert(kOneLaunch<Dim<64, 4, 2>> && !kOneLaunch<Dim<128, 8, 4>>, "delta_bf16_kernel takes up to 64 dims");
template <class D, class E, int MODE>
__global__ __launch_bounds__(256, 2) void backward_bf16_kernel(SequenceArgs a, int blocks, int dq_items, Splits splits, float *parts) {
  static_assert(D::DL <= E::DL, "dq takes the stages of dk and dv");
  constexpr int TILE = kTile * E::DL;
  __shared__ __attribute__((aligned(1024))) bf16 stage0[2 * TILE], stage1[2 * TILE];
  __shared__ __attribute__((aligned(1024))) float stats0[2 * kTile], stats1[2 * kTile];
  __shared__ __attribute__((aligned(16))) Exchange exchange[4];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  const int item = blockIdx.x;
  if (item < dq_items) dq_block<D, MODE, false>(a, blocks, item, stage0, stage1, marks);
  else dkv_block<E, MODE>(a, splits, parts, item - dq_items, stage0, stage1, stats0, stats1, exchange, marks);
}

// delta[row] = dout . out of up to 64 dims: eight lanes a row, 16 bytes each.
__global__ __launch_bounds__(256) void delta_bf16_kernel(SequenceArgs a) {
  const int64_t at = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> 3;
  if (at >= int64_t(a.B) * a.H * a.Nq) return;           // (all lanes of a row)
  const int i = int(at % a.Nq), h = int(at / a.Nq % a.H), b = int(at / a.Nq / a.H), d = (threadIdx.x & 7) * 8;
  bf16x8 of = {}, gf = {}, lf = {};
  if (d < a.Dv) {
    of = *reinterpret_cast<const bf16x8 *>(static_cast<const bf16 *>(a.out) + b * a.os[0] + h * a.os[1] + i * a.os[2] + d);
    gf = *reinterpret_cast<const bf16x8 *>(static_cast<const bf16 *>(a.dout) + b * a.gs[0] + h * a.gs[1] + i * a.gs[2] + d);
    if (a.low) lf = *reinterpret_cast<const bf16x8 *>(static_cast<const bf16 *>(a.low) + at * a.Dv + d);
  }
  float delta = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    delta = __builtin_fmaf(static_cast<float>(of[e]) + static_cast<float>(lf[e]), static_cast<float>(gf[e]), delta);
#pragma unroll
  for (int o = 1; o < 8; o *= 2) delta += __shfl_xor(delta, o, 64);
  if (threadIdx.x % 8 == 0) a.delta[at] = delta;
}

}  // namespace

bool sequence_bf16_backward_fits(const SequenceArgs &a) {
  return sequence_bf16_forward_fits(a) && rows_fit(a.out, a.os, a.Dv, 8) && rows_fit(a.dout, a.gs, a.Dv, 8) && reinterpret_cast<uintptr_t>(a.low) % 16 == 0 &&
         rows_fit(a.dq, a.dqs, a.D, 4) && rows_fit(a.dk, a.dks, a.D, 4) && rows_fit(a.dv, a.dvs, a.Dv, 4);
}


int sequence_bf16_backward(const SequenceArgs &a, const Splits &splits, float *parts, hipStream_t s) {
  const int64_t blocks = ceil_div(int64_t(a.H / a.Hk) * a.Nq, int64_t(kColumns)), kblocks = ceil_div(int64_t(a.Nk), int64_t(kTile));
  return with_dims(a, [&](auto dim, auto mode) {
    typedef decltype(dim) D;
    typedef Dim<D::DL < 64 ? 64 : D::DL, D::KS, D::DT + D::DT % 2> E;    // (two wavefronts share the head dim)
    constexpr int MODE = decltype(mode)::value;
    const int64_t dq_items = blocks * a.Hk * a.B, dkv_items = a.dk || a.dv ? kblocks * a.Hk * a.B * splits.heads * splits.tiles : 0;
    if constexpr (kOneLaunch<E>) {
      if (dq_items > 0) delta_bf16_kernel<<<dim3(unsigned(ceil_div(int64_t(a.B) * a.H * a.Nq, int64_t(32)))), 256, 0, s>>>(a);
      XFH_TRY(check_launch("sequence_attention_backward"));
      return sequence_launch_both(dq_items, dkv_items, [&](int64_t items, int64_t first) {
        backward_bf16_kernel<D, E, MODE><<<dim3(unsigned(items)), 256, 0, s>>>(a, int(blocks), int(first), splits, parts);
      });
    } else {
      if (dq_items > 0) dq_bf16_kernel<D, MODE><<<dim3(unsigned(dq_items)), 256, 0, s>>>(a, int(blocks));
      XFH_TRY(check_launch("sequence_attention_backward"));
      if (dkv_items > 0) dkv_bf16_kernel<E, MODE><<<dim3(unsigned(dkv_items)), 256, 0, s>>>(a, splits, parts);
    }
    return check_launch("sequence_attention_backward");
  });
}

}  // namespace xfh
