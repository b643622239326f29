// Sequence attention in bf16 on 32x32x16 MFMAs (sequence_bf16.h), backward: dq, then dk and dv.
//
// dq: the columns are queries, as in the forward pass. dk and dv: the columns are 64 keys, each 32 of them
// with two wavefronts that take half a tile of queries each; the loop goes over the heads of the group
// and their queries. Two kernels with 3 and 4 products, of which 2 are the same, in place of one with
// 5: the sums of dq need no atomics, and a call gives the same bits every time.
#include "sequence_bf16.h"

namespace xfh {
namespace {

using namespace seq;

// ------------------------------------------------------------------------------ dq

struct SlopeSums { float far, error, far_error; };       // sum P |gap|, sum P (dP - delta), sum P (dP - delta) |gap|

template <class D, int MODE, bool STRICT>
__device__ __forceinline__ void dq_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *stage0, bf16 *stage1,
                                        const Loader<D, 4> &kl, const Loader<D, 4> &vl, const bf16x8 (&qf)[D::KS],
                                        const bf16x8 (&gf)[D::KS], const Score<MODE> &score, int b, int end, int n,
                                        const Span &block, const Span &wave, const Row &row, Marks &marks, float lse,
                                        float delta, f32x16 (&dq)[D::DT], SlopeSums &sums) {
  constexpr int TILE = kTile * D::DL;
  sums = SlopeSums{0.f, 0.f, 0.f};
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
            sums.far = __builtin_fmaf(p, away, sums.far);
            sums.error += ds;
            sums.far_error = __builtin_fmaf(ds, away, sums.far_error);
          }
        }
        w[r] = Score<MODE>::CAP ? ds * bent[r] : ds;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 tf[D::DT];
        ln.transposed_fragments(kt, 2 * rt + s, tf);
        ln.template accumulate<STRICT, false>(tf, weights(w, 8 * s), weights_seen(seen, 8 * s), dq);
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

template <class D, int MODE>
__global__ __launch_bounds__(256, 2) void dq_bf16_kernel(SequenceArgs a, int blocks) {
  constexpr int TILE = kTile * D::DL;
  __shared__ __attribute__((aligned(1024))) bf16 stage0[2 * TILE], stage1[2 * TILE];
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
  dq_walk<D, MODE, false>(a, ln, stage0, stage1, kl, vl, qf, gf, score, b, end, place.n, block, mine, row, marks[wave], lse, delta, dq, sums);
  if (__syncthreads_or(valid && any_bad<D>(dq)))
    dq_walk<D, MODE, true>(a, ln, stage0, stage1, kl, vl, qf, gf, score, b, end, place.n, block, mine, row, marks[wave], lse, delta, dq, sums);
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
__device__ __forceinline__ void dkv_walk(const SequenceArgs &a, const Lane<D> &ln, bf16 *stage0, bf16 *stage1,
                                         float *stats0, float *stats1, Marks &marks, const bf16x8 (&kf)[D::KS],
                                         const bf16x8 (&vf)[D::KS], int b, int hk, int wave, int kb, int kw, int rt, int key,
                                         int document, const Place &place, f32x16 (&dk)[D::DT], f32x16 (&dv)[D::DT]) {
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
    const auto load = [&](bf16 *to, float *stats, int tile) {
      ql.load(to, tile * kTile);
      gl.load(to + TILE, tile * kTile);
      if (wave < 2) {                                    // 64 lse, 64 delta (beyond the end: the last one's)
        const float *from = (wave ? a.delta : a.lse) + at + min(tile * kTile + int(threadIdx.x & 63), a.Nq - 1);
        __builtin_amdgcn_global_load_lds((global_void *)from, (lds_void *)(stats + wave * kTile), 4, 0, 0);
      }
    };
    Walk walk(0, qtiles);
    Step now = walk.next(test);
    const auto compute = [&](const bf16 *qt, const float *stats) {
      if (!now.mine) return;
      const bf16 *gt = qt + TILE;
      const float *lses = stats + rt * 32, *deltas = lses + kTile;
      const int i0 = now.tile * kTile + rt * 32;
      if (!now.whole) mark_queries(a, place, b, i0, marks);
      f32x16 w = zeros16(), dp = zeros16(), bent;
      bf16x8 qf[D::KS], gf[D::KS], qtf[2][D::DT], gtf[2][D::DT];
      ln.row_fragments(qt, rt, qf);
      ln.row_fragments(gt, rt, gf);
      reads_first();
#pragma unroll
      for (int ks = 0; ks < D::KS; ++ks) {
        w = mfma32(qf[ks], kf[ks], w);
        dp = mfma32(gf[ks], vf[ks], dp);
      }
      ln.transposed_fragments(gt, 2 * rt, gtf[0]);
      ln.transposed_fragments(qt, 2 * rt, qtf[0]);
      const float gap = float(i0 + place.shift + 4 * ln.half - key);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float f = 1.f;
        w[r] = score(w[r], gap + float(row_of_register(r)), &f);
        if constexpr (Score<MODE>::CAP) bent[r] = f;
      }
      uint32_t seen = 0xffff;
      if (!now.whole) seen = hide_queries(marks, ln.half, key, document, w);
      ln.transposed_fragments(gt, 2 * rt + 1, gtf[1]);
      ln.transposed_fragments(qt, 2 * rt + 1, qtf[1]);
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
        ln.template accumulate<STRICT, false>(gtf[s], weights(w, 8 * s), sf, dv);
        ln.template accumulate<STRICT, false>(qtf[s], weights(dp, 8 * s), sf, dk);
      }
    };
    if constexpr (STRICT) {                              // rare: one stage will do
      while (now.tile >= 0) {
        ring_barrier();
        load(stage0, stats0, now.tile);
        wait_loads();
        ring_barrier();
        compute(stage0, stats0);
        now = walk.next(test);
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

template <class D, int MODE>
__global__ __launch_bounds__(256, D::DL == 128 ? 1 : 2) void dkv_bf16_kernel(SequenceArgs a, int blocks) {
  constexpr int TILE = kTile * D::DL;
  __shared__ __attribute__((aligned(1024))) bf16 stage0[2 * TILE], stage1[2 * TILE];
  __shared__ __attribute__((aligned(1024))) float stats0[2 * kTile], stats1[2 * kTile];
  __shared__ __attribute__((aligned(16))) Marks marks[4];
  static_assert(sizeof(stage0) >= 2 * D::DT * 16 * 64 * 4, "a key group's sums are joined in a stage");
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
  dkv_walk<D, MODE, false>(a, ln, stage0, stage1, stats0, stats1, marks[wave], kf, vf, b, hk, wave, kb, kw, rt, key, document, place, dk, dv);
  if (__syncthreads_or(valid && (any_bad<D>(dk) || any_bad<D>(dv))))
    dkv_walk<D, MODE, true>(a, ln, stage0, stage1, stats0, stats1, marks[wave], kf, vf, b, hk, wave, kb, kw, rt, key, document, place, dk, dv);
  __syncthreads();
  // The wavefront of the tiles' second halves hands its sums to that of the first.
  float *join = reinterpret_cast<float *>(wave & 1 ? stage1 : stage0) + (threadIdx.x & 63);
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

}  // namespace

bool sequence_bf16_backward_fits(const SequenceArgs &a) {
  return sequence_bf16_forward_fits(a) && rows_fit(a.out, a.os, a.Dv, 8) && rows_fit(a.dout, a.gs, a.Dv, 8) &&
         rows_fit(a.dq, a.dqs, a.D, 4) && rows_fit(a.dk, a.dks, a.D, 4) && rows_fit(a.dv, a.dvs, a.Dv, 4);
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
