// Sequence attention: what its kernels share (arguments, masks, scores).
//
//   x_ij = scale q_i . k_j,  c_ij = cap tanh(x_ij / cap) (cap > 0),  s_ij = c_ij - slope_h |p_i - j|
//   O_i = sum_j P_ij v_j,  P_ij = exp(s_ij - L_i) over the visible keys,  L_i = log sum exp s_ij
// p_i = i + n - Nq is the place of query i in its sequence of n tokens. Query i sees key j iff
//   j < n, and (not causal, or j <= p_i, or j < prefix), and document[p_i] == document[j] >= 0.
// For one query all but the documents is one bound, j < limit; 0 where it sees nothing.
// Scores and L are held in units of log 2 (the kernels take exp2).
#pragma once

#include "common.h"
#include "kernels.h"

namespace xfh {
namespace seq {

constexpr int kTile = 64;                  // tokens of a tile: keys of a loop step, and document ranges

// Documents of a tile of 64 keys: the lowest and highest of its kept keys (lo > hi: none), and
// whether all 64 are kept.
typedef int4 Range;                        // lo, hi, full, unused

struct Place { int n, prefix, shift; };    // of one batch entry: tokens, prefix, p_i - i

__device__ __forceinline__ Place place_of(const SequenceArgs &a, int b) {
  Place p;
  p.n = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  p.prefix = a.prefix ? a.prefix[b] : a.prefix_all;
  p.shift = p.n - a.Nq;
  return p;
}
// Bound on the keys of query i < Nq, documents aside. It does not fall as i rises.
__device__ __forceinline__ int limit_of(const SequenceArgs &a, const Place &p, int i) {
  const int pos = i + p.shift;
  if (a.lengths && pos < 0) return 0;
  return a.causal ? min(p.n, max(pos + 1, p.prefix)) : p.n;
}
struct Row { int limit, document, pos; };
__device__ __forceinline__ Row row_of(const SequenceArgs &a, const Place &p, int b, int i) {
  Row r{0, 0, i + p.shift};
  if (i >= a.Nq) return r;
  r.limit = limit_of(a, p, i);
  if (a.documents) {
    r.document = r.pos >= 0 && r.pos < p.n ? a.documents[int64_t(b) * a.documents_stride + r.pos] : -1;
    if (r.document < 0) r.limit = 0;
  }
  return r;
}

// Range of the documents of queries [i0, i1].
__device__ __forceinline__ Range query_range(const SequenceArgs &a, const Place &p, int b, int i0, int i1) {
  const int p0 = max(i0 + p.shift, 0), p1 = i1 + p.shift;
  if (p1 < 0) return Range{0x7fffffff, -1, 0, 0};
  const Range *r = static_cast<const Range *>(a.ranges) + int64_t(b) * a.tiles;
  Range u = r[p0 / kTile];
  for (int t = p0 / kTile + 1; t <= p1 / kTile; ++t) {
    u.x = min(u.x, r[t].x);
    u.y = max(u.y, r[t].y);
    u.z &= r[t].z;
  }
  return u;
}
__device__ __forceinline__ bool overlap(const Range &u, const Range &w) { return u.x <= w.y && w.x <= u.y; }
// Every pair of a token of one and a token of the other is in one document.
__device__ __forceinline__ bool same_document(const Range &u, const Range &w) {
  return u.z && w.z && u.x == u.y && w.x == w.y && u.x == w.x;
}

// c / cap and its slope. fp32: the library's tanh. bf16: 1 - 2 / (exp(2 t) + 1) on the hardware's
// exp2 and reciprocal, off by at most about 2^-22 (a score of 50 by 1e-5, far below the step of P in bf16).
template <typename T> __device__ __forceinline__ float bend(float t);
template <> __device__ __forceinline__ float bend<float>(float t) { return tanhf(t); }
template <> __device__ __forceinline__ float bend<bf16>(float t) {
  const float e = __builtin_amdgcn_exp2f(t * (2.0f * kLog2e));
  return 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
}
// A query's part of its slope's gradient: all = sum P, far = sum P |gap|, error = sum P (dP - delta), far_error =
// sum P (dP - delta) |gap|. A query that sees nothing has none.
__device__ __forceinline__ float slope_gradient(float all, float far, float error, float far_error) {
  return all == 0.f ? 0.f : -(far_error - error * (far / all)) / all;
}

constexpr float kLowest = -3.402823466e38f;              // running maximum before the first key

// The part of a sequence's keys that a workgroup of a forward pass has, of the columns of its block: part `index` of
// `count`, kept in `slot`. count = 0: none.
//
// Sequences of different lengths share the slots by need: each has parts of at most P tiles, with P the least
// of 64 tries (a lane each) for which all parts fit. 4 x 200 queries of 1500 to 5000 keys, 32 heads on 8,
// D = 128, bf16: 72 us with the join, 79 with two equal parts each; of 5000 keys and three times 300: 51 and 78.
struct Part {
  int b, blk, hk, index, count, slot;
  __device__ __forceinline__ Part(const SequenceArgs &a, const Parts &parts, int blocks, unsigned item) {
    hk = int(item) % a.Hk;
    int rest = int(item) / a.Hk;
    if (!parts.table) {
      index = rest % parts.splits;
      rest /= parts.splits;
      blk = blocks - 1 - rest % blocks;                  // the last queries, which see most under a causal mask, first
      b = rest / blocks;
      count = parts.splits;
      slot = index * a.B + b;
      return;
    }
    slot = rest % parts.slots;
    blk = blocks - 1 - rest / parts.slots;
    const int lane = threadIdx.x & 63;
    const auto tiles_of = [&](int e) { return e < a.B ? (place_of(a, e).n + kTile - 1) / kTile : 0; };
    const int t0 = tiles_of(lane);
    int total = 0, longest = 0;
    for (int e0 = 0; e0 < a.B; e0 += 64) {
      const int t = e0 ? tiles_of(e0 + lane) : t0;
      for (int e = 0; e < min(64, a.B - e0); ++e) {
        const int tiles = __builtin_amdgcn_readlane(t, e);
        total += tiles;
        longest = max(longest, tiles);
      }
    }
    const int low = max(8, (total + parts.slots - 1) / parts.slots), step = (max(longest - low, 0) + 62) / 63;
    const int mine = low + lane * step;                  // (the last lane's: one part each, which fits)
    int sum = 0;
    for (int e0 = 0; e0 < a.B; e0 += 64) {
      const int t = e0 ? tiles_of(e0 + lane) : t0;
      for (int e = 0; e < min(64, a.B - e0); ++e) sum += parts_of(__builtin_amdgcn_readlane(t, e), mine);
    }
    const int per = __builtin_amdgcn_readlane(mine, __builtin_ctzll(__ballot(sum <= parts.slots)));
    int first = 0;
    b = 0;
    count = 0;
    for (int e0 = 0; e0 < a.B && !count; e0 += 64) {
      const int c = parts_of(e0 ? tiles_of(e0 + lane) : t0, per);
      for (int e = 0; e < min(64, a.B - e0); ++e) {
        const int n = __builtin_amdgcn_readlane(c, e);
        if (slot < first + n) {
          b = e0 + e;
          count = n;
          break;
        }
        first += n;
      }
    }
    index = slot - first;
    if (count && index == 0 && hk == 0 && blk == 0 && threadIdx.x == 0) parts.table[b] = make_int2(first, count);
  }
  // At least one part; ceil(tiles / per), by a quotient in floats that is off by at most one.
  __device__ __forceinline__ static int parts_of(int tiles, int per) {
    int c = int(float(tiles + per - 1) * __builtin_amdgcn_rcpf(float(per)));
    c += c * per < tiles;
    c -= (c - 1) * per >= tiles;
    return max(c, 1);
  }
  // Of `end` tiles, this part's.
  __device__ __forceinline__ void take(int &first, int &end) const {
    const int per = (end + count - 1) / count;
    first = min(index * per, end);
    end = min(first + per, end);
  }
};
__device__ __forceinline__ bool several(const Parts &parts) { return parts.splits > 1 || parts.table; }

// A work item of dk and dv: 64 keys, and of the heads of their group and the tiles of their queries the share
// [head0, head1) x [tile0, tile1) that this split has. The first keys, which causal queries see most, first.
struct Share { int head0, head1, tile0, tile1; };
struct KeyItem {
  int b, hk, block, split;
  Share share;
  __device__ __forceinline__ KeyItem(const SequenceArgs &a, const Splits &splits, unsigned item) {
    const int group = a.H / a.Hk, qtiles = (a.Nq + kTile - 1) / kTile, count = splits.heads * splits.tiles;
    hk = int(item) % a.Hk;
    int rest = int(item) / a.Hk;
    b = rest % a.B;
    rest /= a.B;
    split = rest % count;
    block = rest / count;
    const int sh = split % splits.heads, st = split / splits.heads;
    share = {sh * group / splits.heads, (sh + 1) * group / splits.heads, int(int64_t(st) * qtiles / splits.tiles),
             int(int64_t(st + 1) * qtiles / splits.tiles)};
  }
};

// A tile of a walk: its number (-1: none is left), whether this wavefront's columns see any and all of it.
struct Step { int tile; bool mine, whole; };

// The walk over tiles [first, end), 64 of them at a time, one per lane. test(tile) says which of {the
// workgroup needs it, the wavefront needs it, the wavefront's columns see it whole} hold.
struct Needs { bool block, mine, whole; };
struct Walk {
  int first, end;
  uint64_t need = 0, mine = 0, whole = 0;
  __device__ __forceinline__ Walk(int f, int e) : first(f - 64), end(e) {}
  template <class F> __device__ __forceinline__ Step next(F test) {
    while (!need) {
      first += 64;
      if (first >= end) return {-1, false, false};
      const int tile = first + int(threadIdx.x & 63);
      Needs n{false, false, false};
      if (tile < end) n = test(tile);
      need = __ballot(n.block);
      mine = __ballot(n.block && n.mine);
      whole = __ballot(n.block && n.mine && n.whole);
    }
    const int bit = __builtin_ctzll(need);
    need &= need - 1;
    return {first + bit, bool((mine >> bit) & 1), bool((whole >> bit) & 1)};
  }
};

// Bounds and documents of the keys that a run of queries sees.
struct Span { int low, high; Range range; };
__device__ __forceinline__ Span span_of(const SequenceArgs &a, const Place &p, int b, int i0, int i1) {
  Span s{0, 0, Range{0x7fffffff, -1, 0, 0}};
  if (i0 > i1) return s;
  s.low = limit_of(a, p, i0);
  s.high = limit_of(a, p, i1);
  if (a.documents) s.range = query_range(a, p, b, i0, i1);
  return s;
}
__device__ __forceinline__ Needs key_tile_needs(const SequenceArgs &a, int b, int tile, const Span &block, const Span &wave) {
  const int k0 = tile * kTile;
  Needs n{k0 < block.high, k0 < wave.high, k0 + kTile <= wave.low};
  if (a.documents && n.block) {
    const Range r = static_cast<const Range *>(a.ranges)[int64_t(b) * a.tiles + tile];
    n.block = overlap(r, block.range);
    n.mine = n.mine && overlap(r, wave.range);
    n.whole = n.whole && same_document(r, wave.range);
  }
  return n;
}

}  // namespace seq
}  // namespace xfh
