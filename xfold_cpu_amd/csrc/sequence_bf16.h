// Tiles of the bf16 sequence attention kernels (head dims that are multiples of 8, rows on 16 bytes).
//
// Products are 32x32x16 MFMAs with a wavefront's 32 owned tokens as columns: lane l = 32 half + c holds
// column c, rows 8 (r / 4) + 4 half + r % 4 of a 32-row result (r = 0..15). For the next product, over
// these rows, a step of 16 takes registers 8 s .. 8 s + 7 as they are: slot e < 4 of half h is row
// 4 h + e, slot e >= 4 row 8 + 4 h + e - 4, and the other operand is read in the same order.
//
// A tile of 64 tokens lies row-major in LDS, DL elements a row, brought there by direct loads (a
// wavefront writes 1 KB, lane i its bytes [16 i, 16 i + 16)). 16-byte chunk c of row r is at slot
// c ^ swizzle(r), chosen so that the 16 rows (one chunk each) of a row-fragment read, and the 4 rows (4
// chunks each) of a transposing read, lie in different banks (256 bytes). What lies beyond a
// matrix's end is a copy of its last row, beyond the head dim a copy of the row's first chunk: both
// meet weights, or elements of the other operand, that are zero.
#pragma once

#include <algorithm>
#include <type_traits>

#include "sequence.h"

namespace xfh {
namespace seq {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(1))) void global_void;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Head dims up to DL_ in LDS, KS_ steps of 16 in a product over the head dim, DT_ tiles of 32 of it in a result.
template <int DL_, int KS_, int DT_> struct Dim {
  static constexpr int DL = DL_, KS = KS_, DT = DT_;
  static constexpr int ROW_PIECES = 512 / DL;            // rows of a 1 KB piece
  static constexpr int PIECES = kTile / ROW_PIECES;      // pieces of a tile of 64
  static_assert(DL == 32 || DL == 64 || DL == 128, "LDS rows of 64, 128 or 256 bytes");
  static_assert(KS * 16 <= DL && DT * 32 <= DL, "products within the row");
  static __device__ __forceinline__ int swizzle(int row) {
    return (DL == 128 ? (row & 3) << 2 : DL == 64 ? (row & 2) << 1 : 0) | ((row >> 2) & 3);
  }
};

__device__ __forceinline__ f32x16 mfma32(const bf16x8 &a, const bf16x8 &b, const f32x16 &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zeros16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// Row of register r of a 32-row result.
__device__ __forceinline__ constexpr int row_of_register(int r) { return 8 * (r / 4) + r % 4; }   // + 4 half

// Lane offsets (elements) into a tile.
template <class D> struct Lane {
  int half, col, rows, swz, tr[2][D::DT];
  __device__ __forceinline__ Lane() {
    const int lane = threadIdx.x & 63;
    half = lane >> 5;
    col = lane & 31;
    rows = col * D::DL;
    swz = D::swizzle(col) ^ half;
    // Transposing read: 16 lanes take 4 rows of 16 elements, 4 elements a lane; then the same 8 rows on.
    const int i = lane & 15, chunk = 2 * ((lane >> 4) & 1) + (i % 4) / 2;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int row = 8 * s + 4 * half + i / 4;
#pragma unroll
      for (int t = 0; t < D::DT; ++t) tr[s][t] = row * D::DL + ((t * 4 + chunk) ^ D::swizzle(row)) * 8 + 4 * (i & 1);
    }
  }
  // Rows 32 rt .. of a tile, elements 16 ks + 8 half ..: the A operand of a product over the head dim.
  __device__ __forceinline__ bf16x8 row_fragment(const bf16 *tile, int rt, int ks) const {
    return *reinterpret_cast<const bf16x8 *>(tile + rt * 32 * D::DL + rows + ((2 * ks) ^ swz) * 8);
  }
  // Head dims 32 t .. as rows, 16 rows of the tile from 16 kk on as k: the A operand of a product over tokens.
  __device__ __forceinline__ bf16x8 transposed(const bf16 *tile, int t, int kk) const {
    const bf16 *p = tile + kk * 16 * D::DL;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + tr[0][t]));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + tr[1][t]));
    const __attribute__((ext_vector_type(8))) short v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, v);
  }
  // [32 rows of the tile] x [owned columns] over the head dim.
  __device__ __forceinline__ f32x16 product(const bf16 *tile, int rt, const bf16x8 (&own)[D::KS]) const {
    f32x16 acc = zeros16();
#pragma unroll
    for (int ks = 0; ks < D::KS; ++ks) acc = mfma32(row_fragment(tile, rt, ks), own[ks], acc);
    return acc;
  }
  __device__ __forceinline__ void transposed_fragments(const bf16 *tile, int kk, bf16x8 (&f)[D::DT]) const {
#pragma unroll
    for (int t = 0; t < D::DT; ++t) f[t] = transposed(tile, t, kk);
  }
};
// acc += fragments^T w over 16 rows of a tile. STRICT: elements that are not finite are left out and added to
// the columns that see them (`seen`, 1 or 0): with SIGNS as what they are, else as NaN.
template <bool STRICT, bool SIGNS, int T>
__device__ __forceinline__ void add_product(const bf16x8 (&f)[T], const bf16x8 &w, const bf16x8 &seen, f32x16 (&acc)[T]) {
#pragma unroll
  for (int t = 0; t < T; ++t) {
    bf16x8 a = f[t];
    if constexpr (STRICT) {
      bf16x8 up, down;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = static_cast<float>(a[e]);
        const bool bad = !(fabsf(x) < INFINITY);
        up[e] = bf16(bad && !(SIGNS && x < 0.f) ? 1.f : 0.f);
        down[e] = bf16(bad && !(SIGNS && x > 0.f) ? 1.f : 0.f);
        if (bad) a[e] = bf16(0.f);
      }
      const f32x16 ups = mfma32(up, seen, zeros16()), downs = mfma32(down, seen, zeros16());
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (ups[r] > 0.f) acc[t][r] += INFINITY;
        if (downs[r] > 0.f) acc[t][r] -= INFINITY;
      }
    }
    acc[t] = mfma32(a, w, acc[t]);
  }
}


// 8 registers of a result, rounded, as the B operand of a step of 16.
__device__ __forceinline__ bf16x8 weights(const f32x16 &w, int first) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<bf16>(w[first + e]);
  return v;
}
__device__ __forceinline__ bf16x8 weights_seen(uint32_t seen, int first) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = bf16((seen >> (first + e)) & 1 ? 1.f : 0.f);
  return v;
}

// The other lane of a column (the same column in the other half).
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// An owned token's row as B fragments (chunk 2 ks + half), zero beyond D.
template <class D> __device__ __forceinline__ void own_row(bf16x8 (&f)[D::KS], const bf16 *row, int dim, bool valid, int half) {
#pragma unroll
  for (int ks = 0; ks < D::KS; ++ks) {
    bf16x8 z = {};
    const int at = ks * 16 + half * 8;
    f[ks] = valid && at < dim ? *reinterpret_cast<const bf16x8 *>(row + at) : z;
  }
}

// Direct loads of tiles of one matrix ([rows][dim], row stride in elements) by W wavefronts: piece j of
// wavefront w is w + j W.
template <class D, int W, int ROWS = kTile> struct Loader {
  static constexpr int N = ROWS / D::ROW_PIECES / W;
  static_assert(N * D::ROW_PIECES * W == ROWS, "whole pieces for each wavefront");
  uint32_t offset[N];                                    // bytes from the tile's first row
  const bf16 *base;
  int64_t stride;
  int wave, last, dim;                                   // last: the matrix's last row
  __device__ __forceinline__ Loader(const bf16 *b, int64_t s, int rows, int d, int w)
      : base(b), stride(s), wave(w), last(rows - 1), dim(d) {
#pragma unroll
    for (int j = 0; j < N; ++j) offset[j] = uint32_t(int64_t(row(j)) * stride * 2) + chunk(j) * 16;
  }
  __device__ __forceinline__ int row(int j) const {
    return (wave + j * W) * D::ROW_PIECES + int(threadIdx.x & 63) / (D::DL / 8);
  }
  __device__ __forceinline__ uint32_t chunk(int j) const {
    const int c = int(threadIdx.x & 63) % (D::DL / 8) ^ D::swizzle(row(j));
    return c * 8 < dim ? c : 0;
  }
  // Piece j of the rows from `first` (at most the last one) on.
  __device__ __forceinline__ void load_piece(bf16 *tile, int first, int j) const {
    const char *p = reinterpret_cast<const char *>(base + int64_t(first) * stride) + offset[j];
    if (first + ROWS - 1 > last)
      p = reinterpret_cast<const char *>(base + int64_t(min(first + row(j), last)) * stride) + chunk(j) * 16;
    __builtin_amdgcn_global_load_lds((global_void *)p, (lds_void *)(tile + (wave + j * W) * 512), 16, 0, 0);
  }
  __device__ __forceinline__ void load(bf16 *tile, int first) const {
#pragma unroll
    for (int j = 0; j < N; ++j) load_piece(tile, first, j);
  }
};

// Waits for this wavefront's loads (vmcnt 0; the other counters as they are). By the builtin, which the compiler
// counts: after a wait written in assembly it would wait again, for the loads issued since too.
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);
  asm volatile("" ::: "memory");
}

// How a score comes from a dot product: MODE bit 0 = cap, bit 1 = distance slopes (or a scale that is not
// positive). Scores are in log 2 units. Without slopes what is held is something that rises with the score,
// score = unit w + offset, and the exponent's multiply-add does the rest: the dot product itself (MODE 0),
// or (tanh - 1) / 2 = -1 / (exp(2 x / cap) + 1).
template <int MODE> struct Score {
  static constexpr bool CAP = MODE & 1, SLOPE = MODE & 2;
  float unit, offset, to_exponent, cap2, slope;
  __device__ __forceinline__ Score(const SequenceArgs &a, int h)
      : unit(MODE == 1 ? 2.0f * a.cap * kLog2e : a.scale * kLog2e), offset(a.cap * kLog2e),
        to_exponent(CAP ? a.scale * 2.0f * kLog2e / a.cap : 0.f), cap2(a.cap * kLog2e),
        slope(SLOPE && a.slopes ? a.slopes[h] * kLog2e : 0.f) {}
  // gap = p_i - j; `bent` (1 - tanh^2) when asked for.
  __device__ __forceinline__ float operator()(float dot, float gap, float *bent = nullptr) const {
    float w = dot;
    if constexpr (CAP) {
      w = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(dot * to_exponent));
      if (bent) *bent = -4.0f * __builtin_fmaf(w, w, w);
      if constexpr (SLOPE) w = __builtin_fmaf(w, 2.0f * cap2, cap2);
    } else if constexpr (SLOPE) {
      w = dot * unit;
    }
    if constexpr (SLOPE) w = __builtin_fmaf(-slope, fabsf(gap), w);
    return w;
  }
  // exp2(score - m)
  __device__ __forceinline__ float weight(float w, float m) const {
    return __builtin_amdgcn_exp2f(SLOPE ? w - m : __builtin_fmaf(w, unit, MODE == 1 ? offset - m : -m));
  }
  __device__ __forceinline__ float in_log2(float w) const {
    return SLOPE ? w : MODE == 1 ? __builtin_fmaf(w, unit, offset) : w * unit;
  }
};

// What a wavefront looks up to hide pairs: bounds and documents of the rows of a tile, in LDS of its own (a
// lane works out one row; the 16 rows of a lane's registers are then eight 16-byte reads).
struct Marks { int limit[kTile], document[kTile]; };
__device__ __forceinline__ void marks_written() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// Documents of the keys of a tile (k0 ..; beyond n they stay what they were, and are not looked at).
__device__ __forceinline__ void mark_keys(const SequenceArgs &a, int b, int k0, int n, Marks &marks) {
  if (!a.documents) return;
  const int key = k0 + int(threadIdx.x & 63);
  marks_written();                                       // (the tile before is done with them)
  if (key < n) marks.document[threadIdx.x & 63] = a.documents[int64_t(b) * a.documents_stride + key];
  marks_written();
}
// Scores of hidden pairs in rows 32 rt .. of a tile of keys (k0 ..) become -infinity; returns the bits of the seen.
__device__ __forceinline__ uint32_t hide_keys(const SequenceArgs &a, const Marks &marks, int rt, int k0, int half,
                                              const Row &row, f32x16 &w) {
  uint32_t seen = 0;
  const int limit = row.limit - k0 - rt * 32 - 4 * half;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int4 ids{row.document, row.document, row.document, row.document};
    if (a.documents) ids = *reinterpret_cast<const int4 *>(marks.document + rt * 32 + 8 * j + 4 * half);
    const int id[4] = {ids.x, ids.y, ids.z, ids.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool see = (8 * j + e < limit) & (id[e] == row.document);
      w[4 * j + e] = see ? w[4 * j + e] : -INFINITY;
      seen |= see ? 1u << (4 * j + e) : 0u;
    }
  }
  return seen;
}

constexpr int kColumns = 128;                            // columns of a workgroup (32 per wavefront)

// Whether a result holds anything that is not finite.
template <int T> __device__ __forceinline__ bool any_bad(const f32x16 (&o)[T]) {
  bool bad = false;
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad |= !(fabsf(o[t][r]) < INFINITY);
  return bad;
}

// A column's result: dims 32 t + 8 j + 4 half .. + 3, four at a time.
template <int T>
__device__ __forceinline__ void store_column(bf16 *out, int dim, const f32x16 (&o)[T], float scale, int half,
                                             bf16 *low = nullptr) {
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = t * 32 + 8 * j + 4 * half;
      if (d < dim) {
        bf16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<bf16>(o[t][4 * j + e] * scale);
        *reinterpret_cast<bf16x4 *>(out + d) = v;
        if (low) {
          bf16x4 u;
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = static_cast<bf16>(o[t][4 * j + e] * scale - static_cast<float>(v[e]));
          *reinterpret_cast<bf16x4 *>(low + d) = u;
        }
      }
    }
}

// ------------------------------------------------------------------------------ launches

inline int mode_of(const SequenceArgs &a) { return (a.cap > 0.f ? 1 : 0) | (a.slopes || (a.cap <= 0.f && a.scale <= 0.f) ? 2 : 0); }

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

inline bool rows_fit(const void *p, const int64_t *strides, int64_t dim, int64_t unit) {
  if (reinterpret_cast<uintptr_t>(p) % (2 * unit) || dim % unit) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] % unit || strides[i] < 0) return false;
  return strides[2] < (int64_t(1) << 24);                // 64 rows of a tile within 32-bit offsets
}

}  // namespace seq
}  // namespace xfh
