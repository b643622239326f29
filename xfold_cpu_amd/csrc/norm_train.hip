// LayerNorm for training: the forward pass with the rows' statistics kept, and the backward pass.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b
//   g = dy w, dx = r (g - mean(g) - h mean(g h)), dw = sum over rows of dy h, db = sum over rows of dy
//
// Both passes are bound by memory: x in and y out, then x and dy in and dx out, each once (a row
// stays in registers between its sums and its result). A row is owned by LPR lanes of one
// workgroup, 8 CH elements a lane: 16 lanes of a wavefront, a wavefront, or all 256 threads (two
// cross-wavefront sums in LDS). Statistics and sums are fp32, the variance from the deviations.
// 589824 x 128 in bf16: forward 55 us (302 MB, 5.5 TB/s; a copy reaches 6.2), backward 89 (453 MB, 5.1 TB/s) and 4 for
// the parameters; 8192 x 4096 in bf16 27, 45 and 11; 5003 x 769 in fp32, read element by element, 9, 14 and 5.
//
// dw and db need a sum over all rows. Each workgroup of the backward pass walks rows with a stride
// of the grid and keeps its lanes' columns in registers; its row groups are added in LDS, and one
// row of partial sums per workgroup goes to memory. A second kernel adds these in their order, so
// that a result does not depend on the order in which workgroups ran (no atomics).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace xfh {

namespace {

constexpr int kThreads = 256;
constexpr int kRegisterCols = 8 * 8 * kThreads;       // widest row held in registers

template <typename T> __device__ __forceinline__ void load8(const T *p, float *o);
template <> __device__ __forceinline__ void load8<bf16>(const bf16 *p, float *o) {
  const bf16x8 v = *reinterpret_cast<const bf16x8 *>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = static_cast<float>(v[i]);
}
template <> __device__ __forceinline__ void load8<float>(const float *p, float *o) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 v = reinterpret_cast<const float4 *>(p)[i];
    o[4 * i] = v.x; o[4 * i + 1] = v.y; o[4 * i + 2] = v.z; o[4 * i + 3] = v.w;
  }
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float *o);
template <> __device__ __forceinline__ void store8<bf16>(bf16 *p, const float *o) {
  bf16x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<bf16>(o[i]);
  *reinterpret_cast<bf16x8 *>(p) = v;
}
template <> __device__ __forceinline__ void store8<float>(float *p, const float *o) {
#pragma unroll
  for (int i = 0; i < 2; ++i) reinterpret_cast<float4 *>(p)[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
}

// Where a lane's elements of a row are: in runs of 8 (VEC: C a multiple of 8, rows on 16 bytes),
// else one by one with the row's lanes side by side. Chunk c, element e.
template <int LPR, bool VEC> __device__ __forceinline__ int column(int sub, int c, int e) {
  return VEC ? (c * LPR + sub) * 8 + e : (c * 8 + e) * LPR + sub;
}
template <int LPR, int CH, bool VEC, typename T>
__device__ __forceinline__ void load_row(const T *row, int C, int sub, float (&v)[CH][8]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if constexpr (VEC) {
      const int at = column<LPR, VEC>(sub, c, 0);
      if (at < C) {
        load8(row + at, v[c]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = column<LPR, VEC>(sub, c, e);
        v[c][e] = at < C ? to_f32(row[at]) : 0.f;
      }
    }
  }
}
template <int LPR, int CH, bool VEC, typename T>
__device__ __forceinline__ void store_row(T *row, int C, int sub, const float (&v)[CH][8]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if constexpr (VEC) {
      const int at = column<LPR, VEC>(sub, c, 0);
      if (at < C) store8(row + at, v[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = column<LPR, VEC>(sub, c, e);
        if (at < C) row[at] = from_f32<T>(v[c][e]);
      }
    }
  }
}
// The same as stored (to be converted when they are used: loads of a row to come must not be waited for).
template <int LPR, int CH, bool VEC, typename T> struct RawRow {
  T v[CH][8];
  __device__ __forceinline__ void load(const T *row, int C, int sub) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if constexpr (VEC) {
        const int at = column<LPR, VEC>(sub, c, 0);
        typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
        constexpr int N = 8 * int(sizeof(T)) / 16;
        u32x4 u[N];
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = at < C ? reinterpret_cast<const u32x4 *>(row + at)[i] : u32x4{0, 0, 0, 0};
        __builtin_memcpy(v[c], u, sizeof(u));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = column<LPR, VEC>(sub, c, e);
          v[c][e] = at < C ? row[at] : T(0.f);
        }
      }
    }
  }
  __device__ __forceinline__ void get(float (&o)[CH][8]) const {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[c][e] = to_f32(v[c][e]);
  }
};
// A parameter vector in its own type (null: `absent` everywhere).
template <int LPR, int CH, bool VEC>
__device__ __forceinline__ void load_param(const void *p, int dtype, float absent, int C, int sub, float (&v)[CH][8]) {
  if (!p) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = absent;
  } else if (dtype == XFH_F32) {
    load_row<LPR, CH, VEC>(static_cast<const float *>(p), C, sub, v);
  } else {
    load_row<LPR, CH, VEC>(static_cast<const bf16 *>(p), C, sub, v);
  }
}

// Sums of N values over the LPR lanes of a row; `red` holds 4 N floats per call (LPR = 256).
template <int LPR, int N> __device__ __forceinline__ void row_sums(float (&s)[N], float *red) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = group_sum<LPR < 64 ? LPR : 64>(s[i]);
  if constexpr (LPR == 256) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[i * 4 + wave] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = (red[i * 4] + red[i * 4 + 1]) + (red[i * 4 + 2] + red[i * 4 + 3]);
  }
}

struct NormArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  float2 *stats;               // (mean, 1 / deviation) of each row
  float *partial;              // [2][blocks][C]
  int64_t rows, ldx, lddy;
  int C, w_dtype, b_dtype;
  float eps;
};

template <typename T, typename TO, int LPR, int CH, bool VEC>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(NormArgs a) {
  __shared__ float red[4];
  const int sub = threadIdx.x % LPR, C = a.C;
  const int64_t row = int64_t(blockIdx.x) * (kThreads / LPR) + threadIdx.x / LPR;
  if (LPR < 256 && row >= a.rows) return;              // (LPR = 256: the grid is the rows)
  float v[CH][8], w[CH][8], b[CH][8];
  load_row<LPR, CH, VEC>(static_cast<const T *>(a.x) + row * a.ldx, C, sub, v);
  load_param<LPR, CH, VEC>(a.w, a.w_dtype, 1.f, C, sub, w);
  load_param<LPR, CH, VEC>(a.b, a.b_dtype, 0.f, C, sub, b);
  float s[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] += v[c][e];
  row_sums<LPR, 1>(s, red);
  const float mean = s[0] / float(C);
  float q[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[c][e] -= mean;
      if (column<LPR, VEC>(sub, c, VEC ? 0 : e) < C) q[0] += v[c][e] * v[c][e];
    }
  row_sums<LPR, 1>(q, red);
  const float rstd = 1.0f / sqrtf(q[0] / float(C) + a.eps);
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * rstd * w[c][e] + b[c][e];
  store_row<LPR, CH, VEC>(static_cast<TO *>(a.y) + row * C, C, sub, v);
  if (a.stats && sub == 0) a.stats[row] = make_float2(mean, rstd);
}

// A row's dx (in g) from its x (in h; normalised on return) and dy (in g).
template <int LPR, int CH>
__device__ __forceinline__ void backward_row(float (&h)[CH][8], float (&g)[CH][8], const float (&w)[CH][8], float2 st, float inv,
                                             float *red) {
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // Beyond the row's end h is -mean/sigma, but g, and with it every sum, is zero there.
      h[c][e] = (h[c][e] - st.x) * st.y;
      g[c][e] *= w[c][e];
      s[0] += g[c][e];
      s[1] += g[c][e] * h[c][e];
    }
  row_sums<LPR, 2>(s, red);
  const float mg = s[0] * inv, mgh = s[1] * inv;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) g[c][e] = st.y * (g[c][e] - mg - h[c][e] * mgh);
}

template <typename T, typename TO, int LPR, int CH, bool VEC>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(NormArgs a) {
  constexpr int R = kThreads / LPR;                     // rows at a time
  __shared__ float red[8];
  __shared__ float sums[R > 1 ? LPR * 8 : 1][R > 1 ? R + 1 : 1];
  const int sub = threadIdx.x % LPR, group = threadIdx.x / LPR, C = a.C;
  float w[CH][8], dw[CH][8], db[CH][8];
  load_param<LPR, CH, VEC>(a.w, a.w_dtype, 1.f, C, sub, w);
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = db[c][e] = 0.f;
  const float inv = 1.0f / float(C);
  // The next row's loads are issued before the work on this one.
  const int64_t step = int64_t(gridDim.x) * R;
  RawRow<LPR, CH, VEC, T> xr;
  RawRow<LPR, CH, VEC, TO> gr;
  float2 next{};
  const auto fetch = [&](int64_t row) {
    xr.load(static_cast<const T *>(a.x) + row * a.ldx, C, sub);
    gr.load(static_cast<const TO *>(a.dy) + row * a.lddy, C, sub);
    next = a.stats[row];
  };
  int64_t row = int64_t(blockIdx.x) * R + group;
  if (VEC && row < a.rows) fetch(row);
  for (; row < a.rows; row += step) {
    float h[CH][8], g[CH][8], d[CH][8];
    if constexpr (!VEC) fetch(row);                      // (element by element it takes too many registers: 13.8 -> 17.7 us at 5003x769)
    xr.get(h);
    gr.get(g);
    const float2 st = next;
    if (VEC && row + step < a.rows) fetch(row + step);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) d[c][e] = g[c][e];
    backward_row<LPR, CH>(h, g, w, st, inv, red);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[c][e] += d[c][e] * h[c][e];
        db[c][e] += d[c][e];
      }
    if (a.dx) store_row<LPR, CH, VEC>(static_cast<T *>(a.dx) + row * C, C, sub, g);
  }
  if (!a.partial) return;
  float *pw = a.partial + int64_t(blockIdx.x) * C, *pb = pw + int64_t(gridDim.x) * C;
  if constexpr (R == 1) {
    store_row<LPR, CH, VEC>(pw, C, sub, dw);
    store_row<LPR, CH, VEC>(pb, C, sub, db);
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[sub * 8 + e][group] = which ? db[c][e] : dw[c][e];
        __syncthreads();
        for (int i = threadIdx.x; i < LPR * 8; i += kThreads) {
          const int at = column<LPR, VEC>(i / 8, c, i % 8);
          float t = 0.f;
#pragma unroll
          for (int r = 0; r < R; ++r) t += sums[i][r];
          if (at < C) (which ? pb : pw)[at] = t;
        }
      }
  }
}

// Rows wider than the registers hold: a workgroup per row, which it reads again for each sum (from
// the caches as far as they reach), and a second kernel with a thread per column for dw and db. It serves rows over
// 16384 elements, where a copy in registers would spill.
template <typename T, typename TO> __global__ __launch_bounds__(kThreads) void norm_forward_wide_kernel(NormArgs a) {
  __shared__ float red[4];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    TO *y = static_cast<TO *>(a.y) + row * a.C;
    float s[1] = {0.f}, q[1] = {0.f};
    for (int c = threadIdx.x; c < a.C; c += kThreads) s[0] += to_f32(x[c]);
    row_sums<256, 1>(s, red);
    const float mean = s[0] / float(a.C);
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float d = to_f32(x[c]) - mean;
      q[0] += d * d;
    }
    row_sums<256, 1>(q, red);
    const float rstd = 1.0f / sqrtf(q[0] / float(a.C) + a.eps);
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      float t = (to_f32(x[c]) - mean) * rstd;
      if (a.w) t *= load_any(a.w, a.w_dtype, c);
      if (a.b) t += load_any(a.b, a.b_dtype, c);
      y[c] = from_f32<TO>(t);
    }
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(mean, rstd);
  }
}

template <typename T, typename TO> __global__ __launch_bounds__(kThreads) void norm_backward_wide_kernel(NormArgs a) {
  __shared__ float red[8];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    const TO *dy = static_cast<const TO *>(a.dy) + row * a.lddy;
    T *dx = static_cast<T *>(a.dx) + row * a.C;
    const float2 st = a.stats[row];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float g = to_f32(dy[c]) * (a.w ? load_any(a.w, a.w_dtype, c) : 1.f);
      s[0] += g;
      s[1] += g * (to_f32(x[c]) - st.x) * st.y;
    }
    row_sums<256, 2>(s, red);
    const float mg = s[0] / float(a.C), mgh = s[1] / float(a.C);
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float g = to_f32(dy[c]) * (a.w ? load_any(a.w, a.w_dtype, c) : 1.f);
      dx[c] = from_f32<T>(st.y * (g - mg - (to_f32(x[c]) - st.x) * st.y * mgh));
    }
  }
}

template <typename T, typename TO> __global__ __launch_bounds__(kThreads) void norm_columns_kernel(NormArgs a) {
  const int c = int(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= a.C) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float2 st = a.stats[row];
    const float g = to_f32(static_cast<const TO *>(a.dy)[row * a.lddy + c]);
    dw += g * (to_f32(static_cast<const T *>(a.x)[row * a.ldx + c]) - st.x) * st.y;
    db += g;
  }
  a.partial[int64_t(blockIdx.y) * a.C + c] = dw;
  a.partial[(int64_t(gridDim.y) + blockIdx.y) * a.C + c] = db;
}

// out[which][c] = sum over the blocks' partial sums: 16 columns by 64 slices of blocks per workgroup (each
// slice 4 sums in flight), every sum in a fixed order. 4 us for 1024 x 128 sums, 11 for 1024 x 4096 (34 MB in all).
constexpr int kSlices = 64;
__global__ __launch_bounds__(16 * kSlices) void norm_params_kernel(const float *partial, int blocks, int C, void *dw,
                                                                   int dw_dtype, void *db, int db_dtype) {
  __shared__ float part[kSlices][17];
  void *out = blockIdx.y ? db : dw;
  if (!out) return;
  const int dtype = blockIdx.y ? db_dtype : dw_dtype;
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4, c = int(blockIdx.x) * 16 + col;
  const float *p = partial + int64_t(blockIdx.y) * blocks * C + c;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < C) {
    int r = slice;
    for (; r + 3 * kSlices < blocks; r += 4 * kSlices)
#pragma unroll
      for (int u = 0; u < 4; ++u) t[u] += p[int64_t(r + u * kSlices) * C];
    for (; r < blocks; r += kSlices) t[0] += p[int64_t(r) * C];
  }
  part[slice][col] = (t[0] + t[1]) + (t[2] + t[3]);
  for (int n = kSlices / 2; n > 0; n /= 2) {
    __syncthreads();
    if (slice < n) part[slice][col] += part[slice + n][col];
  }
  if (slice == 0 && c < C) {
    if (dtype == XFH_F32) static_cast<float *>(out)[c] = part[0][col];
    else static_cast<bf16 *>(out)[c] = bf16(part[0][col]);
  }
}

// The backward pass of few rows in one launch: workgroups [0, row_blocks) take the rows' dx, the others 64 columns of dw and
// db each, over all rows (4 slices of them, a wavefront each; the four sums of a column are added in order).
// Both read x and dy, of which there is little. 72 x 384 in fp32: 8.8 us of GPU time in the two launches
// above, 4.6 in this one; it is the launch that counts, since the host bounds such calls.
constexpr int64_t kFewRows = 256;
template <typename T, typename TO, int LPR, int CH, bool VEC>
__global__ __launch_bounds__(kThreads) void norm_backward_few_kernel(NormArgs a, int row_blocks, void *dw, int dw_dtype,
                                                                     void *db, int db_dtype) {
  constexpr int R = kThreads / LPR;
  __shared__ float red[8];
  __shared__ float2 part[4][64];
  const int C = a.C;
  if (int(blockIdx.x) >= row_blocks) {
    const int slice = threadIdx.x >> 6, c = (int(blockIdx.x) - row_blocks) * 64 + (threadIdx.x & 63);
    float sw = 0.f, sb = 0.f;
    if (c < C) {
#pragma unroll 4
      for (int64_t row = slice; row < a.rows; row += 4) {
        const float2 st = a.stats[row];
        const float g = to_f32(static_cast<const TO *>(a.dy)[row * a.lddy + c]);
        sw += g * ((to_f32(static_cast<const T *>(a.x)[row * a.ldx + c]) - st.x) * st.y);
        sb += g;
      }
    }
    part[slice][threadIdx.x & 63] = make_float2(sw, sb);
    __syncthreads();
    if (slice || c >= C) return;
    float2 t = part[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      t.x += part[i][threadIdx.x].x;
      t.y += part[i][threadIdx.x].y;
    }
    if (dw) {
      if (dw_dtype == XFH_F32) static_cast<float *>(dw)[c] = t.x;
      else static_cast<bf16 *>(dw)[c] = bf16(t.x);
    }
    if (db) {
      if (db_dtype == XFH_F32) static_cast<float *>(db)[c] = t.y;
      else static_cast<bf16 *>(db)[c] = bf16(t.y);
    }
    return;
  }
  const int sub = threadIdx.x % LPR;
  const int64_t row = int64_t(blockIdx.x) * R + threadIdx.x / LPR;
  if (LPR < 256 && row >= a.rows) return;              // (LPR = 256: a workgroup per row)
  float w[CH][8], h[CH][8], g[CH][8];
  load_row<LPR, CH, VEC>(static_cast<const T *>(a.x) + row * a.ldx, C, sub, h);
  load_row<LPR, CH, VEC>(static_cast<const TO *>(a.dy) + row * a.lddy, C, sub, g);
  load_param<LPR, CH, VEC>(a.w, a.w_dtype, 1.f, C, sub, w);
  const float2 st = a.stats[row];
  backward_row<LPR, CH>(h, g, w, st, 1.0f / float(C), red);
  store_row<LPR, CH, VEC>(static_cast<T *>(a.dx) + row * C, C, sub, g);
}

// Lanes and chunks of a row of C elements (chunks 0: wider than the registers hold).
struct RowShape { int lpr, ch; };
RowShape row_shape(int64_t C) {
  if (C <= 128) return {16, 1};
  if (C <= 256) return {16, 2};
  if (C <= 512) return {64, 1};
  if (C <= 1024) return {64, 2};
  for (int ch = 1; ch <= 8; ch *= 2)
    if (C <= int64_t(ch) * 8 * kThreads) return {256, ch};
  return {256, 0};
}

int64_t backward_blocks(int64_t rows, int64_t C) {
  const RowShape s = row_shape(C);
  if (s.ch == 0) return rows < 64 ? rows : 64;
  // A row of sums per workgroup: with rows that take a whole workgroup, half as many.
  const int64_t groups = ceil_div(rows, kThreads / s.lpr), most = 1024;
  return groups < most ? groups : most;
}

// Where the few rows' launch writes dw and db itself.
struct ParamGrads { void *dw; int dw_dtype; void *db; int db_dtype; };

bool few_rows(const NormArgs &a, const ParamGrads *p) { return p && a.rows <= kFewRows && row_shape(a.C).ch > 0; }

template <typename T, typename TO, int LPR, int CH>
int launch_shape(const NormArgs &a, bool vec, bool backward, int64_t blocks, const ParamGrads *p, hipStream_t s) {
  const dim3 grid{unsigned(blocks)};
  if (backward && few_rows(a, p)) {
    const int row_blocks = a.dx ? int(ceil_div(a.rows, int64_t(kThreads / LPR))) : 0, col_blocks = int(ceil_div(int64_t(a.C), int64_t(64)));
    const dim3 both{unsigned(row_blocks + col_blocks)};
    if (vec) norm_backward_few_kernel<T, TO, LPR, CH, true><<<both, kThreads, 0, s>>>(a, row_blocks, p->dw, p->dw_dtype, p->db, p->db_dtype);
    else norm_backward_few_kernel<T, TO, LPR, CH, false><<<both, kThreads, 0, s>>>(a, row_blocks, p->dw, p->dw_dtype, p->db, p->db_dtype);
  } else if (backward) {
    if (vec) norm_backward_kernel<T, TO, LPR, CH, true><<<grid, kThreads, 0, s>>>(a);
    else norm_backward_kernel<T, TO, LPR, CH, false><<<grid, kThreads, 0, s>>>(a);
  } else {
    if (vec) norm_forward_kernel<T, TO, LPR, CH, true><<<grid, kThreads, 0, s>>>(a);
    else norm_forward_kernel<T, TO, LPR, CH, false><<<grid, kThreads, 0, s>>>(a);
  }
  return check_launch("layer_norm_train");
}

template <typename T, typename TO> int launch_typed(const NormArgs &a, bool backward, const ParamGrads *p, hipStream_t s) {
  const RowShape shape = row_shape(a.C);
  const auto aligned = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool vec = a.C % 8 == 0 && a.ldx % 8 == 0 && (!backward || a.lddy % 8 == 0) && aligned(a.x) && aligned(a.dy) &&
                   aligned(a.w) && aligned(a.b) && aligned(a.y) && aligned(a.dx) && aligned(a.partial);
  // A grid holds fewer than 2^32 threads: more rows go in several launches (as a stride in the kernel they took 65
  // in place of 57 us at 589824x128).
  constexpr int64_t kMostBlocks = int64_t(1) << 22;
  const int64_t most_rows = kMostBlocks * (kThreads / shape.lpr);
  if (!backward && shape.ch > 0 && a.rows > most_rows) {
    for (int64_t row = 0; row < a.rows; row += most_rows) {
      NormArgs part = a;
      part.rows = std::min(most_rows, a.rows - row);
      part.x = static_cast<const T *>(a.x) + row * a.ldx;
      part.y = static_cast<TO *>(a.y) + row * a.C;
      if (a.stats) part.stats = a.stats + row;
      const int status = launch_typed<T, TO>(part, false, p, s);
      if (status != XFH_OK) return status;
    }
    return XFH_OK;
  }
  const int64_t blocks = backward ? backward_blocks(a.rows, a.C) : ceil_div(a.rows, int64_t(kThreads / shape.lpr));
  if (shape.ch == 0) {
    if (!backward) {
      norm_forward_wide_kernel<T, TO><<<dim3(unsigned(std::min(a.rows, kMostBlocks))), kThreads, 0, s>>>(a);
    } else {
      if (a.dx) norm_backward_wide_kernel<T, TO><<<dim3(unsigned(std::min(a.rows, kMostBlocks))), kThreads, 0, s>>>(a);
      if (a.partial)
        norm_columns_kernel<T, TO><<<dim3(unsigned(ceil_div(a.C, int64_t(kThreads))), unsigned(blocks)), kThreads, 0, s>>>(a);
    }
    return check_launch("layer_norm_train");
  }
  if (shape.lpr == 16 && shape.ch == 1) return launch_shape<T, TO, 16, 1>(a, vec, backward, blocks, p, s);
  if (shape.lpr == 16) return launch_shape<T, TO, 16, 2>(a, vec, backward, blocks, p, s);
  if (shape.lpr == 64 && shape.ch == 1) return launch_shape<T, TO, 64, 1>(a, vec, backward, blocks, p, s);
  if (shape.lpr == 64) return launch_shape<T, TO, 64, 2>(a, vec, backward, blocks, p, s);
  if (shape.ch == 1) return launch_shape<T, TO, 256, 1>(a, vec, backward, blocks, p, s);
  if (shape.ch == 2) return launch_shape<T, TO, 256, 2>(a, vec, backward, blocks, p, s);
  if (shape.ch == 4) return launch_shape<T, TO, 256, 4>(a, vec, backward, blocks, p, s);
  return launch_shape<T, TO, 256, 8>(a, vec, backward, blocks, p, s);
}

int launch_norm(const NormArgs &a, int x_dtype, int y_dtype, bool backward, const ParamGrads *p, hipStream_t s) {
  if (x_dtype == XFH_F32 && y_dtype == XFH_F32) return launch_typed<float, float>(a, backward, p, s);
  if (x_dtype == XFH_BF16 && y_dtype == XFH_BF16) return launch_typed<bf16, bf16>(a, backward, p, s);
  if (x_dtype == XFH_BF16 && y_dtype == XFH_F32) return launch_typed<bf16, float>(a, backward, p, s);
  return fail(XFH_EUNSUPPORTED, "layer_norm_train: x and y must be f32 and f32, bf16 and bf16, or bf16 and f32");
}

}  // namespace

int norm_train_forward(const void *x, int x_dtype, int64_t ldx, int64_t rows, int64_t cols, const void *w, int w_dtype,
                       const void *b, int b_dtype, float eps, void *y, int y_dtype, float *stats, hipStream_t s) {
  if (rows == 0 || cols == 0) return XFH_OK;
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.rows = rows; a.C = int(cols); a.w = w; a.w_dtype = w_dtype; a.b = b; a.b_dtype = b_dtype;
  a.eps = eps; a.y = y; a.stats = reinterpret_cast<float2 *>(stats);
  return launch_norm(a, x_dtype, y_dtype, false, nullptr, s);
}

int64_t norm_train_backward_workspace(int64_t rows, int64_t cols) {
  if (rows <= kFewRows && row_shape(cols).ch > 0) return 0;
  return 2 * backward_blocks(rows, cols) * cols * 4;
}

int norm_train_backward(const void *dy, int dy_dtype, int64_t lddy, const void *x, int x_dtype, int64_t ldx, int64_t rows,
                        int64_t cols, const void *w, int w_dtype, const float *stats, void *dx, void *dw, int dw_dtype,
                        void *db, int db_dtype, float *partial, hipStream_t s) {
  if (cols == 0) return XFH_OK;
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.rows = rows; a.C = int(cols); a.w = w; a.w_dtype = w_dtype;
  a.dx = dx; a.stats = reinterpret_cast<float2 *>(const_cast<float *>(stats));
  a.partial = dw || db ? partial : nullptr;
  const ParamGrads grads{dw, dw_dtype, db, db_dtype}, *params = dw || db ? &grads : nullptr;
  if (rows > 0 && (dx || params)) XFH_TRY(launch_norm(a, x_dtype, dy_dtype, true, params, s));
  if (!params || (rows > 0 && few_rows(a, params))) return XFH_OK;
  const int64_t blocks = backward_blocks(rows, cols);    // no rows: sums of nothing, zeros
  norm_params_kernel<<<dim3(unsigned(ceil_div(cols, int64_t(16))), 2), 16 * kSlices, 0, s>>>(partial, int(blocks), int(cols), dw,
                                                                                       dw_dtype, db, db_dtype);
  return check_launch("layer_norm_backward");
}

}  // namespace xfh
