// Layer norm, forward and backward.
//
//   mean = sum x / d, rstd = 1 / sqrt(sum (x - mean)^2 / d + eps), xh = (x - mean) rstd, y = xh w + b
//   h = dy w,  dx = rstd (h - mean(h) - xh mean(h xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound by memory traffic: the forward pass reads a row once and writes one, the backward pass reads two and
// writes one; a row stays in registers between the statistics and their use (the variance is formed from
// deviations of a mean that is already there, so a row with a large common offset loses nothing).  All sums in
// fp32.  A row belongs to WPR waves; with NE elements a lane, the widths up to 64 * WPR * NE are covered.
//
// Measured on 32768 x 4096 bf16: forward 97 us (0.54 GB: 5.5 TB/s), backward with dw and db 158 + 7 us (0.81 GB and 34 MB
// of partial sums: 5.1 TB/s), where a plain copy of 2 GiB reaches 4.95; on 4096 x 768: 5.5 and 8.4 + 2.3 us.
#include "rows.hpp"

namespace bgx {

constexpr int LN_MAX_D = 16384;
constexpr int LN_WAVES = 4;             // waves per workgroup
constexpr int LN_PARTS_MAX = 512;       // workgroups of a backward pass that form dw / db: rows of partial sums

struct NormArgs {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* y;              // forward: y; backward: dx
  float* mean;
  float* rstd;
  float* parts;         // backward: [workgroups][2][d] partial sums of dw, db
  void* dweight;        // backward in one launch: the gradients themselves
  void* dbias;
  int wdtype;
  int row_blocks;       // workgroups that work on rows; those behind sum columns
  int64_t rows;
  int64_t x_stride, dy_stride, y_stride;
  int d;
  float eps;
};

// Sum over the WPR waves of a row: with more than one, through LDS (slot: a pair of alternating buffers, so that
// one barrier per sum is enough).
template <int WPR>
__device__ inline float2 row_sum2(float2 v, float2 (*slot)[LN_WAVES], int& turn) {
  v.x = wave_sum(v.x);
  v.y = wave_sum(v.y);
  if constexpr (WPR > 1) {
    const int w = threadIdx.x / WAVE;
    if ((threadIdx.x & (WAVE - 1)) == 0) slot[turn][w] = v;
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < WPR; ++i) {
      s.x += slot[turn][i].x;
      s.y += slot[turn][i].y;
    }
    turn ^= 1;
    return s;
  }
  return v;
}

// How a row's columns fall to the lanes: chunk c of a lane starts at column (c * WPR * 64 + lane) * EPL.  Where a row is
// no whole number of chunks (RAGGED), the last one is moved back to end with the row -- every load and store stays one
// vector access without a branch around it, a column two lanes hold gets the same value from both, and the sums leave
// out the moved chunk's first `skip` elements.  Lanes past the row's end read the last chunk and count for nothing.
// Rows shorter than a chunk (TINY) go element by element.
enum LnMode { LN_WHOLE, LN_RAGGED, LN_TINY };

template <typename T, int NE, int WPR, int MODE>
struct LnRow {
  static constexpr int EPL = Chunk<T>::N, NC = NE / EPL;
  int first, d;
  __device__ LnRow(int d) : first(WPR == 1 ? threadIdx.x & (WAVE - 1) : threadIdx.x), d(d) {}
  __device__ int start(int c) const { return (c * WPR * WAVE + first) * EPL; }
  __device__ bool used(int c) const { return start(c) < d; }
  __device__ int at(int c) const { return MODE == LN_TINY ? start(c) : min(start(c), d - EPL); }
  // whether element e of chunk c is this lane's to count
  __device__ bool counts(int c, int e) const {
    if constexpr (MODE == LN_WHOLE) return used(c);
    if constexpr (MODE == LN_TINY) return start(c) + e < d;
    return used(c) && at(c) + e >= start(c);
  }
  template <typename U>
  __device__ void load(const U* row, int c, float* f) const {  // EPL elements of a type that may be wider than T
#pragma unroll
    for (int k = 0; k < EPL; k += Chunk<U>::N) Chunk<U>::unpack(load_raw(row, c, k), f + k);
  }
  template <typename U>
  __device__ uint4 load_raw(const U* row, int c, int k = 0) const {
    if constexpr (MODE == LN_TINY) return load_chunk_tail(row, min(start(c) + k, d), d);
    return load_chunk_any(row + at(c) + k);
  }
  __device__ void store(T* row, int c, const float* f) const {
    if (!used(c)) return;
    if constexpr (MODE == LN_TINY)
      store_chunk_tail(row, start(c), d, Chunk<T>::pack(f));
    else
      store_chunk_any(row + at(c), Chunk<T>::pack(f));
  }
  // sum over the chunk's elements that count
  template <typename F>
  __device__ float sum(int c, F f) const {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) s += MODE == LN_WHOLE || counts(c, e) ? f(e) : 0.f;
    return MODE == LN_WHOLE && !used(c) ? 0.f : s;
  }
};

template <typename T, typename WT, int NE, int WPR, int MODE>
__global__ __launch_bounds__(LN_WAVES* WAVE) void layernorm_forward_kernel(NormArgs A) {
  using Row = LnRow<T, NE, WPR, MODE>;
  constexpr int EPL = Row::EPL, NC = Row::NC;
  __shared__ float2 slot[2][LN_WAVES];
  int turn = 0;
  const Row row(A.d);
  const float over_d = 1.0f / A.d;
  const int64_t step = (int64_t)gridDim.x * (LN_WAVES / WPR);
  for (int64_t r = (int64_t)blockIdx.x * (LN_WAVES / WPR) + (WPR == 1 ? threadIdx.x / WAVE : 0); r < A.rows; r += step) {
    const T* xr = (const T*)A.x + r * A.x_stride;
    float x[NE];
    float2 s = make_float2(0.f, 0.f), q = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < NC; ++c) row.load(xr, c, x + c * EPL);
#pragma unroll
    for (int c = 0; c < NC; ++c) s.x += row.sum(c, [&](int e) { return x[c * EPL + e]; });
    const float mean = row_sum2<WPR>(s, slot, turn).x * over_d;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) x[c * EPL + e] -= mean;
      q.x += row.sum(c, [&](int e) { return x[c * EPL + e] * x[c * EPL + e]; });
    }
    const float rstd = 1.0f / sqrtf(row_sum2<WPR>(q, slot, turn).x * over_d + A.eps);
    T* yr = (T*)A.y + r * A.y_stride;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float w[EPL], b[EPL];
      row.load((const WT*)A.weight, c, w);
      if (A.bias != nullptr) {
        row.load((const WT*)A.bias, c, b);
      } else {
#pragma unroll
        for (int e = 0; e < EPL; ++e) b[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < EPL; ++e) b[e] = fmaf(x[c * EPL + e] * rstd, w[e], b[e]);
      row.store(yr, c, b);
    }
    if (A.mean != nullptr && row.first == 0) {
      A.mean[r] = mean;
      A.rstd[r] = rstd;
    }
  }
}

// PARAMS: the workgroup also sums dy xh and dy over its rows, column by column in registers (a lane keeps the same
// columns for every row), adds its waves' sums through LDS in a fixed order and writes one row of partial sums.  The
// next row's x and dy are on their way while a row is worked on (AHEAD; with 64 elements a lane there are no registers
// for it).
template <typename T, typename WT, int NE, int WPR, int MODE, bool PARAMS>
__device__ inline void backward_rows(const NormArgs& A, int blocks) {
  using Row = LnRow<T, NE, WPR, MODE>;
  constexpr int EPL = Row::EPL, NC = Row::NC;
  constexpr bool AHEAD = NE < 64;
  __shared__ float2 slot[2][LN_WAVES];
  __shared__ float colsum[PARAMS && WPR == 1 ? WAVE * NE : 1];
  int turn = 0;
  const Row row(A.d);
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const float over_d = 1.0f / A.d;
  const int64_t step = (int64_t)blocks * (LN_WAVES / WPR);
  float dw[PARAMS ? NE : 1], db[PARAMS ? NE : 1];
  if constexpr (PARAMS) {
#pragma unroll
    for (int e = 0; e < NE; ++e) dw[e] = db[e] = 0.f;
  }
  uint4 xv[NC], gv[NC];
  float mean = 0.f, rstd = 0.f;
  auto fetch = [&](int64_t i) {
    const int64_t r = A.rows - 1 - i;  // from the last row on: the forward pass's last rows may still be cached
    const T* xr = (const T*)A.x + r * A.x_stride;
    const T* gr = (const T*)A.dy + r * A.dy_stride;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      xv[c] = row.load_raw(xr, c);
      gv[c] = row.load_raw(gr, c);
    }
    mean = A.mean[r];
    rstd = A.rstd[r];
  };
  int64_t r = (int64_t)blockIdx.x * (LN_WAVES / WPR) + (WPR == 1 ? wave : 0);
  if (AHEAD && r < A.rows) fetch(r);
  for (; r < A.rows; r += step) {
    if constexpr (!AHEAD) fetch(r);
    float x[NE], h[NE];
    float2 s = make_float2(0.f, 0.f);  // sums of h and of h xh
    const float m = mean, f = rstd;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      Chunk<T>::unpack(xv[c], x + c * EPL);
      Chunk<T>::unpack(gv[c], h + c * EPL);
    }
    if constexpr (AHEAD) fetch(r + step < A.rows ? r + step : r);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float w[EPL];
      row.load((const WT*)A.weight, c, w);
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const int i = c * EPL + e;
        x[i] = (x[i] - m) * f;
        if constexpr (PARAMS) {  // columns that are another lane's, or none, are left out when the sums are written
          dw[i] = fmaf(h[i], x[i], dw[i]);
          db[i] += h[i];
        }
        h[i] *= w[e];
      }
      s.x += row.sum(c, [&](int e) { return h[c * EPL + e]; });
      s.y += row.sum(c, [&](int e) { return h[c * EPL + e] * x[c * EPL + e]; });
    }
    if (A.y == nullptr) continue;
    s = row_sum2<WPR>(s, slot, turn);
    const float mh = s.x * over_d, mx = s.y * over_d;
    T* dxr = (T*)A.y + (A.rows - 1 - r) * A.y_stride;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float o[EPL];
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = f * (h[c * EPL + e] - mh - x[c * EPL + e] * mx);
      row.store(dxr, c, o);
    }
  }
  if constexpr (PARAMS) {
    float* part = A.parts + (int64_t)blockIdx.x * 2 * A.d;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float* acc = which == 0 ? dw : db;
      if constexpr (WPR == 1) {
        for (int w = 1; w < LN_WAVES; ++w) {  // wave w hands its sums to wave 0
          __syncthreads();
          if (wave == w) {
#pragma unroll
            for (int e = 0; e < NE; ++e) colsum[e * WAVE + lane] = acc[e];
          }
          __syncthreads();
          if (wave == 0) {
#pragma unroll
            for (int e = 0; e < NE; ++e) acc[e] += colsum[e * WAVE + lane];
          }
        }
      }
      if (WPR > 1 || wave == 0) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < EPL; ++e)
            if (row.counts(c, e)) part[(int64_t)which * A.d + row.at(c) + e] = acc[c * EPL + e];
      }
    }
  }
}

template <typename T, typename WT, int NE, int WPR, int MODE, bool PARAMS>
__global__ __launch_bounds__(LN_WAVES* WAVE) void layernorm_backward_kernel(NormArgs A) {
  backward_rows<T, WT, NE, WPR, MODE, PARAMS>(A, gridDim.x);
}

// dw and db need a row's statistics only, which the forward pass has left: for few rows, workgroups behind those of the
// rows sum two chunks of columns each over all rows, 128 rows at a time, and everything is one launch without a
// workspace (x and dy are read twice, the second time from the caches).  Measured in one launch / in two: 1531 x 1001 fp32
// 13.2 / 12.9 us, 4096 x 768 bf16 29.6 / 11.6; 64 x 768 the same time on the card, and 4 us less of the caller's.
constexpr int LN_FEW = 1024;
template <typename T, int MODE>
__device__ inline void backward_columns(const NormArgs& A, int block) {
  constexpr int EPL = Chunk<T>::N, GROUPS = LN_WAVES * WAVE / 2;
  __shared__ float sums[GROUPS][2 * EPL * 2 + 1];
  const int lane = threadIdx.x & 1, group = threadIdx.x >> 1;
  const int start = (block * 2 + lane) * EPL, at = min(start, A.d - EPL);
  float dw[EPL], db[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) dw[e] = db[e] = 0.f;
#pragma unroll 4
  for (int64_t r = group; r < A.rows; r += GROUPS) {
    float x[EPL], g[EPL];
    Chunk<T>::unpack(load_chunk_any((const T*)A.x + r * A.x_stride + at), x);
    Chunk<T>::unpack(load_chunk_any((const T*)A.dy + r * A.dy_stride + at), g);
    const float mean = A.mean[r], rstd = A.rstd[r];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      dw[e] = fmaf(g[e], (x[e] - mean) * rstd, dw[e]);
      db[e] += g[e];
    }
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    sums[group][lane * EPL + e] = dw[e];
    sums[group][(2 + lane) * EPL + e] = db[e];
  }
  for (int half = GROUPS / 2; half > 0; half /= 2) {
    __syncthreads();
    for (int i = threadIdx.x; i < half * 4 * EPL; i += LN_WAVES * WAVE)
      sums[i / (4 * EPL)][i % (4 * EPL)] += sums[i / (4 * EPL) + half][i % (4 * EPL)];
  }
  __syncthreads();
  const int i = threadIdx.x;  // 2 x 2 x EPL sums
  if (i < 4 * EPL) {
    const int begin = (block * 2 + i / EPL % 2) * EPL, col = min(begin, A.d - EPL) + i % EPL;
    void* out = i < 2 * EPL ? A.dweight : A.dbias;
    if (begin < A.d && col >= begin && out != nullptr) store_as(out, col, sums[0][i], A.wdtype);
  }
}

template <typename T, typename WT, int NE, int WPR, int MODE>
__global__ __launch_bounds__(LN_WAVES* WAVE) void layernorm_backward_few_kernel(NormArgs A) {
  if ((int)blockIdx.x < A.row_blocks)
    backward_rows<T, WT, NE, WPR, MODE, false>(A, A.row_blocks);
  else
    backward_columns<T, MODE>(A, blockIdx.x - A.row_blocks);
}

// dw[c], db[c] = sum over the n_parts rows of partial sums, in a fixed order: 64 groups of rows per column, joined
// through LDS.  grid.y = 0: dw, 1: db.
constexpr int LN_COLS = 16, LN_GROUPS = 64;
__global__ __launch_bounds__(LN_COLS* LN_GROUPS) void layernorm_params_kernel(const float* __restrict__ parts, int n_parts,
                                                                              int d, void* dw, void* db, int dtype) {
  __shared__ float sums[LN_GROUPS][LN_COLS + 1];
  const int lane = threadIdx.x % LN_COLS, group = threadIdx.x / LN_COLS, col = blockIdx.x * LN_COLS + lane;
  const float* p = parts + (int64_t)blockIdx.y * d + min(col, d - 1);
  float s = 0.f;
#pragma unroll 8
  for (int i = group; i < n_parts; i += LN_GROUPS) s += p[(int64_t)i * 2 * d];
  sums[group][lane] = s;
  __syncthreads();
  for (int half = LN_GROUPS / 2; half > 0; half /= 2) {
    if (group < half) sums[group][lane] += sums[group + half][lane];
    __syncthreads();
  }
  void* out = blockIdx.y == 0 ? dw : db;
  if (group == 0 && col < d && out != nullptr) store_as(out, col, sums[0][lane], dtype);
}

static int ln_check(int64_t rows, int d, int dtype, int wdtype) {
  BGX_REQUIRE(rows >= 0 && d >= 1, BGX_E_ARG, "layer norm: rows=%lld d=%d", (long long)rows, d);
  BGX_REQUIRE(d <= LN_MAX_D, BGX_E_SHAPE, "layer norm: d=%d, the kernels hold rows of at most %d elements", d, LN_MAX_D);
  BGX_REQUIRE(dtype >= BGX_F32 && dtype <= BGX_BF16, BGX_E_DTYPE, "layer norm: dtype %d", dtype);
  BGX_REQUIRE(wdtype == dtype || wdtype == BGX_F32, BGX_E_DTYPE,
              "layer norm: weight dtype %d; it is that of x (%d) or fp32", wdtype, dtype);
  return 0;
}

static int ln_grid(int64_t rows, int wpr, int most) {
  const int64_t wgs = (rows + LN_WAVES / wpr - 1) / (LN_WAVES / wpr);
  return (int)(wgs < most ? wgs : most);
}

// Elements per lane and waves per row: one wave up to 2048 elements, the whole workgroup beyond.
#define BGX_LN_WIDTHS(d, CALL)      \
  if ((d) <= 512) CALL(8, 1)        \
  else if ((d) <= 1024) CALL(16, 1) \
  else if ((d) <= 2048) CALL(32, 1) \
  else if ((d) <= 4096) CALL(16, 4) \
  else if ((d) <= 8192) CALL(32, 4) \
  else CALL(64, 4)

template <typename T, typename WT>
static int ln_forward(const NormArgs& A, hipStream_t stream) {
#define BGX_LN_LAUNCH(NE, WPR, MODE) \
  layernorm_forward_kernel<T, WT, NE, WPR, MODE><<<ln_grid(A.rows, WPR, 8192), LN_WAVES * WAVE, 0, stream>>>(A)
#define BGX_LN_CALL(NE, WPR)                                \
  {                                                         \
    if (std::is_same<T, WT>::value && A.d % Chunk<T>::N == 0) \
      BGX_LN_LAUNCH(NE, WPR, (std::is_same<T, WT>::value ? LN_WHOLE : LN_RAGGED)); \
    else                                                    \
      BGX_LN_LAUNCH(NE, WPR, LN_RAGGED);                    \
  }
  if (A.d < Chunk<T>::N) BGX_LN_LAUNCH(8, 1, LN_TINY);
  else BGX_LN_WIDTHS(A.d, BGX_LN_CALL)
#undef BGX_LN_CALL
#undef BGX_LN_LAUNCH
  BGX_HIP(hipGetLastError());
  return 0;
}

template <typename T, typename WT, bool PARAMS>
static int ln_backward(const NormArgs& A, int grid, hipStream_t stream) {
#define BGX_LN_LAUNCH(NE, WPR, MODE) \
  layernorm_backward_kernel<T, WT, NE, WPR, MODE, PARAMS><<<grid, LN_WAVES * WAVE, 0, stream>>>(A)
#define BGX_LN_CALL(NE, WPR)                                \
  {                                                         \
    if (std::is_same<T, WT>::value && A.d % Chunk<T>::N == 0) \
      BGX_LN_LAUNCH(NE, WPR, (std::is_same<T, WT>::value ? LN_WHOLE : LN_RAGGED)); \
    else                                                    \
      BGX_LN_LAUNCH(NE, WPR, LN_RAGGED);                    \
  }
  if (A.d < Chunk<T>::N) BGX_LN_LAUNCH(8, 1, LN_TINY);
  else BGX_LN_WIDTHS(A.d, BGX_LN_CALL)
#undef BGX_LN_CALL
#undef BGX_LN_LAUNCH
  BGX_HIP(hipGetLastError());
  return 0;
}

template <typename T, typename WT>
static int ln_backward_few(const NormArgs& A, hipStream_t stream) {
  const int grid = A.row_blocks + (A.d + 2 * Chunk<T>::N - 1) / (2 * Chunk<T>::N);
#define BGX_LN_LAUNCH(NE, WPR, MODE) \
  layernorm_backward_few_kernel<T, WT, NE, WPR, MODE><<<grid, LN_WAVES * WAVE, 0, stream>>>(A)
#define BGX_LN_CALL(NE, WPR)                                \
  {                                                         \
    if (std::is_same<T, WT>::value && A.d % Chunk<T>::N == 0) \
      BGX_LN_LAUNCH(NE, WPR, (std::is_same<T, WT>::value ? LN_WHOLE : LN_RAGGED)); \
    else                                                    \
      BGX_LN_LAUNCH(NE, WPR, LN_RAGGED);                    \
  }
  BGX_LN_WIDTHS(A.d, BGX_LN_CALL)
#undef BGX_LN_CALL
#undef BGX_LN_LAUNCH
  BGX_HIP(hipGetLastError());
  return 0;
}

int layernorm_forward_impl(const void* x, int64_t x_stride, const void* weight, const void* bias, int wdtype,
                           int64_t rows, int d, int dtype, float eps, void* y, int64_t y_stride, float* mean,
                           float* rstd, void* stream) {
  if (int rc = ln_check(rows, d, dtype, wdtype)) return rc;
  if (rows == 0) return 0;
  BGX_REQUIRE(x && y && weight, BGX_E_ARG, "layer norm: null x, y or weight");
  BGX_REQUIRE((mean == nullptr) == (rstd == nullptr), BGX_E_ARG, "layer norm: mean and rstd come together");
  BGX_REQUIRE(x_stride >= d && y_stride >= d, BGX_E_ARG, "layer norm: row strides %lld, %lld below d=%d",
              (long long)x_stride, (long long)y_stride, d);
  NormArgs A{};
  A.x = x;
  A.weight = weight;
  A.bias = bias;
  A.y = y;
  A.mean = mean;
  A.rstd = rstd;
  A.rows = rows;
  A.x_stride = x_stride;
  A.y_stride = y_stride;
  A.d = d;
  A.eps = eps;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == BGX_F32) return ln_forward<float, float>(A, s);
  if (dtype == BGX_F16) return wdtype == BGX_F32 ? ln_forward<f16_t, float>(A, s) : ln_forward<f16_t, f16_t>(A, s);
  return wdtype == BGX_F32 ? ln_forward<bf16_t, float>(A, s) : ln_forward<bf16_t, bf16_t>(A, s);
}

static int ln_wpr(int d) { return d <= 2048 ? 1 : 4; }

// One launch for everything; rows shorter than the longest chunk of any type go the other way.
static bool ln_few(int64_t rows, int d) { return rows <= LN_FEW && d >= 8; }

size_t layernorm_backward_workspace_bytes(int64_t rows, int d) {
  if (rows <= 0 || d <= 0 || d > LN_MAX_D || ln_few(rows, d)) return 0;
  return (size_t)ln_grid(rows, ln_wpr(d), LN_PARTS_MAX) * 2 * d * sizeof(float);
}

int layernorm_backward_impl(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* weight,
                            int wdtype, const float* mean, const float* rstd, int64_t rows, int d, int dtype, void* dx,
                            int64_t dx_stride, void* dweight, void* dbias, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = ln_check(rows, d, dtype, wdtype)) return rc;
  hipStream_t s = (hipStream_t)stream;
  const bool params = dweight != nullptr || dbias != nullptr;
  if (!params && (dx == nullptr || rows == 0)) return 0;
  BGX_REQUIRE(rows == 0 || (dy && x && weight && mean && rstd), BGX_E_ARG, "layer norm backward: null operand");
  BGX_REQUIRE(rows == 0 || (x_stride >= d && dy_stride >= d && (dx == nullptr || dx_stride >= d)), BGX_E_ARG,
              "layer norm backward: row stride below d=%d", d);
  if (params) {
    const size_t need = layernorm_backward_workspace_bytes(rows, d);
    BGX_REQUIRE(need == 0 || (ws != nullptr && ws_bytes >= need), BGX_E_WORKSPACE,
                "layer norm backward: workspace of %zu bytes, %zu needed", ws_bytes, need);
  }
  const bool few = params && rows > 0 && ln_few(rows, d);
  const int parts = !params || few || rows == 0 ? 0 : ln_grid(rows, ln_wpr(d), LN_PARTS_MAX);
  if (rows > 0) {
    NormArgs A{};
    A.x = x;
    A.dy = dy;
    A.weight = weight;
    A.y = dx;
    A.mean = const_cast<float*>(mean);
    A.rstd = const_cast<float*>(rstd);
    A.parts = (float*)ws;
    A.dweight = dweight;
    A.dbias = dbias;
    A.wdtype = wdtype;
    A.rows = rows;
    A.x_stride = x_stride;
    A.dy_stride = dy_stride;
    A.y_stride = dx_stride;
    A.d = d;
    const int grid = parts ? parts : ln_grid(rows, ln_wpr(d), 8192);
    A.row_blocks = dx != nullptr ? grid : 0;
    int rc;
#define BGX_LN_BACKWARD(T, WT)                                 \
  rc = few      ? ln_backward_few<T, WT>(A, s)                 \
       : params ? ln_backward<T, WT, true>(A, grid, s)         \
                : ln_backward<T, WT, false>(A, grid, s)
    if (dtype == BGX_F32)
      BGX_LN_BACKWARD(float, float);
    else if (dtype == BGX_F16 && wdtype == BGX_F32)
      BGX_LN_BACKWARD(f16_t, float);
    else if (dtype == BGX_F16)
      BGX_LN_BACKWARD(f16_t, f16_t);
    else if (wdtype == BGX_F32)
      BGX_LN_BACKWARD(bf16_t, float);
    else
      BGX_LN_BACKWARD(bf16_t, bf16_t);
#undef BGX_LN_BACKWARD
    if (rc) return rc;
  }
  if (params && !few) {
    layernorm_params_kernel<<<dim3((d + LN_COLS - 1) / LN_COLS, 2), LN_COLS * LN_GROUPS, 0, s>>>(
        (const float*)ws, parts, d, dweight, dbias, wdtype);
    BGX_HIP(hipGetLastError());
  }
  return 0;
}

}  // namespace bgx
