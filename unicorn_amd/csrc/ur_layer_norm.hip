// ur_layer_norm.hip -- layer normalisation over the last dimension, forward and backward, with the sums of the
// weight's and the bias's gradients.
//
//   m = sum(x) / D      v = sum((x - m)^2) / D      r = 1 / sqrt(v + eps)      h = (x - m) r      y = h w + b
//   g = dy w            dx = r (g - mean(g) - h mean(g h))          dw = sum_rows(dy h)       db = sum_rows(dy)
//
// Everything is bound by memory: x is read once (dy too in the backward) and one result written, so a row stays in
// registers between its statistics and its result.  Statistics, sums and the arithmetic are fp32; a result is rounded to
// its type once.  The variance is the sum of squared differences from the mean already known (two passes over
// registers), not E[x^2] - m^2, which loses all its digits when the mean is large.
#include "ur_rows.h"

#include <algorithm>

using namespace ur;

namespace {

struct LnParams {
  const void* x;
  int64_t x_stride;
  const void* dy;
  int64_t dy_stride;
  const void* w;
  const void* b;
  int param_dtype;
  int64_t rows, cols;
  int64_t block0;  // the first workgroup of this launch
  float eps;
  void* y;  // forward: y; backward: dx
  float* mean;
  float* rstd;
  float* ws;      // partial results of this call
  int64_t chunk;  // long rows: elements of a row one workgroup takes
  int chunks;
  int parts;      // backward: workgroups that sum the parameters' gradients (0: not wanted), each with a row of `ws_parts`
  float* ws_parts;
  void* dw;
  void* db;
};

// A thread's vector of a row.  The vector that would reach over the row's end is moved back to end with the row: its first
// `skip` elements belong to the vector before it and are left out of sums (and stored twice, with the same value), so that no
// access is partial.  A vector wholly behind the end has skip >= kN.
template <typename T>
struct Span {
  int at, skip;
  __device__ __forceinline__ Span(int vec, int cols) {
    const int over = (vec + 1) * Elem<T>::kN - cols;
    skip = min(max(over, 0), Elem<T>::kN);
    at = min(vec * Elem<T>::kN, cols - Elem<T>::kN);
  }
};

// rows shorter than a vector are read element by element: `at` is negative there
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec load_span(const T* __restrict__ row, int at) {
  if (at >= 0) return *reinterpret_cast<const typename Elem<T>::Vec*>(row + at);
  typename Elem<T>::Vec v;
#pragma unroll
  for (int j = 0; j < Elem<T>::kN; ++j) v[j] = at + j >= 0 ? row[at + j] : (T)0.0f;
  return v;
}
template <typename T>
__device__ __forceinline__ void store_span(T* __restrict__ row, int at, typename Elem<T>::Vec v) {
  if (at >= 0) {
    *reinterpret_cast<typename Elem<T>::Vec*>(row + at) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < Elem<T>::kN; ++j)
    if (at + j >= 0) row[at + j] = v[j];
}

// parameters of a vector's columns as floats
template <typename T>
__device__ __forceinline__ void load_params(const void* p, int dtype, int64_t at, float missing, float (&out)[Elem<T>::kN]) {
  constexpr int N = Elem<T>::kN;
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = missing;
  } else if (dtype == UR_F32 && N == 8 && at >= 0) {
    const f32x4* f = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const f32x4 lo = f[0], hi = f[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[j] = lo[j];
      out[(4 + j) % N] = hi[j];
    }
  } else if (dtype == UR_F32 && N == 8) {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = at + j >= 0 ? static_cast<const float*>(p)[at + j] : missing;
  } else {
    const auto v = load_span<T>(static_cast<const T*>(p), at);
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = (float)v[j];
  }
}

// ---- rows that fit the registers of TPR threads, NV 16-byte vectors each -------------------------------------------
// Forward: 65536 x 1024 bf16 50 us (5.4 TB/s), 8192 x 4096 fp32 50 us (5.3), 6151 x 1926 fp16 of stride 1961 12.4 us (3.8: rows
// that start anywhere, and a short launch); 192 x 512 fp32 3.2 us, the latency of one row.  Rows that take a whole workgroup of
// 1024 threads are stored past the caches (2000 x 20000 fp32 77 us against 89; shorter rows lose: 65536 x 1024 bf16 51 against 49).
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR <= 64 ? 256 : TPR) k_ln_fwd(const LnParams P) {
  constexpr int N = Elem<T>::kN, kRows = TPR <= 64 ? 256 / TPR : 1;
  __shared__ float part[2][TPR <= 64 ? 1 : TPR / 64];
  const int t = threadIdx.x % TPR, cols = (int)P.cols;
  const int64_t want = (P.block0 + blockIdx.x) * kRows + threadIdx.x / TPR;
  const bool mine = want < P.rows;
  const int64_t row = mine ? want : P.rows - 1;  // (idle lanes take part in the lane exchanges)
  const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
  typename Elem<T>::Vec v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = load_span<T>(x, Span<T>(t + i * TPR, cols).at);
  float s[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int skip = Span<T>(t + i * TPR, cols).skip;
#pragma unroll
    for (int j = 0; j < N; ++j) s[0] += j >= skip ? (float)v[i][j] : 0.0f;
  }
  sum_threads<TPR, 1>(s, part[0]);
  const float inv_d = 1.0f / (float)P.cols;
  const float mean = s[0] * inv_d;
  float q[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int skip = Span<T>(t + i * TPR, cols).skip;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = j >= skip ? (float)v[i][j] - mean : 0.0f;
      q[0] = __builtin_fmaf(d, d, q[0]);
    }
  }
  sum_threads<TPR, 1>(q, part[1]);
  const float rstd = 1.0f / sqrtf(q[0] * inv_d + P.eps);
  if (mine && t == 0 && P.mean) {
    P.mean[row] = mean;
    P.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(P.y) + row * P.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Span<T> at(t + i * TPR, cols);
    if (at.skip >= N || !mine) continue;
    float w[N], b[N];
    load_params<T>(P.w, P.param_dtype, at.at, 1.0f, w);
    load_params<T>(P.b, P.param_dtype, at.at, 0.0f, b);
    typename Elem<T>::Vec o;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = (T)__builtin_fmaf(((float)v[i][j] - mean) * rstd, w[j], b[j]);
    if constexpr (TPR == 1024) store16_past<T>(y, at.at, P.cols, o);
    else store_span<T>(y, at.at, o);
  }
}

// Backward: workgroups of 1024 threads, 1024 / TPR rows at a time, walk over the rows with the next rows' loads in flight; a
// thread keeps its columns' weights and their sums of dy h and dy in registers on the way.  At the end the groups of threads
// are added in order and stored as one row of partial sums, which k_ln_param_sums adds up: no atomics, the same result
// every time.  Large workgroups, one for each CU, because every one of them leaves 2 D floats behind.
// 65536 x 1024 bf16 79 us + 4.7 for the sums (402 MB: 4.9 TB/s); with 512 workgroups 89.  8192 x 4096 fp32 82 us (4.9);
// 2048 x 16384 bf16 66 us, of which 26 go into the partial sums (33 MB written and read again).
constexpr int kBwdThreads = 1024, kBwdBlocks = 256;
// A thread adds at most so many rows' terms in fp32 before its sum joins the others in 64 bits (k_ln_param_sums): an fp32 sum
// loses up to half a step a term.  From 128 rounds of 256 workgroups on there are more workgroups than resident at once;
// their partial rows are 1/32 of x at the most.
constexpr int kSerialRows = 128;

// a workgroup's sum of one column (which: 0 weight, 1 bias): to its partial row, or, from the only workgroup, to the result
__device__ __forceinline__ void put_sum(const LnParams& P, int part, int which, int64_t col, float v) {
  if (P.parts > 1) {
    P.ws_parts[((int64_t)part * 2 + which) * P.cols + col] = v;
  } else {
    void* out = which ? P.db : P.dw;
    if (out) store_from_float(out, P.param_dtype, col, v);
  }
}

// adds up what lanes TPR, 2 TPR, ... apart hold
template <int TPR>
__device__ __forceinline__ float sum_subgroups(float v) {
  if constexpr (TPR <= 8) v += __uint_as_float(dpp32<0x128>(__float_as_uint(v)));  // (rotation by 8 of 16 lanes)
  if constexpr (TPR <= 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (TPR <= 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(kBwdThreads) k_ln_bwd(const LnParams P) {
  using Vec = typename Elem<T>::Vec;
  constexpr int N = Elem<T>::kN, kRows = kBwdThreads / TPR, kWavesPerRow = TPR > 64 ? TPR / 64 : 1;
  constexpr int kSets = TPR < 64 ? kBwdThreads / 64 : kRows;  // of sums, once a wave's groups are added
  __shared__ float part[2][kBwdThreads / 64][2];
  __shared__ float sums[kSets > 1 ? kSets : 1][kSets > 1 ? 2 * TPR * N : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, wave = threadIdx.x >> 6, cols = (int)P.cols;
  float w[NV][N], aw[NV][N], ab[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_params<T>(P.w, P.param_dtype, Span<T>(t + i * TPR, cols).at, 1.0f, w[i]);
#pragma unroll
    for (int j = 0; j < N; ++j) aw[i][j] = ab[i][j] = 0.0f;
  }
  const float inv_d = 1.0f / (float)P.cols;
  const int64_t groups = (P.rows + kRows - 1) / kRows;
  Vec v[NV], u[NV];
  float mean, rstd;
  const auto fetch = [&](int64_t rg, Vec (&xv)[NV], Vec (&dv)[NV], float& mu, float& rs) {
    const int64_t row = min(rg * kRows + sub, P.rows - 1);
    const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
    const T* dy = static_cast<const T*>(P.dy) + row * P.dy_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = Span<T>(t + i * TPR, cols).at;
      xv[i] = load_span<T>(x, at);
      dv[i] = load_span<T>(dy, at);
    }
    mu = P.mean[row];
    rs = P.rstd[row];
  };
  fetch(blockIdx.x, v, u, mean, rstd);
  int flip = 0;
  for (int64_t rg = blockIdx.x; rg < groups; rg += gridDim.x) {
    Vec v2[NV], u2[NV];
    float mean2, rstd2;
    fetch(min(rg + gridDim.x, groups - 1), v2, u2, mean2, rstd2);
    const bool mine = rg * kRows + sub < P.rows;
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int skip = mine ? Span<T>(t + i * TPR, cols).skip : N;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float h = ((float)v[i][j] - mean) * rstd, d = (float)u[i][j], g = d * w[i][j];
        if (j >= skip) {
          s[0] += g;
          s[1] = __builtin_fmaf(g, h, s[1]);
          aw[i][j] = __builtin_fmaf(d, h, aw[i][j]);
          ab[i][j] += d;
        }
      }
    }
    s[0] = reduce_lanes<(TPR < 64 ? TPR : 64), OpSum>(s[0]);
    s[1] = reduce_lanes<(TPR < 64 ? TPR : 64), OpSum>(s[1]);
    if constexpr (TPR > 64) {
      if ((threadIdx.x & 63) == 0) {
        part[flip][wave][0] = s[0];
        part[flip][wave][1] = s[1];
      }
      __syncthreads();
      s[0] = s[1] = 0.0f;
#pragma unroll
      for (int k = 0; k < kWavesPerRow; ++k) {
        s[0] += part[flip][sub * kWavesPerRow + k][0];
        s[1] += part[flip][sub * kWavesPerRow + k][1];
      }
      flip ^= 1;  // (the next row's partial sums go to the other half: one barrier a row is enough)
    }
    if (P.y != nullptr && mine) {
      const float c1 = s[0] * inv_d, c2 = s[1] * inv_d;
      T* dx = static_cast<T*>(P.y) + (rg * kRows + sub) * P.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Span<T> at(t + i * TPR, cols);
        if (at.skip >= N) continue;
        Vec o;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float h = ((float)v[i][j] - mean) * rstd, g = (float)u[i][j] * w[i][j];
          o[j] = (T)(rstd * (g - c1 - h * c2));
        }
        store_span<T>(dx, at.at, o);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = v2[i];
      u[i] = u2[i];
    }
    mean = mean2;
    rstd = rstd2;
  }
  if (P.parts == 0) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (kSets > 1) {
      const int set = TPR < 64 ? wave : sub;
      if constexpr (TPR < 64) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          aw[i][j] = sum_subgroups<TPR>(aw[i][j]);
          ab[i][j] = sum_subgroups<TPR>(ab[i][j]);
        }
      }
      if (i) __syncthreads();
      if (TPR >= 64 || (threadIdx.x & 63) < TPR) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          sums[set][t * N + j] = aw[i][j];
          sums[set][(TPR + t) * N + j] = ab[i][j];
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < 2 * TPR * N; c += kBwdThreads) {
        float total = 0.0f;
        for (int k = 0; k < kSets; ++k) total += sums[k][c];
        const int which = c / (TPR * N), vec = c % (TPR * N) / N, j = c % N;
        const Span<T> at(vec + i * TPR, cols);
        if (j >= at.skip) put_sum(P, blockIdx.x, which, at.at + j, total);
      }
    } else {
      const Span<T> at(t + i * TPR, cols);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j >= at.skip) {
          put_sum(P, blockIdx.x, 0, at.at + j, aw[i][j]);
          put_sum(P, blockIdx.x, 1, at.at + j, ab[i][j]);
        }
    }
  }
}

// Backward of few rows, in one launch: dx and the parameters' gradients depend on nothing but x, dy and the statistics, so some
// workgroups do rows (a wave each) and the others strips of 16 vectors of columns through all rows; what both read is in L2.
constexpr int kSmallThreads = 256, kStripVecs = 16, kStripRows = kSmallThreads / kStripVecs;
template <typename T>
__global__ void __launch_bounds__(kSmallThreads) k_ln_bwd_small(const LnParams P, int row_blocks) {
  using Vec = typename Elem<T>::Vec;
  constexpr int N = Elem<T>::kN;
  __shared__ float sums[kStripRows][2 * kStripVecs * N];
  const int cols = (int)P.cols, vecs = (cols + N - 1) / N;
  if ((int)blockIdx.x < row_blocks) {
    const int64_t row = (int64_t)blockIdx.x * (kSmallThreads / 64) + (threadIdx.x >> 6);
    if (row >= P.rows) return;
    const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
    const T* dy = static_cast<const T*>(P.dy) + row * P.dy_stride;
    T* dx = static_cast<T*>(P.y) + row * P.cols;
    const float mean = P.mean[row], rstd = P.rstd[row];
    float s0 = 0.0f, s1 = 0.0f;
    for (int v = threadIdx.x & 63; v < vecs; v += 64) {
      const Span<T> at(v, cols);
      const Vec xv = load_span<T>(x, at.at), dv = load_span<T>(dy, at.at);
      float w[N];
      load_params<T>(P.w, P.param_dtype, at.at, 1.0f, w);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j >= at.skip) {
          const float g = (float)dv[j] * w[j];
          s0 += g;
          s1 = __builtin_fmaf(g, ((float)xv[j] - mean) * rstd, s1);
        }
    }
    const float inv_d = 1.0f / (float)P.cols;
    const float c1 = reduce_lanes<64, OpSum>(s0) * inv_d, c2 = reduce_lanes<64, OpSum>(s1) * inv_d;
    for (int v = threadIdx.x & 63; v < vecs; v += 64) {
      const Span<T> at(v, cols);
      const Vec xv = load_span<T>(x, at.at), dv = load_span<T>(dy, at.at);
      float w[N];
      load_params<T>(P.w, P.param_dtype, at.at, 1.0f, w);
      Vec o;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float h = ((float)xv[j] - mean) * rstd;
        o[j] = (T)(rstd * ((float)dv[j] * w[j] - c1 - h * c2));
      }
      store_span<T>(dx, at.at, o);
    }
    return;
  }
  const int strip = blockIdx.x - row_blocks, t = threadIdx.x % kStripVecs, grp = threadIdx.x / kStripVecs;
  const Span<T> at(strip * kStripVecs + t, cols);
  float aw[N], ab[N];
#pragma unroll
  for (int j = 0; j < N; ++j) aw[j] = ab[j] = 0.0f;
#pragma unroll 4
  for (int64_t row = grp; row < P.rows; row += kStripRows) {
    const Vec xv = load_span<T>(static_cast<const T*>(P.x) + row * P.x_stride, at.at);
    const Vec dv = load_span<T>(static_cast<const T*>(P.dy) + row * P.dy_stride, at.at);
    const float mean = P.mean[row], rstd = P.rstd[row];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      aw[j] = __builtin_fmaf((float)dv[j], ((float)xv[j] - mean) * rstd, aw[j]);
      ab[j] += (float)dv[j];
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    sums[grp][t * N + j] = aw[j];
    sums[grp][(kStripVecs + t) * N + j] = ab[j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * kStripVecs * N; c += kSmallThreads) {
    float total = 0.0f;
    for (int g = 0; g < kStripRows; ++g) total += sums[g][c];
    const int which = c / (kStripVecs * N), vec = c % (kStripVecs * N) / N, j = c % N;
    const Span<T> to(strip * kStripVecs + vec, cols);
    void* out = which ? P.db : P.dw;
    if (out && j >= to.skip) store_from_float(out, P.param_dtype, to.at + j, total);
  }
}

// dw, db = the sums of the partial rows: 32 columns a workgroup (one 128-byte line of a partial row), up to 32 groups of
// threads over the partial rows (no more than there are of them: 64 x 65000 bf16, 8 rows, the backward 22.5 us against 28.5
// with 32), added in 64 bits and in a fixed order.
__global__ void __launch_bounds__(1024) k_ln_param_sums(const LnParams P) {
  __shared__ double acc[32][33];
  const int c = threadIdx.x & 31, grp = threadIdx.x >> 5, groups = blockDim.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;  // 0 .. 2 D
  double s = 0.0;
  if (col < 2 * P.cols)
    for (int p = grp; p < P.parts; p += groups) s += (double)P.ws_parts[(int64_t)p * 2 * P.cols + col];
  acc[grp][c] = s;
  __syncthreads();
  if (grp != 0 || col >= 2 * P.cols) return;
  double total = 0.0;
  for (int g = 0; g < groups; ++g) total += acc[g][c];
  if (col < P.cols) {
    if (P.dw) store_from_float(P.dw, P.param_dtype, col, (float)total);
  } else if (P.db) {
    store_from_float(P.db, P.param_dtype, col - P.cols, (float)total);
  }
}

// ---- long rows: a row is split over workgroups ----------------------------------------------------------------------
// Forward: (1) every chunk's mean and sum of squared differences from it, (2) each chunk's workgroup merges the row's
// chunks and writes its part.  x is read twice, the second time mostly from the caches, which the results' stores leave alone:
// 129 x 65536 fp32 5.5 + 11 us (34 MB each way; with ordinary stores 6 + 12.5; one workgroup a row, with 64 elements a thread,
// took 25).
constexpr int kLongThreads = 256, kLongVecs = 4;

// parameters of columns col ..., as far as they lie inside the row
template <typename T>
__device__ __forceinline__ void load_params_part(const void* p, int dtype, int64_t col, int64_t cols, float missing,
                                                 float (&out)[Elem<T>::kN]) {
  constexpr int N = Elem<T>::kN;
  if (p != nullptr && col + N <= cols) {
    load_params<T>(p, dtype, col, missing, out);
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = p != nullptr && col + j < cols ? load_as_float(p, dtype, col + j) : missing;
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads) k_ln_long_stats(const LnParams P) {
  constexpr int N = Elem<T>::kN;
  __shared__ float part[2][kLongThreads / 64];
  const int64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
  const int64_t c0 = (int64_t)blockIdx.x * P.chunk, c1 = min(c0 + P.chunk, P.cols);
  float n = 0.0f, mean = 0.0f, m2 = 0.0f;
  for (int64_t base = c0; base < c1; base += kLongThreads * kLongVecs * N) {
    typename Elem<T>::Vec v[kLongVecs];
    float s[1] = {0.0f}, q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < kLongVecs; ++i) {
      v[i] = load16<T>(x, base + (int64_t)(threadIdx.x + i * kLongThreads) * N, c1, (T)0.0f);
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += (float)v[i][j];
    }
    sum_threads<kLongThreads, 1>(s, part[0]);
    const float cnt = (float)min((int64_t)(kLongThreads * kLongVecs * N), c1 - base), m = s[0] / cnt;
#pragma unroll
    for (int i = 0; i < kLongVecs; ++i) {
      const int64_t left = c1 - (base + (int64_t)(threadIdx.x + i * kLongThreads) * N);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = (float)v[i][j] - m;
        if (j < left) q[0] = __builtin_fmaf(d, d, q[0]);
      }
    }
    sum_threads<kLongThreads, 1>(q, part[1]);
    // merge of two sets' means and squared sums
    const float d = m - mean, total = n + cnt;
    mean += d * (cnt / total);
    m2 += q[0] + d * d * (n * (cnt / total));
    n = total;
  }
  if (threadIdx.x == 0) {
    P.ws[(row * P.chunks + blockIdx.x) * 2] = mean;
    P.ws[(row * P.chunks + blockIdx.x) * 2 + 1] = m2;
  }
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads) k_ln_long_apply(const LnParams P) {
  constexpr int N = Elem<T>::kN;
  const int64_t row = blockIdx.y;
  const float* st = P.ws + row * P.chunks * 2;
  const int lane = threadIdx.x & 63;
  float s = 0.0f;
  for (int i = lane; i < P.chunks; i += 64)
    s = __builtin_fmaf(st[2 * i], (float)min(P.chunk, P.cols - i * P.chunk), s);
  const float mean = reduce_lanes<64, OpSum>(s) / (float)P.cols;
  float q = 0.0f;
  for (int i = lane; i < P.chunks; i += 64) {
    const float d = st[2 * i] - mean;
    q += st[2 * i + 1] + d * d * (float)min(P.chunk, P.cols - i * P.chunk);
  }
  const float rstd = 1.0f / sqrtf(reduce_lanes<64, OpSum>(q) / (float)P.cols + P.eps);
  if (blockIdx.x == 0 && threadIdx.x == 0 && P.mean) {
    P.mean[row] = mean;
    P.rstd[row] = rstd;
  }
  const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
  T* y = static_cast<T*>(P.y) + row * P.cols;
  const int64_t c0 = (int64_t)blockIdx.x * P.chunk, c1 = min(c0 + P.chunk, P.cols);
  for (int64_t col = c0 + (int64_t)threadIdx.x * N; col < c1; col += kLongThreads * N) {
    const auto v = load16<T>(x, col, c1, (T)0.0f);
    float w[N], b[N];
    load_params_part<T>(P.w, P.param_dtype, col, P.cols, 1.0f, w);
    load_params_part<T>(P.b, P.param_dtype, col, P.cols, 0.0f, b);
    typename Elem<T>::Vec o;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = (T)__builtin_fmaf(((float)v[j] - mean) * rstd, w[j], b[j]);
    store16_past<T>(y, col, c1, o);
  }
}

// Backward: (1) every chunk's sums of g and g h, (2) a workgroup takes a strip of columns through a range of rows: dx, and
// its columns' partial weight sums; (3) k_ln_param_sums.  x and dy are read twice: 1024 x 32768 bf16 77 us in all, 60 of them
// without the weights' gradients (82 and 65 with ordinary stores); 129 x 65536 fp32 36 us.
template <typename T>
__global__ void __launch_bounds__(kLongThreads) k_ln_long_bwd_sums(const LnParams P) {
  constexpr int N = Elem<T>::kN;
  __shared__ float part[2 * (kLongThreads / 64)];
  const int64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
  const T* dy = static_cast<const T*>(P.dy) + row * P.dy_stride;
  const float mean = P.mean[row], rstd = P.rstd[row];
  const int64_t c0 = (int64_t)blockIdx.x * P.chunk, c1 = min(c0 + P.chunk, P.cols);
  float s[2] = {0.0f, 0.0f};
  for (int64_t col = c0 + (int64_t)threadIdx.x * N; col < c1; col += kLongThreads * N) {
    const auto v = load16<T>(x, col, c1, (T)0.0f), u = load16<T>(dy, col, c1, (T)0.0f);
    float w[N];
    load_params_part<T>(P.w, P.param_dtype, col, P.cols, 1.0f, w);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float g = (float)u[j] * w[j];
      if (col + j < c1) {
        s[0] += g;
        s[1] = __builtin_fmaf(g, ((float)v[j] - mean) * rstd, s[1]);
      }
    }
  }
  sum_threads<kLongThreads, 2>(s, part);
  if (threadIdx.x == 0) {
    P.ws[(row * P.chunks + blockIdx.x) * 2] = s[0];
    P.ws[(row * P.chunks + blockIdx.x) * 2 + 1] = s[1];
  }
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads) k_ln_long_bwd_apply(const LnParams P) {
  constexpr int N = Elem<T>::kN;
  const int lane = threadIdx.x & 63;
  const int64_t col = ((int64_t)blockIdx.x * kLongThreads + threadIdx.x) * N;
  const bool inside = col < P.cols;
  float w[N], aw[N], ab[N];
  load_params_part<T>(P.w, P.param_dtype, inside ? col : 0, P.cols, 1.0f, w);
#pragma unroll
  for (int j = 0; j < N; ++j) aw[j] = ab[j] = 0.0f;
  struct Fetched {
    typename Elem<T>::Vec x, dy;
    float mean, rstd, s0, s1;
  };
  const int64_t at = inside ? col : 0;  // (idle threads read along: all lanes take part in the sums)
  const auto fetch = [&](int64_t row) {
    Fetched f;
    f.x = load16<T>(static_cast<const T*>(P.x) + row * P.x_stride, at, P.cols, (T)0.0f);
    f.dy = load16<T>(static_cast<const T*>(P.dy) + row * P.dy_stride, at, P.cols, (T)0.0f);
    f.mean = P.mean[row];
    f.rstd = P.rstd[row];
    f.s0 = f.s1 = 0.0f;
    const float* st = P.ws + row * P.chunks * 2;
    for (int i = lane; i < P.chunks; i += 64) {
      f.s0 += st[2 * i];
      f.s1 += st[2 * i + 1];
    }
    return f;
  };
  Fetched now = fetch(blockIdx.y);
  for (int64_t row = blockIdx.y; row < P.rows; row += gridDim.y) {
    const Fetched next = fetch(min(row + gridDim.y, P.rows - 1));
    const float c1 = reduce_lanes<64, OpSum>(now.s0) / (float)P.cols, c2 = reduce_lanes<64, OpSum>(now.s1) / (float)P.cols;
    typename Elem<T>::Vec o;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float h = ((float)now.x[j] - now.mean) * now.rstd, d = (float)now.dy[j];
      aw[j] = __builtin_fmaf(d, h, aw[j]);
      ab[j] += d;
      o[j] = (T)(now.rstd * (d * w[j] - c1 - h * c2));
    }
    if (P.y && inside) store16_past<T>(static_cast<T*>(P.y) + row * P.cols, col, P.cols, o);
    now = next;
  }
  if (P.parts == 0 || !inside) return;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (col + j < P.cols) {
      put_sum(P, blockIdx.y, 0, col + j, aw[j]);
      put_sum(P, blockIdx.y, 1, col + j, ab[j]);
    }
}

// ---- which kernel a call takes ---------------------------------------------------------------------------------------
struct LnPlan {
  int tpr, nv;      // threads a row and vectors a thread; tpr == 0: long rows, -1: backward of few rows in one launch
  int64_t chunk;    // long rows
  int chunks;
  int grid;         // backward: workgroups (register rows) or row ranges (long rows) = rows of partial sums
  int64_t ws_stats, ws_parts;  // floats
};

// Forward: few rows of more vectors than this are split as well (16 x 65000 bf16: 7.4 against 12.1 us; at 32768 columns or 128
// rows one workgroup a row is as good or better).
constexpr int kSplitVecs = 4096, kSplitRows = 64;
// Backward: up to this many rows and vectors in one launch (192 x 512 fp32: 3.7 against 6.8 us, and a launch less for the host;
// 512 x 512: 6.0 against 7.0, 1000 x 512: 10.1 against 7.6, 192 x 1926: 8.7 against 8.1).  The two cross between 512 and 1000 rows
// of 128 vectors; 256 keeps away from there, since what the strips lose grows with the rows and the gain does not.
constexpr int kSmallRows = 256, kSmallVecs = 128;
LnPlan ln_plan(int64_t rows, int64_t cols, int dtype, bool backward) {
  LnPlan p{};
  const int n = 16 / dtype_bytes(dtype);
  const int64_t vecs = ceil_div(cols, n);
  struct Shape { int tpr, nv; };
  static constexpr Shape kFwd[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {512, 2}, {512, 4}, {1024, 4},
                                   {1024, 8}};
  static constexpr Shape kBwd[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {128, 2}, {256, 2}, {512, 2}, {1024, 2}};
  const Shape* shapes = backward ? kBwd : kFwd;
  const int count = backward ? (int)(sizeof(kBwd) / sizeof(Shape)) : (int)(sizeof(kFwd) / sizeof(Shape));
  if (backward && rows <= kSmallRows && vecs <= kSmallVecs) {
    p.tpr = -1;
    return p;
  }
  const bool split = !backward && vecs > kSplitVecs && rows <= kSplitRows;
  for (int i = 0; i < count && !split; ++i)
    if (vecs <= (int64_t)shapes[i].tpr * shapes[i].nv) {
      p.tpr = shapes[i].tpr;
      p.nv = shapes[i].nv;
      break;
    }
  if (p.tpr) {
    const int64_t groups = ceil_div(rows, kBwdThreads / p.tpr);
    p.grid = (int)ceil_div(groups, std::min<int64_t>(ceil_div(groups, kBwdBlocks), kSerialRows));  // (all as many rows)
    p.ws_parts = backward && p.grid > 1 ? (int64_t)p.grid * 2 * cols : 0;
    return p;
  }
  // chunks of at least one vector a thread: about 1024 workgroups in all, at most 1024 for a row
  const int64_t step = (int64_t)kLongThreads * n;
  const int64_t per = std::max(ceil_div(cols, 1024), std::min<int64_t>(ceil_div(rows * cols, 1024), kLongVecs * step));
  p.chunk = ceil_div(per, step) * step;
  p.chunks = (int)ceil_div(cols, p.chunk);
  p.ws_stats = rows * p.chunks * 2;
  const int64_t strips = ceil_div(cols, (int64_t)kLongThreads * n);
  // row ranges: about 1024 workgroups, and 8 rows at least, kSerialRows at most, for the 2 D floats a range leaves behind (as far
  // as the grid's second dimension goes: 8.4 million rows of more than 4096 vectors are not in memory)
  p.grid = (int)std::min<int64_t>(ceil_div(rows, 8), ceil_div(1024, strips));
  p.grid = (int)std::max<int64_t>(p.grid, std::min<int64_t>(ceil_div(rows, kSerialRows), 65535));
  p.ws_parts = backward && p.grid > 1 ? (int64_t)p.grid * 2 * cols : 0;
  return p;
}

int check_common(const void* x, int64_t x_stride, int dtype, int param_dtype, int64_t rows, int64_t cols) {
  if (!x) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (!known_dtype(dtype)) return set_error(UR_ERR_INVALID_ARG, "bad dtype %d", dtype);
  if (param_dtype != dtype && param_dtype != UR_F32)
    return set_error(UR_ERR_INVALID_ARG, "parameters must have the input's type or fp32");
  if (rows <= 0 || cols <= 0) return set_error(UR_ERR_INVALID_ARG, "rows and cols must be positive");
  if (rows > 0x7fffffff || cols > 0x7fffffff) return set_error(UR_ERR_UNSUPPORTED, "rows and cols must be below 2^31");
  if (x_stride < cols && rows > 1) return set_error(UR_ERR_INVALID_ARG, "row stride below the row length");
  return UR_OK;
}

template <typename T>
int launch_fwd(const LnPlan& p, const LnParams& P, hipStream_t st) {
  if (p.tpr == 0) {
    for (int64_t r0 = 0; r0 < P.rows; r0 += 65535) {  // (the grid's second dimension holds 65535 rows)
      LnParams Q = P;
      Q.rows = std::min<int64_t>(65535, P.rows - r0);
      Q.x = static_cast<const T*>(P.x) + r0 * P.x_stride;
      Q.y = static_cast<T*>(P.y) + r0 * P.cols;
      Q.mean = P.mean ? P.mean + r0 : nullptr;
      Q.rstd = P.rstd ? P.rstd + r0 : nullptr;
      Q.ws = P.ws + r0 * P.chunks * 2;
      const dim3 grid(P.chunks, (unsigned)Q.rows);
      k_ln_long_stats<T><<<grid, kLongThreads, 0, st>>>(Q);
      k_ln_long_apply<T><<<grid, kLongThreads, 0, st>>>(Q);
    }
    return launch_status("ur_layer_norm_forward");
  }
  const int per = p.tpr <= 64 ? 256 / p.tpr : 1;
  in_pieces(ceil_div(P.rows, per), p.tpr <= 64 ? 256 : p.tpr, [&](int64_t first, unsigned grid) {
    LnParams Q = P;
    Q.block0 = first;
#define UR_LN(TPR, NV) \
  if (p.tpr == TPR && p.nv == NV) k_ln_fwd<T, TPR, NV><<<grid, TPR <= 64 ? 256 : TPR, 0, st>>>(Q);
    UR_LN(8, 1) UR_LN(16, 1) UR_LN(32, 1) UR_LN(64, 1) UR_LN(64, 2) UR_LN(64, 4) UR_LN(256, 2) UR_LN(512, 2) UR_LN(512, 4)
    UR_LN(1024, 4) UR_LN(1024, 8)
#undef UR_LN
  });
  return launch_status("ur_layer_norm_forward");
}

template <typename T>
int launch_bwd(const LnPlan& p, const LnParams& P, hipStream_t st) {
  if (p.tpr < 0) {
    const int row_blocks = P.y ? (int)ceil_div(P.rows, kSmallThreads / 64) : 0;
    const int strips = P.dw || P.db ? (int)ceil_div(P.cols, kStripVecs * Elem<T>::kN) : 0;
    k_ln_bwd_small<T><<<row_blocks + strips, kSmallThreads, 0, st>>>(P, row_blocks);
    return launch_status("ur_layer_norm_backward");
  }
  if (p.tpr == 0) {
    for (int64_t r0 = 0; r0 < P.rows; r0 += 65535) {
      LnParams Q = P;
      Q.rows = std::min<int64_t>(65535, P.rows - r0);
      Q.x = static_cast<const T*>(P.x) + r0 * P.x_stride;
      Q.dy = static_cast<const T*>(P.dy) + r0 * P.dy_stride;
      Q.mean = P.mean + r0;
      Q.rstd = P.rstd + r0;
      Q.ws = P.ws + r0 * P.chunks * 2;
      k_ln_long_bwd_sums<T><<<dim3(P.chunks, (unsigned)Q.rows), kLongThreads, 0, st>>>(Q);
    }
    const unsigned strips = (unsigned)ceil_div(P.cols, (int64_t)kLongThreads * Elem<T>::kN);
    k_ln_long_bwd_apply<T><<<dim3(strips, p.grid), kLongThreads, 0, st>>>(P);
  } else {
    const dim3 grid(p.grid);
#define UR_LN(TPR, NV) \
  if (p.tpr == TPR && p.nv == NV) k_ln_bwd<T, TPR, NV><<<grid, kBwdThreads, 0, st>>>(P);
    UR_LN(8, 1) UR_LN(16, 1) UR_LN(32, 1) UR_LN(64, 1) UR_LN(64, 2) UR_LN(128, 2) UR_LN(256, 2) UR_LN(512, 2) UR_LN(1024, 2)
#undef UR_LN
  }
  if (P.parts > 1) {
    int groups = 2;
    while (groups < 32 && groups < P.parts) groups *= 2;
    k_ln_param_sums<<<dim3((unsigned)ceil_div(2 * P.cols, 32)), 32 * groups, 0, st>>>(P);
  }
  return launch_status("ur_layer_norm_backward");
}

}  // namespace

extern "C" {

int64_t ur_layer_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype, int backward) {
  if (!known_dtype(dtype)) return set_error(UR_ERR_INVALID_ARG, "bad dtype %d", dtype);
  if (rows <= 0 || cols <= 0 || rows > 0x7fffffff || cols > 0x7fffffff)
    return set_error(UR_ERR_INVALID_ARG, "rows and cols must be positive and below 2^31");
  const LnPlan p = ln_plan(rows, cols, dtype, backward != 0);
  return (p.ws_stats + p.ws_parts) * 4;
}

int ur_layer_norm_forward(const void* x, int64_t x_row_stride, const void* weight, const void* bias, int dtype,
                          int param_dtype, int64_t rows, int64_t cols, float eps, void* y, float* mean, float* rstd,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_common(x, x_row_stride, dtype, param_dtype, rows, cols)) return rc;
  if (!y) return set_error(UR_ERR_INVALID_ARG, "null output pointer");
  if ((mean == nullptr) != (rstd == nullptr)) return set_error(UR_ERR_INVALID_ARG, "mean and rstd go together");
  if (!(eps >= 0.0f)) return set_error(UR_ERR_INVALID_ARG, "eps must not be negative");
  const LnPlan p = ln_plan(rows, cols, dtype, false);
  const size_t need = (size_t)(p.ws_stats + p.ws_parts) * 4;
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  LnParams P{};
  P.x = x; P.x_stride = x_row_stride; P.w = weight; P.b = bias; P.param_dtype = param_dtype;
  P.rows = rows; P.cols = cols; P.eps = eps; P.y = y; P.mean = mean; P.rstd = rstd;
  P.ws = static_cast<float*>(workspace); P.chunk = p.chunk; P.chunks = p.chunks;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) return launch_fwd<float>(p, P, st);
  if (dtype == UR_F16) return launch_fwd<_Float16>(p, P, st);
  return launch_fwd<__bf16>(p, P, st);
}

int ur_layer_norm_backward(const void* grad_y, int64_t grad_row_stride, const void* x, int64_t x_row_stride,
                           const void* weight, const float* mean, const float* rstd, int dtype, int param_dtype,
                           int64_t rows, int64_t cols, void* grad_x, void* grad_weight, void* grad_bias,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_common(x, x_row_stride, dtype, param_dtype, rows, cols)) return rc;
  if (!grad_y || !mean || !rstd) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (grad_row_stride < cols && rows > 1) return set_error(UR_ERR_INVALID_ARG, "row stride below the row length");
  if (!grad_x && !grad_weight && !grad_bias) return set_error(UR_ERR_INVALID_ARG, "no gradient asked for");
  const LnPlan p = ln_plan(rows, cols, dtype, true);
  const size_t need = (size_t)(p.ws_stats + p.ws_parts) * 4;
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  LnParams P{};
  P.x = x; P.x_stride = x_row_stride; P.dy = grad_y; P.dy_stride = grad_row_stride; P.w = weight;
  P.param_dtype = param_dtype; P.rows = rows; P.cols = cols; P.y = grad_x;
  P.mean = const_cast<float*>(mean); P.rstd = const_cast<float*>(rstd);
  P.ws = static_cast<float*>(workspace); P.chunk = p.chunk; P.chunks = p.chunks;
  P.parts = (grad_weight || grad_bias) ? p.grid : 0; P.ws_parts = P.ws + p.ws_stats;
  P.dw = grad_weight; P.db = grad_bias;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) return launch_bwd<float>(p, P, st);
  if (dtype == UR_F16) return launch_bwd<_Float16>(p, P, st);
  return launch_bwd<__bf16>(p, P, st);
}

}  // extern "C"
