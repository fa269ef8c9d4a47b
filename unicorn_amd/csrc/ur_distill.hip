// ur_distill.hip -- distillation from a teacher's top logits: per row, the divergence of the student's distribution over
// all V classes from the teacher's over the k classes whose logits are known.
//
//   p = softmax(t / T) over the row's filled slots        q = softmax(z / T) over V
//   loss = T^2 sum_j p_j (log p_j - log q_{i_j})          dz_v = g T (q_v - sum_{j: i_j = v} p_j)
//
// Bound by memory: the forward reads z once (running maximum and sum of exponentials), the backward reads it again and
// writes the gradient.  Sums are fp32; log p - log q, a difference that is small where the student has learnt, is formed in 64
// bits.
#include "ur_rows.h"

#include <algorithm>

using namespace ur;

namespace {

constexpr double kLog2e = 1.44269504088896340736;
constexpr int kThreads = 256;   // workgroups that take several rows
constexpr int kMaxTop = 1024;   // slots of a row: the backward keeps their classes and shares in LDS
constexpr int kGroupTop = 64;   // ... where a workgroup takes several rows

struct DistillParams {
  const void* z;
  int64_t stride;
  int64_t rows, cols;
  int64_t block0;  // the first workgroup of this launch
  const void* t;
  int t_dtype;
  const void* index;
  bool index64;
  int top;
  double temperature;
  float scale;     // log2(e) / T
  double scale64, inv_t;  // the same in 64 bits; 1 / T
  float* stats;  // (rows, 2): maximum of z, sum of exp((z - max) / T)
  float* loss;   // (rows) or one value
  int reduction;
  double* partial;  // reductions: (partials, 2) sums of losses and numbers of rows that have a teacher
  int64_t partials;
  float* split_stats;  // split rows: (rows, splits, 2) maxima and sums of the parts
  int splits;
  int64_t chunk;
  const float* g;
  int64_t g_stride;
  void* grad;
};

__device__ __forceinline__ int64_t slot_class(const DistillParams& P, int64_t row, int j) {
  const int64_t i = row * P.top + j;
  return P.index64 ? static_cast<const int64_t*>(P.index)[i] : (int64_t)static_cast<const int32_t*>(P.index)[i];
}

// exp((v - m) / T), scale = log2(e) / T, by the hardware's exponential (1 ulp) of a product that is rounded once, which costs
// |v - m| / T 2^-24 beside it.  (With the product's rest as a second term 5 to 7 % slower and no nearer to 64 bits: an fp32
// gradient is off by 1.1e-7 of its norm either way, the formulas in torch's fp32 operations by 1.25e-7.)  An infinite maximum makes inf - inf of the equal ones, as the definition does.
__device__ __forceinline__ float exp_diff(float v, float m, float scale) { return __builtin_amdgcn_exp2f((v - m) * scale); }

// exp((v - m) / T) to 2 ulp whatever the size of the argument: the argument is formed in 64 bits and split into a whole
// power of two and a rest in [-1/2, 1/2] (a slot's share of the teacher; a 64-bit exponential costs ten times as much)
__device__ __forceinline__ float exp_slot(float v, float m, double scale) {
  const double y = ((double)v - (double)m) * scale, whole = rint(y);
  if (y < -150.0) return 0.0f;
  return __builtin_ldexpf(__builtin_amdgcn_exp2f((float)(y - whole)), (int)whole);
}

// merges (m, s) of two sets of numbers: s is relative to m; m = -inf with s = 0 is the empty set
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float scale) {
  const float top = __builtin_fmaxf(m, m2);
  if (top == -__builtin_inff()) {
    s += s2;  // (both empty, or NaN)
    return;
  }
  s = (m == top ? s : s * exp_diff(m, top, scale)) + (m2 == top ? s2 : s2 * exp_diff(m2, top, scale));
  m = top;
}

// Running maximum and sum of row elements [c0, c1), threads t, t + n, ... of a group: B loads at a time, one rescaling of the
// sum for each batch that holds a new maximum.
template <typename T, int B>
__device__ __forceinline__ void add_batch(const typename Elem<T>::Vec (&v)[B], float scale, float& m, float& s) {
  constexpr int N = Elem<T>::kN;
  float top = (float)v[0][0];
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int j = 0; j < N; ++j) top = __builtin_fmaxf(top, (float)v[b][j]);
  if (top > m) {
    s = m == -__builtin_inff() ? s : s * exp_diff(m, top, scale);
    m = top;
  }
  const float ref = m == -__builtin_inff() ? 0.0f : m;  // (nothing but -inf so far: every term is 0)
  float part[B] = {};
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int j = 0; j < N; ++j) part[b] += exp_diff((float)v[b][j], ref, scale);
#pragma unroll
  for (int b = 0; b < B; ++b) s += part[b];
}

// The vector at `col` of a range that ends at c1 and holds at least one vector: where it would reach over the end it is moved
// back to end there, and what belongs to the vector before it reads as `fill`.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec load_back(const T* __restrict__ z, int64_t col, int64_t c1, T fill) {
  constexpr int N = Elem<T>::kN;
  const int64_t at = min(col, c1 - N);
  auto v = *reinterpret_cast<const typename Elem<T>::Vec*>(z + at);
  const int skip = (int)min(col - at, (int64_t)N);
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = j < skip ? fill : v[j];
  return v;
}

template <typename T, int B>
__device__ __forceinline__ void row_part(const T* __restrict__ z, int64_t c0, int64_t c1, int t, int n, float scale, float& m,
                                         float& s) {
  constexpr int N = Elem<T>::kN;
  using Vec = typename Elem<T>::Vec;
  m = -__builtin_inff();
  s = 0.0f;
  const int64_t step = (int64_t)n * N;
  for (int64_t col = c0 + (int64_t)t * N; col < c1; col += B * step) {
    Vec v[B];
    if (col + (B - 1) * step + N <= c1) {
#pragma unroll
      for (int b = 0; b < B; ++b) v[b] = *reinterpret_cast<const Vec*>(z + col + b * step);
    } else if (c1 - c0 >= N) {
#pragma unroll
      for (int b = 0; b < B; ++b) v[b] = load_back<T>(z, col + b * step, c1, (T)-__builtin_inff());
    } else {
#pragma unroll
      for (int b = 0; b < B; ++b) v[b] = load16<T>(z, col + b * step, c1, (T)-__builtin_inff());
    }
    add_batch<T, B>(v, scale, m, s);
  }
}

template <int L>
__device__ __forceinline__ void merge_lanes(float& m, float& s, float scale) {
  const float top = reduce_lanes<L, OpMax>(m);
  if (top != -__builtin_inff() && m != top) s *= exp_diff(m, top, scale);
  s = reduce_lanes<L, OpSum>(s);
  m = top;
}

template <int L>
__device__ __forceinline__ bool any_lane(bool v) {
  const uint64_t b = __ballot(v);
  if (L == 64) return b != 0;
  return ((b >> ((threadIdx.x & 63) / L * L)) & ((1ull << (L & 63)) - 1)) != 0;
}

// A slot of a row's teacher, and (where z is given) the student's logit of its class.
struct Slot {
  int cls;    // -1: empty, -2: a class that there is none of
  float t, z;
};
template <typename T>
__device__ __forceinline__ Slot slot_at(const DistillParams& P, int64_t row, const T* __restrict__ z, int j) {
  Slot s{-1, 0.0f, 0.0f};
  if (j >= P.top) return s;
  const int64_t c = slot_class(P, row, j);
  if (c < 0) return s;
  s.t = load_as_float(P.t, P.t_dtype, row * P.top + j);
  s.cls = c < P.cols ? (int)c : -2;
  if (z != nullptr && c < P.cols) s.z = (float)z[c];
  return s;
}

// The teacher of a row, by L lanes: maximum and sum of exponentials of its filled slots, and whether there is one; a class
// outside [0, V) makes the sum NaN.  `own`: slot threadIdx.x % L, fetched before the row was read (its two dependent
// loads would stand at the end of every row otherwise).  With kLoss also sum_j e_j ((t_j - max t) - (z_j - z_max)), of which
// the loss is made.
struct Teacher {
  float m, e;  // maximum; the own slot's exponential
  double s, cross;
  bool any;
};
template <typename T, int L, bool kLoss>
__device__ __forceinline__ Teacher row_teacher(const DistillParams& P, int64_t row, const T* __restrict__ z, const Slot& own,
                                               float z_max) {
  const int lane = threadIdx.x % L;
  float m = -__builtin_inff();
  bool any = false, bad = false;
  Slot at = own;
  for (int j = lane; j < P.top; j += L) {
    if (j != lane) at = slot_at<T>(P, row, static_cast<const T*>(nullptr), j);
    if (at.cls == -1) continue;
    bad |= at.cls == -2 || at.t != at.t;
    any |= at.t != -__builtin_inff();
    m = __builtin_fmaxf(m, at.t);
  }
  m = reduce_lanes<L, OpMax>(m);
  bad = any_lane<L>(bad);
  any = any_lane<L>(any) || bad;
  Teacher r{m, 0.0f, 0.0, 0.0, any};
  at = own;
  for (int j = lane; j < P.top; j += L) {
    if (j != lane) at = slot_at<T>(P, row, kLoss ? z : nullptr, j);
    if (at.cls == -1) continue;
    const float e = exp_slot(at.t, m, P.scale64);
    if (j == lane) r.e = e;
    r.s += (double)e;
    if (kLoss && e != 0.0f)
      r.cross = __builtin_fma((double)e, ((double)at.t - (double)m) - ((double)at.z - (double)z_max), r.cross);
  }
  r.s = bad ? __builtin_nan("") : sum_lanes<L>(r.s);
  if (kLoss) r.cross = sum_lanes<L>(r.cross);
  return r;
}

// Loss of a row from its softmax statistics, by L lanes; keeps the statistics and, without a reduction, stores the loss.
//   sum_j p_j (log p_j - log q_j) = sum_j p_j ((t_j - max t) - (z_j - max z)) / T + log(sum exp z / sum exp t)
template <typename T, int L>
__device__ __forceinline__ double row_loss(const DistillParams& P, int64_t row, const T* __restrict__ z, const Slot& own, float m,
                                           float s, bool store, bool& taught) {
  const Teacher teacher = row_teacher<T, L, true>(P, row, z, own, m);
  taught = teacher.any;
  const double inv_s = 1.0 / teacher.s;
  const double loss =
      teacher.any ? (teacher.cross * inv_s * P.inv_t + log((double)s * inv_s)) * P.temperature * P.temperature : 0.0;
  if (threadIdx.x % L == 0 && store) {
    if (P.stats) {
      P.stats[2 * row] = m;
      P.stats[2 * row + 1] = s;
    }
    if (P.reduction == UR_REDUCE_NONE) P.loss[row] = (float)loss;
  }
  return loss;  // (a reduction adds the rows in 64 bits and rounds once)
}

// the reduced loss from the sum of the rows' losses and the number of rows that have a teacher; keeps the factor for the
// backward
__device__ __forceinline__ void reduced_loss(const DistillParams& P, double sum, double taught) {
  const double factor = P.reduction == UR_REDUCE_MEAN ? 1.0 / (taught > 0.0 ? taught : 1.0) : 1.0;
  P.loss[0] = (float)(sum * factor);
  if (P.stats) P.stats[2 * P.rows] = (float)factor;
}

// Forward, L lanes a row (a row of few classes), kThreads / L rows a workgroup.  100000 x 6 fp32 13 us, 30000 x 128 bf16 10,
// 32768 x 1000 bf16 32 us (2.1 TB/s; 21 without the teacher's part): bound by the teacher's 64-bit arithmetic, once a wave.
template <typename T, int L>
__global__ void __launch_bounds__(kThreads) k_distill_fwd_rows(const DistillParams P) {
  constexpr int R = kThreads / L;
  __shared__ double part[2][R];
  const int t = threadIdx.x % L, sub = threadIdx.x / L;
  const int64_t want = (P.block0 + blockIdx.x) * R + sub;
  const bool mine = want < P.rows;
  const int64_t row = mine ? want : P.rows - 1;  // (idle lanes take part in the exchanges)
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  const float scale = P.scale;
  const Slot own = slot_at<T>(P, row, z, t);
  float m, s;
  row_part<T, 2>(z, 0, P.cols, t, L, scale, m, s);
  merge_lanes<L>(m, s, scale);
  bool taught;
  const double loss = row_loss<T, L>(P, row, z, own, m, s, mine, taught);
  if (P.partial == nullptr) return;
  if (t == 0) {
    part[0][sub] = mine ? loss : 0.0;
    part[1][sub] = mine && taught ? 1.0 : 0.0;
  }
  __syncthreads();
  if (threadIdx.x) return;
  double a = 0.0, n = 0.0;
  for (int r = 0; r < R; ++r) {
    a += part[0][r];
    n += part[1][r];
  }
  if (P.partials == 1) {
    reduced_loss(P, a, n);
  } else {
    P.partial[2 * (P.block0 + blockIdx.x)] = a;
    P.partial[2 * (P.block0 + blockIdx.x) + 1] = n;
  }
}

// a workgroup's maximum and sum, in every thread
template <int W>
__device__ __forceinline__ void merge_waves(float (&part)[2][W], float& m, float& s, float scale) {
  merge_lanes<64>(m, s, scale);
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = m;
    part[1][threadIdx.x >> 6] = s;
  }
  __syncthreads();
  m = part[0][0];
  s = part[1][0];
  for (int w = 1; w < W; ++w) merge(m, s, part[0][w], part[1][w], scale);
}

template <typename T>
__device__ __forceinline__ void finish_row(const DistillParams& P, int64_t row, const T* z, const Slot& own, float m, float s) {
  bool taught;
  const double loss = row_loss<T, 64>(P, row, z, own, m, s, true, taught);
  if (P.partial && threadIdx.x == 0) {
    P.partial[2 * row] = loss;
    P.partial[2 * row + 1] = taught ? 1.0 : 0.0;
  }
}

// Forward, one workgroup a row.  8192 x 32768 bf16 101 us by itself (5.3 TB/s; 512 and 1024 threads 113 and 180), 111 between the
// backwards of a training step (4.8), 4096 x 32768 fp32 98 us (5.5), 2000 x 20000 fp32 39 us (4.1), 4096 x 8101 fp16 17 us (3.9
// TB/s: one exponential and six other instructions an element, and the teacher at each row's end).
template <typename T>
__global__ void __launch_bounds__(kThreads) k_distill_fwd(const DistillParams P) {
  __shared__ float part[2][kThreads / 64];
  const int64_t row = P.block0 + blockIdx.x;
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  const float scale = P.scale;
  Slot own{-1, 0.0f, 0.0f};
  if (threadIdx.x < 64) own = slot_at<T>(P, row, z, threadIdx.x);
  float m, s;
  row_part<T, 4>(z, 0, P.cols, threadIdx.x, kThreads, scale, m, s);
  merge_waves(part, m, s, scale);
  if (threadIdx.x < 64) finish_row<T>(P, row, z, own, m, s);
}

// Forward, too few rows to fill the chip: a row is split over workgroups, whose maxima and sums a second launch merges.
// 3 x 131071 bf16: 3.1 + 3.7 us, two latencies; one workgroup a row took 29.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_distill_split(const DistillParams P) {
  __shared__ float part[2][kThreads / 64];
  const int64_t row = blockIdx.y, c0 = (int64_t)blockIdx.x * P.chunk;
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  const float scale = P.scale;
  float m, s;
  row_part<T, 1>(z, c0, min(c0 + P.chunk, P.cols), threadIdx.x, kThreads, scale, m, s);
  merge_waves(part, m, s, scale);
  if (threadIdx.x == 0) {
    float* out = P.split_stats + 2 * (row * P.splits + blockIdx.x);
    out[0] = m;
    out[1] = s;
  }
}
template <typename T>
__global__ void __launch_bounds__(64) k_distill_join(const DistillParams P) {
  const int64_t row = blockIdx.x;
  const float scale = P.scale;
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  const Slot own = slot_at<T>(P, row, z, threadIdx.x);
  float m = -__builtin_inff(), s = 0.0f;
  for (int i = threadIdx.x; i < P.splits; i += 64) {
    const float* in = P.split_stats + 2 * (row * P.splits + i);
    merge(m, s, in[0], in[1], scale);
  }
  merge_lanes<64>(m, s, scale);
  finish_row<T>(P, row, z, own, m, s);
}

// sum or mean of the rows' losses, in 64 bits and in a fixed order
__global__ void __launch_bounds__(1024) k_distill_reduce(const DistillParams P) {
  __shared__ double part[2][16];
  double a = 0.0, n = 0.0;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < P.partials; r += 1024) {
    a += P.partial[2 * r];
    n += P.partial[2 * r + 1];
  }
  a = sum_lanes<64>(a);
  n = sum_lanes<64>(n);
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = a;
    part[1][threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  a = n = 0.0;
  for (int w = 0; w < 16; ++w) {
    a += part[0][w];
    n += part[1][w];
  }
  reduced_loss(P, a, n);
}

// ---- backward: all of q first, then the teacher's classes are written again with their shares taken off.  A class that
// several slots name gets the sum of their shares, written by the first of them.

// classes and shares of a row's slots, by L lanes; returns 0: no teacher, 1: a teacher, 2: NaN
template <typename T, int L>
__device__ __forceinline__ int row_shares(const DistillParams& P, int64_t row, int* cls, float* share) {
  constexpr const T* kNoLogits = nullptr;
  Slot at = slot_at<T>(P, row, kNoLogits, threadIdx.x % L);
  const Teacher teacher = row_teacher<T, L, false>(P, row, kNoLogits, at, 0.0f);
  const float inv_s = (float)(1.0 / teacher.s);
  for (int j = threadIdx.x % L; j < P.top; j += L) {
    if (j >= L) at = slot_at<T>(P, row, kNoLogits, j);
    cls[j] = at.cls;
    share[j] = at.cls == -1 ? 0.0f : (j < L ? teacher.e : exp_slot(at.t, teacher.m, P.scale64)) * inv_s;
  }
  return !teacher.any ? 0 : teacher.s != teacher.s ? 2 : 1;
}

struct RowGrad {
  float g, m, inv_s, scale;
  bool zero;
  __device__ __forceinline__ float q(float z) const { return exp_diff(z, m, scale) * inv_s; }
};
__device__ __forceinline__ RowGrad row_grad(const DistillParams& P, int64_t row, int taught) {
  RowGrad r;
  r.g = (float)P.temperature * (P.reduction == UR_REDUCE_NONE ? P.g[row * P.g_stride] : P.g[0] * P.stats[2 * P.rows]);
  if (taught == 2) r.g = __builtin_nanf("");
  r.zero = taught == 0;
  r.m = P.stats[2 * row];
  r.inv_s = 1.0f / P.stats[2 * row + 1];
  r.scale = P.scale;
  return r;
}

// g q of row elements [c0, c1), threads t, t + n, ...
template <typename T, int B>
__device__ __forceinline__ void write_q(const RowGrad& r, const T* __restrict__ z, T* __restrict__ out, int64_t c0, int64_t c1, int t,
                                        int n) {
  constexpr int N = Elem<T>::kN;
  using Vec = typename Elem<T>::Vec;
  int64_t col = c0 + (int64_t)t * N;
  const int64_t step = (int64_t)n * N;
  for (; col + (B - 1) * step + N <= c1; col += B * step) {
    Vec v[B];
#pragma unroll
    for (int b = 0; b < B; ++b) v[b] = *reinterpret_cast<const Vec*>(z + col + b * step);
#pragma unroll
    for (int b = 0; b < B; ++b) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[b][j] = r.zero ? (T)0.0f : (T)(r.g * r.q((float)v[b][j]));
      __builtin_nontemporal_store(v[b], reinterpret_cast<Vec*>(out + col + b * step));
    }
  }
  if (col >= c1) return;
  Vec v[B];
  if (c1 - c0 >= N) {  // (a vector moved back to the end writes some places twice, with the same numbers)
#pragma unroll
    for (int b = 0; b < B; ++b) v[b] = *reinterpret_cast<const Vec*>(z + min(col + b * step, c1 - N));
#pragma unroll
    for (int b = 0; b < B; ++b) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[b][j] = r.zero ? (T)0.0f : (T)(r.g * r.q((float)v[b][j]));
      if (col + b * step < c1) *reinterpret_cast<Vec*>(out + min(col + b * step, c1 - N)) = v[b];
    }
    return;
  }
#pragma unroll
  for (int b = 0; b < B; ++b) v[b] = load16<T>(z, col + b * step, c1, (T)0.0f);
#pragma unroll
  for (int b = 0; b < B; ++b) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[b][j] = r.zero ? (T)0.0f : (T)(r.g * r.q((float)v[b][j]));
    store16<T>(out, col + b * step, c1, v[b]);
  }
}

// the classes of [c0, c1) that slots name, threads t, t + n, ...
template <typename T>
__device__ __forceinline__ void write_shares(const DistillParams& P, const RowGrad& r, const T* __restrict__ z, T* __restrict__ out,
                                             const int* cls, const float* share, int64_t c0, int64_t c1, int t, int n) {
  if (r.zero) return;
  for (int j = t; j < P.top; j += n) {
    const int c = cls[j];
    if (c < c0 || c >= c1 || c < 0) continue;
    float p = 0.0f;
    bool first = true;
    for (int i = 0; i < P.top; ++i)
      if (cls[i] == c) {
        first &= i >= j;
        p += share[i];
      }
    if (first) out[c] = (T)(r.g * (r.q((float)z[c]) - p));
  }
}

// L lanes a row, kThreads / L rows a workgroup; a wave's stores to one place stay in their order.  32768 x 1000 bf16 41 us
// (3.2 TB/s), 30000 x 128 bf16 11, 100000 x 6 fp32 7: the teacher's reductions are made again, once a wave.
template <typename T, int L>
__global__ void __launch_bounds__(kThreads) k_distill_bwd_rows(const DistillParams P) {
  constexpr int R = kThreads / L;
  __shared__ int cls[R][kGroupTop];
  __shared__ float share[R][kGroupTop];
  const int t = threadIdx.x % L, sub = threadIdx.x / L;
  const int64_t want = (P.block0 + blockIdx.x) * R + sub;
  const bool mine = want < P.rows;
  const int64_t row = mine ? want : P.rows - 1;
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  T* out = static_cast<T*>(P.grad) + row * P.cols;
  const RowGrad r = row_grad(P, row, row_shares<T, L>(P, row, cls[sub], share[sub]));
  if (mine) write_q<T, 2>(r, z, out, 0, P.cols, t, L);
  wave_lds_handoff();
  if (mine) write_shares<T>(P, r, z, out, cls[sub], share[sub], 0, P.cols, t, L);
}

// A workgroup takes one row or (P.splits > 1) a part of one.  8192 x 32768 bf16 213 us (5.0 TB/s; with ordinary stores 250),
// 4096 x 32768 fp32 210 us (5.1), 2000 x 20000 fp32 63 us (5.1), 4096 x 8101 fp16 31.5 us (4.2), 3 x 131071 bf16 10.3 us.
template <typename T, int TH>
__global__ void __launch_bounds__(TH) k_distill_bwd(const DistillParams P) {
  __shared__ int cls[kMaxTop];
  __shared__ float share[kMaxTop];
  __shared__ int taught;
  const int64_t row = P.splits > 1 ? blockIdx.y : P.block0 + blockIdx.x;
  const int64_t c0 = P.splits > 1 ? (int64_t)blockIdx.x * P.chunk : 0, c1 = P.splits > 1 ? min(c0 + P.chunk, P.cols) : P.cols;
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  T* out = static_cast<T*>(P.grad) + row * P.cols;
  if (threadIdx.x < 64) {
    const int state = row_shares<T, 64>(P, row, cls, share);
    if (threadIdx.x == 0) taught = state;
  }
  __syncthreads();
  const RowGrad r = row_grad(P, row, taught);
  write_q<T, 4>(r, z, out, c0, c1, threadIdx.x, TH);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the stores have arrived before other waves write the same places
  __syncthreads();
  write_shares<T>(P, r, z, out, cls, share, c0, c1, threadIdx.x, TH);
}

// ---- which kernel a call takes ---------------------------------------------------------------------------------------
struct DistillPlan {
  int lanes;         // lanes a row (8, 16, 64), or 0: workgroups
  int bwd_threads;   // backward: threads of a workgroup that takes a row
  int splits;        // workgroups a row
  int64_t chunk;     // classes of a part
  int64_t partials;  // workgroups that hand a sum to the reduction
  int64_t ws_bytes;
};

DistillPlan distill_plan(int64_t rows, int64_t cols, int dtype, int reduction) {
  DistillPlan p{0, 256, 1, cols, rows, 0};
  const int n = 16 / dtype_bytes(dtype);
  const int64_t vecs = ceil_div(cols, n);
  if (vecs <= 16) p.lanes = 8;
  else if (vecs <= 64) p.lanes = 16;
  else if (vecs <= 256) p.lanes = 64;
  if (p.lanes) {
    p.partials = ceil_div(rows, kThreads / p.lanes);
  } else if (rows >= 512) {
    // Large workgroups walk few rows at a time through memory, which the backward's mixed reads and writes like -- where a
    // row is a whole number of their batches of 4 vectors a thread, or nearly (8192 x 32768 bf16: 208 us with 1024 threads,
    // 226 with 512, 240 with 256; 2000 x 20000 fp32, 1.2 batches of 1024 threads: 76, 67, 72).
    for (int th : {1024, 512})
      if (p.bwd_threads == 256 && vecs >= 4 * th && (th == 512 || 10 * ceil_div(vecs, 4096) * 4096 <= 11 * vecs)) p.bwd_threads = th;
  } else {
    // parts of at least one vector a thread, and about 1024 workgroups
    const int64_t want = std::min<int64_t>(ceil_div(cols, (int64_t)256 * n), std::max<int64_t>(1, 1024 / rows));
    p.chunk = ceil_div(ceil_div(cols, want), (int64_t)256 * n) * (256 * n);
    p.splits = (int)ceil_div(cols, p.chunk);
  }
  const int64_t reduce = reduction == UR_REDUCE_NONE ? 0 : p.partials * 16;
  p.ws_bytes = reduce + (p.splits > 1 ? rows * p.splits * 8 : 0);
  return p;
}

template <typename T>
void launch_fwd(const DistillPlan& p, const DistillParams& P, hipStream_t st) {
  if (p.splits > 1) {
    k_distill_split<T><<<dim3(p.splits, (unsigned)P.rows), kThreads, 0, st>>>(P);
    k_distill_join<T><<<(unsigned)P.rows, 64, 0, st>>>(P);
  } else {
    in_pieces(p.lanes ? p.partials : P.rows, kThreads, [&](int64_t first, unsigned grid) {
      DistillParams Q = P;
      Q.block0 = first;
      if (p.lanes == 8) k_distill_fwd_rows<T, 8><<<grid, kThreads, 0, st>>>(Q);
      else if (p.lanes == 16) k_distill_fwd_rows<T, 16><<<grid, kThreads, 0, st>>>(Q);
      else if (p.lanes == 64) k_distill_fwd_rows<T, 64><<<grid, kThreads, 0, st>>>(Q);
      else k_distill_fwd<T><<<grid, kThreads, 0, st>>>(Q);
    });
  }
  if (P.reduction != UR_REDUCE_NONE && !(p.lanes && p.partials == 1)) k_distill_reduce<<<1, 1024, 0, st>>>(P);
}

template <typename T>
void launch_bwd(const DistillPlan& p, const DistillParams& P, hipStream_t st) {
  if (p.splits > 1) {
    k_distill_bwd<T, 256><<<dim3(p.splits, (unsigned)P.rows), 256, 0, st>>>(P);
    return;
  }
  const int lanes = P.top <= kGroupTop ? p.lanes : 0;
  in_pieces(lanes ? ceil_div(P.rows, kThreads / lanes) : P.rows, lanes ? kThreads : p.bwd_threads, [&](int64_t first, unsigned grid) {
    DistillParams Q = P;
    Q.block0 = first;
    if (lanes == 8) k_distill_bwd_rows<T, 8><<<grid, kThreads, 0, st>>>(Q);
    else if (lanes == 16) k_distill_bwd_rows<T, 16><<<grid, kThreads, 0, st>>>(Q);
    else if (lanes == 64) k_distill_bwd_rows<T, 64><<<grid, kThreads, 0, st>>>(Q);
    else if (p.bwd_threads == 256) k_distill_bwd<T, 256><<<grid, 256, 0, st>>>(Q);
    else if (p.bwd_threads == 512) k_distill_bwd<T, 512><<<grid, 512, 0, st>>>(Q);
    else k_distill_bwd<T, 1024><<<grid, 1024, 0, st>>>(Q);
  });
}

int check_common(const void* logits, int64_t stride, int dtype, int64_t rows, int64_t cols, const void* teacher,
                 int teacher_dtype, const void* index, int index_bytes, int top, double temperature, int reduction) {
  if (!logits || !teacher || !index) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (!known_dtype(dtype) || !known_dtype(teacher_dtype)) return set_error(UR_ERR_INVALID_ARG, "bad dtype");
  if (index_bytes != 4 && index_bytes != 8) return set_error(UR_ERR_INVALID_ARG, "indices have 4 or 8 bytes");
  if (rows <= 0 || cols <= 0 || top <= 0) return set_error(UR_ERR_INVALID_ARG, "rows, cols and top must be positive");
  if (rows > 0x7fffffff || cols > 0x7fffffff) return set_error(UR_ERR_UNSUPPORTED, "rows and cols must be below 2^31");
  if (top > kMaxTop) return set_error(UR_ERR_UNSUPPORTED, "at most %d teacher slots", kMaxTop);
  if (stride < cols && rows > 1) return set_error(UR_ERR_INVALID_ARG, "row stride below the row length");
  const float scale = (float)(kLog2e / temperature), t32 = (float)temperature;
  if (!(t32 > 0.0f) || !(t32 - t32 == 0.0f) || !(scale > 0.0f) || !(scale - scale == 0.0f))
    return set_error(UR_ERR_INVALID_ARG, "temperature must be positive and finite, and so must its reciprocal");
  if (reduction != UR_REDUCE_NONE && reduction != UR_REDUCE_SUM && reduction != UR_REDUCE_MEAN)
    return set_error(UR_ERR_INVALID_ARG, "bad reduction %d", reduction);
  return UR_OK;
}

void fill_common(DistillParams& P, const void* logits, int64_t stride, int64_t rows, int64_t cols, const void* teacher,
                 int teacher_dtype, const void* index, int index_bytes, int top, double temperature, int reduction) {
  P.z = logits; P.stride = stride; P.rows = rows; P.cols = cols; P.t = teacher; P.t_dtype = teacher_dtype;
  P.index = index; P.index64 = index_bytes == 8; P.top = top; P.temperature = temperature;
  P.scale64 = kLog2e / temperature; P.inv_t = 1.0 / temperature; P.scale = (float)P.scale64; P.reduction = reduction;
}

}  // namespace

extern "C" {

int64_t ur_distill_workspace_bytes(int64_t rows, int64_t cols, int dtype, int reduction) {
  if (!known_dtype(dtype)) return set_error(UR_ERR_INVALID_ARG, "bad dtype %d", dtype);
  if (rows <= 0 || cols <= 0 || rows > 0x7fffffff || cols > 0x7fffffff)
    return set_error(UR_ERR_INVALID_ARG, "rows and cols must be positive and below 2^31");
  return distill_plan(rows, cols, dtype, reduction).ws_bytes;
}

int ur_distill_forward(const void* logits, int64_t row_stride, int dtype, int64_t rows, int64_t cols, const void* teacher,
                       int teacher_dtype, const void* index, int index_bytes, int top, double temperature, int reduction,
                       float* loss, float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_common(logits, row_stride, dtype, rows, cols, teacher, teacher_dtype, index, index_bytes, top,
                            temperature, reduction))
    return rc;
  if (!loss) return set_error(UR_ERR_INVALID_ARG, "null output pointer");
  const DistillPlan plan = distill_plan(rows, cols, dtype, reduction);
  const size_t need = (size_t)plan.ws_bytes;
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  DistillParams P{};
  fill_common(P, logits, row_stride, rows, cols, teacher, teacher_dtype, index, index_bytes, top, temperature, reduction);
  P.loss = loss; P.stats = stats;
  P.splits = plan.splits; P.chunk = plan.chunk; P.partials = plan.partials;
  char* ws = static_cast<char*>(workspace);
  if (reduction != UR_REDUCE_NONE) {
    P.partial = reinterpret_cast<double*>(ws);
    ws += plan.partials * 16;
  }
  if (plan.splits > 1) P.split_stats = reinterpret_cast<float*>(ws);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) launch_fwd<float>(plan, P, st);
  else if (dtype == UR_F16) launch_fwd<_Float16>(plan, P, st);
  else launch_fwd<__bf16>(plan, P, st);
  return launch_status("ur_distill_forward");
}

int ur_distill_backward(const float* grad_loss, int64_t grad_stride, const void* logits, int64_t row_stride, int dtype,
                        int64_t rows, int64_t cols, const void* teacher, int teacher_dtype, const void* index,
                        int index_bytes, int top, double temperature, int reduction, const float* stats,
                        void* grad_logits, void* stream) {
  if (int rc = check_common(logits, row_stride, dtype, rows, cols, teacher, teacher_dtype, index, index_bytes, top,
                            temperature, reduction))
    return rc;
  if (!grad_loss || !stats) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (!grad_logits) return set_error(UR_ERR_INVALID_ARG, "null output pointer");
  DistillParams P{};
  fill_common(P, logits, row_stride, rows, cols, teacher, teacher_dtype, index, index_bytes, top, temperature, reduction);
  P.g = grad_loss; P.g_stride = grad_stride; P.stats = const_cast<float*>(stats); P.grad = grad_logits;
  const DistillPlan plan = distill_plan(rows, cols, dtype, reduction);
  P.splits = plan.splits; P.chunk = plan.chunk;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) launch_bwd<float>(plan, P, st);
  else if (dtype == UR_F16) launch_bwd<_Float16>(plan, P, st);
  else launch_bwd<__bf16>(plan, P, st);
  return launch_status("ur_distill_backward");
}

}  // extern "C"
