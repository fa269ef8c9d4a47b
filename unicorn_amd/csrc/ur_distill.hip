// ur_distill.hip -- distillation from a teacher's top logits: per row, the divergence of the student's distribution over
// all V classes from the teacher's over the k classes whose logits are known.
//
//   p = softmax(t / T) over the row's filled slots        q = softmax(z / T) over V
//   loss = T^2 sum_j p_j (log p_j - log q_{i_j})          dz_v = g T (q_v - sum_{j: i_j = v} p_j)
//
// Bound by memory: the forward reads z once (running maximum and sum of exponentials), the backward reads it again and
// writes the gradient.  Sums are fp32; the k-slot arithmetic, a difference of logarithms that is small where the student has
// learnt, is in 64 bits.
#include "ur_rows.h"

#include <algorithm>

using namespace ur;

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxTop = 1024;  // slots of a row: the backward keeps their classes and shares in LDS

struct DistillParams {
  const void* z;
  int64_t stride;
  int64_t rows, cols;
  const void* t;
  int t_dtype;
  const void* index;
  bool index64;
  int top;
  float temperature, inv_t;
  float* stats;  // (rows, 2): maximum of z, sum of exp((z - max) / T)
  float* loss;   // (rows) or one value
  int reduction;
  float* row_loss;  // rows that are reduced: their losses ...
  float* taught;    // ... and 1 where the row has a teacher; backward: factor of the reduction (one value)
  float* ws;        // long rows: (rows, splits, 2) partial maxima and sums
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

// exp((v - m) / T); an infinite maximum would make inf - inf of the equal ones, as the definition does
__device__ __forceinline__ float exp_diff(float v, float m, float scale) { return exp2f((v - m) * scale); }

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

// running maximum and sum of row elements [c0, c1), threads t, t + n, ... of a group
template <typename T>
__device__ __forceinline__ void row_part(const T* __restrict__ z, int64_t c0, int64_t c1, int t, int n, float scale, float& m,
                                         float& s) {
  constexpr int N = Elem<T>::kN;
  m = -__builtin_inff();
  s = 0.0f;
  for (int64_t col = c0 + (int64_t)t * N; col < c1; col += (int64_t)n * N) {
    const auto v = load16<T>(z, col, c1, (T)-__builtin_inff());
    float top = (float)v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) top = __builtin_fmaxf(top, (float)v[j]);
    if (top > m) {
      s = m == -__builtin_inff() ? s : s * exp_diff(m, top, scale);
      m = top;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m;  // (nothing but -inf so far: every term is 0)
#pragma unroll
    for (int j = 0; j < N; ++j) s += exp_diff((float)v[j], ref, scale);
  }
}

template <int L>
__device__ __forceinline__ void merge_lanes(float& m, float& s, float scale) {
  const float top = reduce_lanes<L, OpMax>(m);
  if (top != -__builtin_inff() && m != top) s *= exp_diff(m, top, scale);
  s = reduce_lanes<L, OpSum>(s);
  m = top;
}

__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ double wave_max(double v) {
  for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}

// The teacher of a row, by one wave: maximum and sum of exponentials of its filled slots.  Returns whether there is one; a
// class outside [0, V) makes the sum NaN.
struct Teacher {
  double m, s;
  bool any;
};
__device__ Teacher row_teacher(const DistillParams& P, int64_t row) {
  const int lane = threadIdx.x & 63;
  double m = -__builtin_inf();
  bool any = false, bad = false;
  for (int j = lane; j < P.top; j += 64) {
    const int64_t c = slot_class(P, row, j);
    if (c < 0) continue;
    const double t = (double)load_as_float(P.t, P.t_dtype, row * P.top + j);
    bad |= c >= P.cols || t != t;
    any |= t != -__builtin_inf();
    m = fmax(m, t);
  }
  m = wave_max(m);
  bad = __any(bad);
  any = __any(any) || bad;
  double s = 0.0;
  for (int j = lane; j < P.top; j += 64) {
    if (slot_class(P, row, j) < 0) continue;
    s += exp(((double)load_as_float(P.t, P.t_dtype, row * P.top + j) - m) * (double)P.inv_t);
  }
  s = wave_sum(s);
  return {m, bad ? __builtin_nan("") : s, any};
}

// loss of a row from its softmax statistics, by one wave
template <typename T>
__device__ void row_loss(const DistillParams& P, int64_t row, const T* __restrict__ z, float m, float s) {
  const int lane = threadIdx.x & 63;
  const Teacher teacher = row_teacher(P, row);
  double loss = 0.0;
  if (teacher.any) {
    const double inv_t = 1.0 / (double)P.temperature;
    const double log_s = log((double)s), log_ps = log(teacher.s);
    for (int j = lane; j < P.top; j += 64) {
      const int64_t c = slot_class(P, row, j);
      if (c < 0) continue;
      if (c >= P.cols) {
        loss = __builtin_nan("");
        continue;
      }
      const double log_p = ((double)load_as_float(P.t, P.t_dtype, row * P.top + j) - teacher.m) * inv_t - log_ps;
      const double log_q = ((double)(float)z[c] - (double)m) * inv_t - log_s;
      const double p = exp(log_p);
      if (p != 0.0) loss += p * (log_p - log_q);
    }
    loss = wave_sum(loss) * (double)P.temperature * (double)P.temperature;
  }
  if (lane == 0) {
    if (P.stats) {
      P.stats[2 * row] = m;
      P.stats[2 * row + 1] = s;
    }
    if (P.reduction == UR_REDUCE_NONE) {
      P.loss[row] = (float)loss;
    } else {
      P.row_loss[row] = (float)loss;
      P.taught[row] = teacher.any ? 1.0f : 0.0f;
    }
  }
}

// one workgroup a row
template <typename T>
__global__ void __launch_bounds__(kThreads) k_distill_fwd(const DistillParams P) {
  __shared__ float part[2][kWaves];
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  const float scale = P.inv_t * kLog2e;
  float m, s;
  row_part<T>(z, 0, P.cols, threadIdx.x, kThreads, scale, m, s);
  merge_lanes<64>(m, s, scale);
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = m;
    part[1][threadIdx.x >> 6] = s;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  m = part[0][0];
  s = part[1][0];
  for (int w = 1; w < kWaves; ++w) merge(m, s, part[0][w], part[1][w], scale);
  row_loss<T>(P, row, z, m, s);
}

// sum or mean of the rows' losses, in 64 bits and in a fixed order; keeps the factor for the backward
__global__ void __launch_bounds__(1024) k_distill_reduce(const DistillParams P) {
  __shared__ double part[2][16];
  double a = 0.0, n = 0.0;
  for (int64_t r = threadIdx.x; r < P.rows; r += 1024) {
    a += (double)P.row_loss[r];
    n += (double)P.taught[r];
  }
  a = wave_sum(a);
  n = wave_sum(n);
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
  const double factor = P.reduction == UR_REDUCE_MEAN ? 1.0 / (n > 0.0 ? n : 1.0) : 1.0;
  P.loss[0] = (float)(a * factor);
  if (P.stats) P.stats[2 * P.rows] = (float)factor;
}

// Backward, one workgroup a row: all of q first, then the teacher's classes are written again with their shares taken off.
// A class that several slots name gets the sum of their shares, written by the first of them.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_distill_bwd(const DistillParams P) {
  constexpr int N = Elem<T>::kN;
  __shared__ int cls[kMaxTop];
  __shared__ float share[kMaxTop];
  __shared__ int taught;
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(P.z) + row * P.stride;
  T* out = static_cast<T*>(P.grad) + row * P.cols;
  const float scale = P.inv_t * kLog2e, m = P.stats[2 * row], s = P.stats[2 * row + 1];
  if (threadIdx.x < 64) {
    const Teacher teacher = row_teacher(P, row);
    for (int j = threadIdx.x; j < P.top; j += 64) {
      const int64_t c = slot_class(P, row, j);
      cls[j] = (c < 0 || c >= P.cols) ? -1 : (int)c;
      const double t = (double)load_as_float(P.t, P.t_dtype, row * P.top + j);
      share[j] = c < 0 ? 0.0f : (float)(exp((t - teacher.m) * (double)P.inv_t) / teacher.s);
    }
    if (threadIdx.x == 0) taught = !teacher.any ? 0 : teacher.s != teacher.s ? 2 : 1;
  }
  __syncthreads();
  float g = P.temperature * (P.reduction == UR_REDUCE_NONE ? P.g[row * P.g_stride] : P.g[0] * P.stats[2 * P.rows]);
  if (taught == 2) g = __builtin_nanf("");
  const bool zero = taught == 0;
  const float inv_s = 1.0f / s;
  for (int64_t col = (int64_t)threadIdx.x * N; col < P.cols; col += kThreads * N) {
    const auto v = load16<T>(z, col, P.cols, (T)0.0f);
    typename Elem<T>::Vec o;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = zero ? (T)0.0f : (T)(g * (exp_diff((float)v[j], m, scale) * inv_s));
    store16<T>(out, col, P.cols, o);
  }
  __syncthreads();
  if (zero) return;
  for (int j = threadIdx.x; j < P.top; j += kThreads) {
    const int c = cls[j];
    if (c < 0) continue;
    float p = 0.0f;
    bool first = true;
    for (int i = 0; i < P.top; ++i)
      if (cls[i] == c) {
        first &= i >= j;
        p += share[i];
      }
    if (first) out[c] = (T)(g * (exp_diff((float)z[c], m, scale) * inv_s - p));
  }
}

int check_common(const void* logits, int64_t stride, int dtype, int64_t rows, int64_t cols, const void* teacher,
                 int teacher_dtype, const void* index, int index_bytes, int top, float temperature, int reduction) {
  if (!logits || !teacher || !index) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (!known_dtype(dtype) || !known_dtype(teacher_dtype)) return set_error(UR_ERR_INVALID_ARG, "bad dtype");
  if (index_bytes != 4 && index_bytes != 8) return set_error(UR_ERR_INVALID_ARG, "indices have 4 or 8 bytes");
  if (rows <= 0 || cols <= 0 || top <= 0) return set_error(UR_ERR_INVALID_ARG, "rows, cols and top must be positive");
  if (rows > 0x7fffffff || cols > 0x7fffffff) return set_error(UR_ERR_UNSUPPORTED, "rows and cols must be below 2^31");
  if (top > kMaxTop) return set_error(UR_ERR_UNSUPPORTED, "at most %d teacher slots", kMaxTop);
  if (stride < cols && rows > 1) return set_error(UR_ERR_INVALID_ARG, "row stride below the row length");
  if (!(temperature > 0.0f) || !(temperature - temperature == 0.0f) || !(1.0f / temperature > 0.0f) ||
      !(1.0f / temperature - 1.0f / temperature == 0.0f))
    return set_error(UR_ERR_INVALID_ARG, "temperature must be positive and finite, and so must its reciprocal");
  if (reduction != UR_REDUCE_NONE && reduction != UR_REDUCE_SUM && reduction != UR_REDUCE_MEAN)
    return set_error(UR_ERR_INVALID_ARG, "bad reduction %d", reduction);
  return UR_OK;
}

void fill_common(DistillParams& P, const void* logits, int64_t stride, int64_t rows, int64_t cols, const void* teacher,
                 int teacher_dtype, const void* index, int index_bytes, int top, float temperature, int reduction) {
  P.z = logits; P.stride = stride; P.rows = rows; P.cols = cols; P.t = teacher; P.t_dtype = teacher_dtype;
  P.index = index; P.index64 = index_bytes == 8; P.top = top; P.temperature = temperature;
  P.inv_t = 1.0f / temperature; P.reduction = reduction;
}

}  // namespace

extern "C" {

int64_t ur_distill_workspace_bytes(int64_t rows, int64_t cols, int dtype, int reduction) {
  if (!known_dtype(dtype)) return set_error(UR_ERR_INVALID_ARG, "bad dtype %d", dtype);
  if (rows <= 0 || cols <= 0 || rows > 0x7fffffff || cols > 0x7fffffff)
    return set_error(UR_ERR_INVALID_ARG, "rows and cols must be positive and below 2^31");
  return reduction == UR_REDUCE_NONE ? 0 : rows * 2 * 4;
}

int ur_distill_forward(const void* logits, int64_t row_stride, int dtype, int64_t rows, int64_t cols, const void* teacher,
                       int teacher_dtype, const void* index, int index_bytes, int top, float temperature, int reduction,
                       float* loss, float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_common(logits, row_stride, dtype, rows, cols, teacher, teacher_dtype, index, index_bytes, top,
                            temperature, reduction))
    return rc;
  if (!loss) return set_error(UR_ERR_INVALID_ARG, "null output pointer");
  const size_t need = (size_t)ur_distill_workspace_bytes(rows, cols, dtype, reduction);
  if (workspace_bytes < need || (need && !workspace))
    return set_error(UR_ERR_WORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, need);
  DistillParams P{};
  fill_common(P, logits, row_stride, rows, cols, teacher, teacher_dtype, index, index_bytes, top, temperature, reduction);
  P.loss = loss; P.stats = stats;
  if (reduction != UR_REDUCE_NONE) {
    P.row_loss = static_cast<float*>(workspace);
    P.taught = P.row_loss + rows;
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) k_distill_fwd<float><<<(unsigned)rows, kThreads, 0, st>>>(P);
  else if (dtype == UR_F16) k_distill_fwd<_Float16><<<(unsigned)rows, kThreads, 0, st>>>(P);
  else k_distill_fwd<__bf16><<<(unsigned)rows, kThreads, 0, st>>>(P);
  if (reduction != UR_REDUCE_NONE) k_distill_reduce<<<1, 1024, 0, st>>>(P);
  return launch_status("ur_distill_forward");
}

int ur_distill_backward(const float* grad_loss, int64_t grad_stride, const void* logits, int64_t row_stride, int dtype,
                        int64_t rows, int64_t cols, const void* teacher, int teacher_dtype, const void* index,
                        int index_bytes, int top, float temperature, int reduction, const float* stats,
                        void* grad_logits, void* stream) {
  if (int rc = check_common(logits, row_stride, dtype, rows, cols, teacher, teacher_dtype, index, index_bytes, top,
                            temperature, reduction))
    return rc;
  if (!grad_loss || !stats) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (!grad_logits) return set_error(UR_ERR_INVALID_ARG, "null output pointer");
  DistillParams P{};
  fill_common(P, logits, row_stride, rows, cols, teacher, teacher_dtype, index, index_bytes, top, temperature, reduction);
  P.g = grad_loss; P.g_stride = grad_stride; P.stats = const_cast<float*>(stats); P.grad = grad_logits;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) k_distill_bwd<float><<<(unsigned)rows, kThreads, 0, st>>>(P);
  else if (dtype == UR_F16) k_distill_bwd<_Float16><<<(unsigned)rows, kThreads, 0, st>>>(P);
  else k_distill_bwd<__bf16><<<(unsigned)rows, kThreads, 0, st>>>(P);
  return launch_status("ur_distill_backward");
}

}  // extern "C"
