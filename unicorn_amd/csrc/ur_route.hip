// ur_route.hip -- routing: the top-k of a row's candidates, their weights, and how often each candidate was taken.
//
//   s = softmax(l) or sigmoid(l)            c = s + bias (selection only; without a bias the order of l is the order of s)
//   groups of E / G consecutive candidates: a group's value is its largest c, or the sum of its two largest (of the one
//   it has); the best `top_groups` groups stay                   ties, here and below: the lowest index
//   indices = the k largest c left, largest first               weights = scale * s / sum of the chosen s, or scale * s
//   A candidate with l = -inf (or bias = -inf) is never chosen; slots that nothing is left for get index -1, weight 0.
//
// Which of two close scores is larger would depend on the last bit of an exponential, so the order is DEFINED as that of
// the 64-bit scores.
#include "ur_rows.h"

#include <algorithm>

using namespace ur;

namespace {

constexpr int kMaxCands = 1024, kMaxTop = 64, kMaxGroups = 64;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxBlocks = 1024;  // workgroups of the forward = rows of partial counts

struct RouteParams {
  const void* logits;
  int64_t stride;
  const float* bias;
  int64_t rows;
  int cands, top_k, groups, per_group, top_groups;
  bool sigmoid, top2, renormalize;
  float scale;
  float* weights;
  int64_t* indices;
  int32_t* counts;
  int32_t* ws;  // (workgroups, cands) partial counts
  int parts;
  const float* grad_w;
  void* grad;
};

// ---- order-preserving keys: larger value = larger unsigned number, NaN above everything, 0 = not eligible -----------
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // (-0 -> +0)
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));  // (NaN -> NaN)
}

__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// ---- the choice in 64 bits, one wave for a row; lane j < k returns slot j's candidate or -1 --------------------------
// `vals`: LDS of this wave, one double per candidate; `poisoned`: the row's softmax is NaN (a NaN or +inf among its logits).
template <typename T>
__device__ int choose_wide(const RouteParams& P, const T* __restrict__ row, double* vals, bool& poisoned) {
  constexpr int kItems = kMaxCands / 64;
  const int lane = threadIdx.x & 63, E = P.cands;
  const double inf = __builtin_inf();
  double m = -inf, z = 1.0;
  if (!P.sigmoid) {
    float mf = -__builtin_inff();
    for (int e = lane; e < E; e += 64) mf = __builtin_fmaxf(mf, (float)row[e]);
    mf = reduce_lanes<64, OpMax>(mf);
    m = mf == -__builtin_inff() ? 0.0 : (double)mf;
    z = 0.0;
    for (int e = lane; e < E; e += 64) z += exp((double)(float)row[e] - m);
    z = wave_sum(z);
  }
  poisoned = z != z;
  uint64_t key[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int e = lane + 64 * i;
    key[i] = 0;
    if (e < E) {
      const double l = (double)(float)row[e];
      const double s = P.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - m) / z;
      const double c = P.bias ? s + (double)P.bias[e] : l;
      const bool ok = l != -inf && !(P.bias && c == -inf);
      key[i] = ok ? order_key(c) : 0;
      // a group's value: by scores where they are added, by the order of the keys else
      if (P.groups > 1) vals[e] = !ok ? -inf : (P.bias || !P.top2) ? c : s;
    }
  }
  if (P.groups > 1) {
    wave_lds_handoff();
    uint64_t g = 0;
    if (lane < P.groups) {
      uint64_t a = 0, b = 0;  // the two largest (0: none)
      for (int i = 0; i < P.per_group; ++i) {
        const double v = vals[lane * P.per_group + i];
        const uint64_t k = v == -inf ? 0 : order_key(v);
        b = k > a ? a : (k > b ? k : b);
        a = k > a ? k : a;
      }
      g = (P.top2 && a && b) ? order_key(key_value(a) + key_value(b)) : a;
    }
    int rank = 0;
    for (int o = 0; o < P.groups; ++o) {
      const uint64_t other = __shfl(g, o);
      rank += other > g || (other == g && o < lane);
    }
    const uint64_t kept = __ballot(lane < P.groups && rank < P.top_groups);
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (lane + 64 * i < E && !((kept >> ((lane + 64 * i) / P.per_group)) & 1)) key[i] = 0;
    wave_lds_handoff();  // (the next row writes `vals` again)
  }
  int mine = -1;
  for (int r = 0; r < P.top_k; ++r) {
    uint64_t best = 0;
    int at = E;
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (key[i] > best) {
        best = key[i];
        at = lane + 64 * i;
      }
    for (int o = 32; o; o >>= 1) {
      const uint64_t ob = __shfl_xor(best, o);
      const int oa = __shfl_xor(at, o);
      if (ob > best || (ob == best && oa < at)) {
        best = ob;
        at = oa;
      }
    }
    if (best == 0) break;
    if (lane == r) mine = at;
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (lane + 64 * i == at) key[i] = 0;
  }
  return mine;
}

// ---- weights of the chosen, LPR lanes a row: lane j holds slot j -------------------------------------------------------
struct Chosen {
  float share;   // s_j / sum of the chosen s (renormalised), or s_j
  float comp;    // 1 - s_j of a sigmoid
};

// l: slot j's logit, `filled`: whether slot j holds a candidate; m, z: the row's softmax (needed only when not renormalised)
template <int LPR>
__device__ __forceinline__ Chosen chosen_share(bool sigmoid, bool renormalize, float l, bool filled, float m, float z) {
  Chosen r{0.0f, 1.0f};
  const float em = expf(-fabsf(l));  // in (0, 1]: no overflow on either side
  if (sigmoid) r.comp = l >= 0.0f ? em / (1.0f + em) : 1.0f / (1.0f + em);
  if (!renormalize) {
    r.share = !filled ? 0.0f : sigmoid ? (l >= 0.0f ? 1.0f / (1.0f + em) : em / (1.0f + em)) : expf(l - m) / z;
    if (l != l) r.share = filled ? l : 0.0f;
    return r;
  }
  // only ratios matter: the common factor exp(max) is left out, so scores far below the smallest number still share
  const float x = sigmoid ? __builtin_fminf(l, 0.0f) : l;
  const float top = reduce_lanes<LPR, OpMax>(filled ? x : -__builtin_inff());
  float a = filled ? expf(x - top) : 0.0f;
  if (sigmoid && filled) a /= 1.0f + em;
  if (filled && l != l) a = l;
  const float total = reduce_lanes<LPR, OpSum>(a);
  r.share = total == 0.0f ? 0.0f : a / total;
  return r;
}

// maximum and sum of exponentials of a row, LPR lanes
template <typename T, int LPR>
__device__ __forceinline__ void row_softmax(const T* __restrict__ row, int E, int t, float& m, float& z) {
  float mf = -__builtin_inff();
  for (int e = t; e < E; e += LPR) mf = __builtin_fmaxf(mf, (float)row[e]);
  mf = reduce_lanes<LPR, OpMax>(mf);
  m = mf == -__builtin_inff() ? 0.0f : mf;
  float s = 0.0f;
  for (int e = t; e < E; e += LPR) s += expf((float)row[e] - m);
  z = reduce_lanes<LPR, OpSum>(s);
  if (z == 0.0f) z = 1.0f;  // nothing eligible: every score is 0
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_route_fwd(const RouteParams P) {
  __shared__ int hist[kMaxCands];
  __shared__ double vals[kWaves][kMaxCands];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int e = threadIdx.x; e < P.cands; e += kThreads) hist[e] = 0;
  __syncthreads();
  for (int64_t row = (int64_t)blockIdx.x * kWaves + wave; row < P.rows; row += (int64_t)gridDim.x * kWaves) {
    const T* l = static_cast<const T*>(P.logits) + row * P.stride;
    bool poisoned;
    const int at = choose_wide<T>(P, l, vals[wave], poisoned);
    float m = 0.0f, z = 1.0f;
    if (!P.sigmoid && !P.renormalize) row_softmax<T, 64>(l, P.cands, lane, m, z);
    const Chosen c = chosen_share<64>(P.sigmoid, P.renormalize, at >= 0 ? (float)l[at] : 0.0f, at >= 0, m, z);
    if (lane < P.top_k) {
      P.weights[row * P.top_k + lane] = poisoned ? __builtin_nanf("") : P.scale * c.share;
      P.indices[row * P.top_k + lane] = at;
      if (at >= 0) atomicAdd(&hist[at], 1);
    }
  }
  __syncthreads();
  int32_t* out = P.parts > 1 ? P.ws + (int64_t)blockIdx.x * P.cands : P.counts;
  for (int e = threadIdx.x; e < P.cands; e += kThreads) out[e] = hist[e];
}

// counts = the sums of the workgroups' counts: 32 candidates a workgroup, 32 groups of threads over the partial rows
__global__ void __launch_bounds__(1024) k_route_counts(const RouteParams P) {
  __shared__ int acc[32][33];
  const int c = threadIdx.x & 31, grp = threadIdx.x >> 5, e = blockIdx.x * 32 + c;
  int s = 0;
  if (e < P.cands)
    for (int p = grp; p < P.parts; p += 32) s += P.ws[(int64_t)p * P.cands + e];
  acc[grp][c] = s;
  __syncthreads();
  if (grp != 0 || e >= P.cands) return;
  int total = 0;
  for (int g = 0; g < 32; ++g) total += acc[g][c];
  P.counts[e] = total;
}

// Backward, with w_j = share_j * scale:
//   renormalised: d share_j = sum_i share_i (dw_j - dw_i), written as differences: a row with one choice gets exactly 0,
//     and nothing cancels where one choice has nearly all the weight;
//     softmax: dl_j = scale share_j d_j for the chosen, exactly 0 for all others; sigmoid: times (1 - s_j)
//   not renormalised: sigmoid: dl_j = scale dw_j s_j (1 - s_j); softmax: dl_e = s_e (ds_e - sum_j ds_j s_j), every candidate
template <typename T>
__global__ void __launch_bounds__(kThreads) k_route_bwd(const RouteParams P) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= P.rows) return;  // (whole waves)
  const T* l = static_cast<const T*>(P.logits) + row * P.stride;
  T* out = static_cast<T*>(P.grad) + row * P.cands;
  const int64_t slot = lane < P.top_k ? P.indices[row * P.top_k + lane] : -1;
  const bool filled = slot >= 0 && slot < P.cands;
  const int at = filled ? (int)slot : -1;
  const float dw = filled ? P.grad_w[row * P.top_k + lane] : 0.0f;
  const bool dense = !P.sigmoid && !P.renormalize;
  float m = 0.0f, z = 1.0f;
  if (dense) row_softmax<T, 64>(l, P.cands, lane, m, z);
  const Chosen c = chosen_share<64>(P.sigmoid, P.renormalize, filled ? (float)l[at] : 0.0f, filled, m, z);
  float g;
  if (P.renormalize) {
    float d = 0.0f;
    for (int i = 0; i < P.top_k; ++i) {
      const float wi = __shfl(c.share, i), di = __shfl(dw, i);
      d = __builtin_fmaf(wi, dw - di, d);
    }
    g = P.scale * c.share * d * c.comp;
  } else {
    g = P.scale * dw * c.share * c.comp;  // (softmax: ds_j s_j)
  }
  const float dot = dense ? reduce_lanes<64, OpSum>(filled ? g : 0.0f) : 0.0f;
  // a NaN in a softmax is in every score: the forward left it in every weight of the row
  const float first = P.weights[row * P.top_k];
  const bool poisoned = !P.sigmoid && first != first;
  for (int base = 0; base < P.cands; base += 64) {  // (whole waves: lanes read each other's slots)
    const int e = base + lane;
    float v = poisoned ? first : 0.0f;
    if (dense && e < P.cands) v = -(expf((float)l[e] - m) / z) * dot;
    for (int j = 0; j < P.top_k; ++j) {
      const int aj = __shfl(at, j);
      const float gj = __shfl(g, j);
      if (aj == e) v += gj;
    }
    if (e < P.cands) out[e] = (T)v;
  }
}

int check_common(const void* logits, int64_t stride, int dtype, int64_t rows, int cands, int top_k, int score) {
  if (!logits) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (!known_dtype(dtype)) return set_error(UR_ERR_INVALID_ARG, "bad dtype %d", dtype);
  if (rows <= 0 || cands <= 0 || top_k <= 0) return set_error(UR_ERR_INVALID_ARG, "rows, cands and top_k must be positive");
  if (cands > kMaxCands || top_k > kMaxTop)
    return set_error(UR_ERR_UNSUPPORTED, "at most %d candidates and %d choices", kMaxCands, kMaxTop);
  if (rows > 0x7fffffff) return set_error(UR_ERR_UNSUPPORTED, "rows must be below 2^31");
  if (top_k > cands) return set_error(UR_ERR_INVALID_ARG, "top_k above the number of candidates");
  if (score != UR_SCORE_SOFTMAX && score != UR_SCORE_SIGMOID) return set_error(UR_ERR_INVALID_ARG, "bad score %d", score);
  if (stride < cands && rows > 1) return set_error(UR_ERR_INVALID_ARG, "row stride below the row length");
  return UR_OK;
}

int route_parts(int64_t rows) { return (int)std::min<int64_t>(ceil_div(rows, kWaves), kMaxBlocks); }

}  // namespace

extern "C" {

int64_t ur_route_workspace_bytes(int64_t rows, int cands) {
  if (rows <= 0 || cands <= 0 || rows > 0x7fffffff || cands > kMaxCands)
    return set_error(UR_ERR_INVALID_ARG, "bad rows or cands");
  const int parts = route_parts(rows);
  return parts > 1 ? (int64_t)parts * cands * 4 : 0;
}

int ur_route_forward(const void* logits, int64_t row_stride, int dtype, const float* bias, int64_t rows, int cands,
                     int top_k, int score, int groups, int top_groups, int group_score, int renormalize, float scale,
                     float* weights, int64_t* indices, int32_t* counts, void* workspace, size_t workspace_bytes,
                     void* stream) {
  if (int rc = check_common(logits, row_stride, dtype, rows, cands, top_k, score)) return rc;
  if (!weights || !indices || !counts) return set_error(UR_ERR_INVALID_ARG, "null output pointer");
  if (groups <= 0 || cands % groups) return set_error(UR_ERR_INVALID_ARG, "groups must divide the number of candidates");
  if (groups > kMaxGroups) return set_error(UR_ERR_UNSUPPORTED, "at most %d groups", kMaxGroups);
  if (top_groups <= 0 || top_groups > groups) return set_error(UR_ERR_INVALID_ARG, "top_groups must be 1 .. groups");
  if (top_k > top_groups * (cands / groups))
    return set_error(UR_ERR_INVALID_ARG, "top_k above the number of candidates in top_groups groups");
  if (group_score != UR_GROUP_MAX && group_score != UR_GROUP_TOP2)
    return set_error(UR_ERR_INVALID_ARG, "bad group_score %d", group_score);
  if (!(scale - scale == 0.0f)) return set_error(UR_ERR_INVALID_ARG, "scale must be finite");
  const size_t need = (size_t)ur_route_workspace_bytes(rows, cands);
  if (workspace_bytes < need || (need && !workspace))
    return set_error(UR_ERR_WORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, need);
  RouteParams P{};
  P.logits = logits; P.stride = row_stride; P.bias = bias; P.rows = rows; P.cands = cands; P.top_k = top_k;
  P.groups = groups; P.per_group = cands / groups; P.top_groups = top_groups;
  P.sigmoid = score == UR_SCORE_SIGMOID; P.top2 = group_score == UR_GROUP_TOP2; P.renormalize = renormalize != 0;
  P.scale = scale; P.weights = weights; P.indices = indices; P.counts = counts;
  P.ws = static_cast<int32_t*>(workspace); P.parts = route_parts(rows);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) k_route_fwd<float><<<P.parts, kThreads, 0, st>>>(P);
  else if (dtype == UR_F16) k_route_fwd<_Float16><<<P.parts, kThreads, 0, st>>>(P);
  else k_route_fwd<__bf16><<<P.parts, kThreads, 0, st>>>(P);
  if (P.parts > 1) k_route_counts<<<(unsigned)ceil_div(cands, 32), 1024, 0, st>>>(P);
  return launch_status("ur_route_forward");
}

int ur_route_backward(const float* grad_weights, const void* logits, int64_t row_stride, int dtype, int64_t rows,
                      int cands, const float* weights, const int64_t* indices, int top_k, int score, int renormalize, float scale,
                      void* grad_logits, void* stream) {
  if (int rc = check_common(logits, row_stride, dtype, rows, cands, top_k, score)) return rc;
  if (!grad_weights || !weights || !indices) return set_error(UR_ERR_INVALID_ARG, "null input pointer");
  if (!grad_logits) return set_error(UR_ERR_INVALID_ARG, "null output pointer");
  if (!(scale - scale == 0.0f)) return set_error(UR_ERR_INVALID_ARG, "scale must be finite");
  RouteParams P{};
  P.logits = logits; P.stride = row_stride; P.rows = rows; P.cands = cands; P.top_k = top_k;
  P.sigmoid = score == UR_SCORE_SIGMOID; P.renormalize = renormalize != 0; P.scale = scale;
  P.indices = const_cast<int64_t*>(indices); P.grad_w = grad_weights; P.weights = const_cast<float*>(weights); P.grad = grad_logits;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)ceil_div(rows, kWaves);
  if (dtype == UR_F32) k_route_bwd<float><<<grid, kThreads, 0, st>>>(P);
  else if (dtype == UR_F16) k_route_bwd<_Float16><<<grid, kThreads, 0, st>>>(P);
  else k_route_bwd<__bf16><<<grid, kThreads, 0, st>>>(P);
  return launch_status("ur_route_backward");
}

}  // extern "C"
