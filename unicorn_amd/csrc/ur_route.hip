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
#include <type_traits>

using namespace ur;

namespace {

constexpr int kMaxCands = 1024, kMaxTop = 64, kMaxGroups = 64;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kSteps = 32;  // rounds of the forward between two looks at the rows that are to be chosen again
typedef float f32x4_lds __attribute__((ext_vector_type(4)));
// Workgroups of the forward a CU, as many as are resident at once (of four waves, one on each SIMD): four of at most 128
// registers; three for 16 candidates of fp32 a lane and, for LDS, for the longest rows.  One round of them and no more: a
// second, short round lasts as long as a full one (131072 x 256 with 768 resident: 1024 workgroups 104 us, 768 workgroups 87).
// Five or six of fewer registers gain nothing (131072 x 64: 39 against 40 us): the forward is bound by instruction issue.
constexpr int kCus = 256;
constexpr int resident(int item_bytes, int lpr, int ipl) { return ipl == 16 && (lpr == 64 || item_bytes == 4) ? 3 : 4; }

struct RouteParams {
  const void* logits;
  int64_t stride;
  const float* bias;
  int64_t rows;
  int64_t block0;  // the first workgroup of this launch
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

// ---- order-preserving keys: larger value = larger unsigned number, NaN like +inf, 0 = not eligible -------------------
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) v = __builtin_inf();
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // (-0 -> +0)
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // (not NaN)
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// exp in 64 bits, to 2 ulp: x = n ln 2 + r, |r| <= ln 2 / 2, the Taylor sum of r to r^13 / 13!.  Its constants are made where
// they are used: the library's are kept in 22 registers over the whole loop over rows, of which almost none gets here.
template <uint64_t kBits>
__device__ __forceinline__ double constant() {
  uint32_t lo, hi;
  asm volatile("s_mov_b32 %0, %2\n\ts_mov_b32 %1, %3" : "=s"(lo), "=s"(hi) : "i"((uint32_t)kBits), "i"((uint32_t)(kBits >> 32)));
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
#define UR_CONSTANT(value) constant<__builtin_bit_cast(uint64_t, (double)(value))>()
__device__ __forceinline__ double exp64(double x) {
  const double y = __builtin_fmin(__builtin_fmax(x, -1100.0), 1100.0), n = rint(y * UR_CONSTANT(1.4426950408889634));
  const double r = __builtin_fma(n, UR_CONSTANT(-2.3190468138462996e-17), __builtin_fma(n, UR_CONSTANT(-0.6931471805599453), y));
  double p = UR_CONSTANT(1.0 / 6227020800.0);
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 479001600.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 39916800.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 3628800.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 362880.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 40320.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 5040.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 720.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 120.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 24.0));
  p = __builtin_fma(p, r, UR_CONSTANT(1.0 / 6.0));
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return x != x ? x : ldexp(p, (int)n);
}
#undef UR_CONSTANT

// the largest of the wave's numbers, in every lane
template <int kStep = 0>
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, other_lane<kStep>(v));
  if constexpr (kStep < 5) v = wave_max<kStep + 1>(v);
  return v;
}

// ---- the choice in 64 bits, one wave for a row; lane j < k returns slot j's candidate or -1 --------------------------
// `store`: LDS of this wave, 8 bytes a candidate: the keys.  Few rows come here, but a launch of few rows lasts as long as the
// one that does: the maxima go through lane exchanges in registers.
template <typename T>
__device__ int choose_wide(const RouteParams& P, const T* __restrict__ row, uint64_t* store) {
  const int lane = threadIdx.x & 63, E = P.cands;
  const double inf = __builtin_inf();
  double m = 0.0, z = 1.0;
  if (!P.sigmoid) {
    float mf = -__builtin_inff();
    for (int e = lane; e < E; e += 64) mf = __builtin_fmaxf(mf, (float)row[e]);
    mf = reduce_lanes<64, OpMax>(mf);
    m = mf == -__builtin_inff() ? 0.0 : (double)mf;
    z = 0.0;
    for (int e = lane; e < E; e += 64) z += exp64((double)(float)row[e] - m);
    z = sum_lanes<64>(z);
  }
  // key of a candidate's c (by_score: of s where c would be the bare logit), 0 where it is not eligible
  const auto key = [&](int e, bool by_score) -> uint64_t {
    const double l = (double)(float)row[e];
    if (l == -inf) return 0;
    if (!P.bias && !by_score) return order_key(l);
    const double s = P.sigmoid ? 1.0 / (1.0 + exp64(-l)) : exp64(l - m) / z;
    const double b = P.bias ? (double)P.bias[e] : 0.0, c = s + b;
    return b == -inf ? 0 : order_key(c);
  };
  wave_lds_handoff();
  for (int e = lane; e < E; e += 64) store[e] = key(e, P.groups > 1 && P.top2);
  wave_lds_handoff();
  if (P.groups > 1) {
    uint64_t g = 0;
    if (lane < P.groups) {
      uint64_t a = 0, b = 0;  // the two largest (0: none)
#pragma unroll 4
      for (int i = 0; i < P.per_group; ++i) {
        const uint64_t k = store[lane * P.per_group + i];
        b = k > a ? a : (k > b ? k : b);
        a = k > a ? k : a;
      }
      g = (P.top2 && a && b) ? order_key(key_value(a) + key_value(b)) : a;
    }
    int rank = 0;
    for (int o = 0; o < P.groups; ++o) {
      const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(g >> 32), o) << 32) |
                             (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)g, o);
      rank += other > g || (other == g && o < lane);
    }
    const uint64_t kept = __ballot(lane < P.groups && rank < P.top_groups);
    wave_lds_handoff();
    for (int e = lane; e < E; e += 64) {
      if (!((kept >> (e / P.per_group)) & 1)) store[e] = 0;
      else if (!P.bias && P.top2) store[e] = key(e, false);
    }
    wave_lds_handoff();
  }
  int mine = -1;
  for (int r = 0; r < P.top_k; ++r) {
    uint64_t best = 0;
    int at = E;
    for (int e = lane; e < E; e += 64)
      if (store[e] > best) {
        best = store[e];
        at = e;
      }
    // the largest key by halves, then the lowest index among those that hold it
    const uint32_t hi = wave_max((uint32_t)(best >> 32));
    const bool high = (uint32_t)(best >> 32) == hi;
    const uint32_t lo = wave_max(high ? (uint32_t)best : 0);
    if (hi == 0 && lo == 0) break;
    at = kMaxCands - (int)wave_max(high && (uint32_t)best == lo ? (uint32_t)(kMaxCands - at) : 0);
    if (lane == r) mine = at;
    if ((at & 63) == lane) store[at] = 0;  // (read by this lane only)
  }
  wave_lds_handoff();
  return mine;
}

// ---- weights of the chosen, LPR lanes a row: lane j holds slot j -------------------------------------------------------
// (reciprocals are the hardware's: 1 ulp instead of half a one, for one instruction instead of the ten of a division)
struct Chosen {
  float share;   // s_j / sum of the chosen s (renormalised), or s_j
  float comp;    // 1 - s_j of a sigmoid
};

// l: slot j's logit, `filled`: whether slot j holds a candidate; m, z: the row's softmax (needed only when not renormalised)
template <int LPR>
__device__ __forceinline__ Chosen chosen_share(bool sigmoid, bool renormalize, float l, bool filled, float m, float z) {
  Chosen r{0.0f, 1.0f};
  float a, top = 0.0f;
  if (sigmoid) {
    const float em = expf(-fabsf(l)), inv = __builtin_amdgcn_rcpf(1.0f + em);  // (em in (0, 1]: no overflow on either side)
    r.comp = l >= 0.0f ? em * inv : inv;
    a = l >= 0.0f ? inv : em * inv;
    // Renormalised, only ratios matter: where all scores of a row are tiny the common factor is left out, so that they share
    // also below the smallest number.
    if (renormalize) {
      top = reduce_lanes<LPR, OpMax>(filled ? __builtin_fminf(l, 0.0f) : -__builtin_inff());
      if (__any(top < -60.0f)) {
        if (top < -60.0f) a = expf(__builtin_fminf(l, 0.0f) - top) * inv;
      }
    }
  } else {
    if (renormalize) top = reduce_lanes<LPR, OpMax>(filled ? l : -__builtin_inff());
    a = renormalize ? expf(l - top) : expf(l - m) * __builtin_amdgcn_rcpf(z);
  }
  a = !filled ? 0.0f : l != l ? l : a;
  r.share = a;
  if (renormalize) {
    const float total = reduce_lanes<LPR, OpSum>(a);
    r.share = total == 0.0f ? 0.0f : a * __builtin_amdgcn_rcpf(total);
  }
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

// ---- forward: LPR lanes a row, IPL consecutive candidates a lane -----------------------------------------------------
// The choice is made in fp32 and redone in 64 bits (choose_wide) for the rows where fp32 cannot tell: with a bias, when two
// neighbours of the order -- the last one taken and any candidate left among them, or the last group taken and the first one
// left -- are closer than fp32's error and are not the same (logit, bias) twice.  Without a bias the logits themselves are compared
// and nothing has to be redone.  Such rows are noted and done after every kSteps rounds, outside the loop over rows, which
// has the registers to itself then.
//
// Bound by instruction issue, not by memory: 131072 rows of 256 bf16, sigmoid with bias and 4 of 8 groups, top 8: 67 us (67 MB
// read: 1 TB/s; 54 without the 64-bit choice; 70 where the biases are all 0, as they are at first), softmax without a bias 36 us; 4099 x 64: 7 us, half of it the latency of a
// row that is done in 64 bits.  All logits equal (every row is done in 64 bits): 580 us.
//
// The top-k is not taken by k rounds of a maximum: the (k+1)-th largest of the lanes' maxima is a lower bound of the (k+1)-th
// largest candidate; the few candidates that reach it (about 10 of 256) go to a list in LDS as (key, index) and each finds
// its rank by counting the larger ones.

// the number that the lane kXor away holds, inside 16 lanes
template <int kXor>
__device__ __forceinline__ float across(float v) {
  if constexpr (kXor == 4) return across<7>(across<3>(v));
  constexpr int kCtrl = kXor == 1 ? kDppXor1 : kXor == 2 ? kDppXor2 : kXor == 3 ? 0x1B : kXor == 7 ? kDppHalfMirror
                      : kXor == 8 ? 0x128 : kDppMirror;
  return __uint_as_float(dpp32<kCtrl>(__float_as_uint(v)));
}
// A step of a sorting network over 16 lanes, largest first: of each pair of lanes the lower takes the larger number.  `way`: +inf
// in the lower lane, -inf in the other, which makes the median of three a maximum or a minimum without a comparison.
template <int kXor>
__device__ __forceinline__ float sort_step(float v, float way) { return __builtin_amdgcn_fmed3f(v, across<kXor>(v), way); }
__device__ __forceinline__ float sort16(float v, const float (&way)[4]) {
  v = sort_step<1>(v, way[0]);
  v = sort_step<1>(sort_step<3>(v, way[1]), way[0]);
  v = sort_step<1>(sort_step<2>(sort_step<7>(v, way[2]), way[1]), way[0]);
  return sort_step<1>(sort_step<2>(sort_step<4>(sort_step<15>(v, way[3]), way[2]), way[1]), way[0]);
}

// lane i of this lane's row of LPR (i the same in the whole wave)
template <int LPR>
__device__ __forceinline__ float row_lane(float v, int i) {
  if constexpr (LPR == 64) return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), i));
  else return __shfl(v, i, LPR);
}

// maxima over lanes 16 and 32 apart
template <int LPR>
__device__ __forceinline__ float max_rows(float v) {
  if constexpr (LPR >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if constexpr (LPR >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// (131072 x 256: with the maxima ranked by comparing each with all others instead of this network 7 us more.)
// A finite lower bound (or the lowest finite number) of the (k+1)-th largest value, from the maxima of two sets of values a
// lane.  (Two, because groups that were not taken leave lanes empty: with half of 16 lanes left, their 16 sets still bound
// the 9th largest.)
template <int LPR>
__device__ __forceinline__ float prune_bound(float v, float w, int k) {
  constexpr float kInf = __builtin_inff();
  float bound;
  if (LPR == 16 || (LPR > 16 && k + 1 <= 8)) {  // 32 sets: lanes 16, 32, 48 apart are put together
    v = max_rows<LPR>(v);
    w = max_rows<LPR>(w);
    const int t = threadIdx.x & 15;
    float way[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) way[i] = (t >> i) & 1 ? -kInf : kInf;
    // the 16 largest of both, in an order that four more steps sort; the (k+1)-th largest is lane k's
    v = __builtin_fmaxf(sort16(v, way), across<15>(sort16(w, way)));
    v = sort_step<1>(sort_step<2>(sort_step<4>(sort_step<8>(v, way[3]), way[2]), way[1]), way[0]);
    bound = reduce_lanes<16, OpMax>(t >= k ? v : -kInf);
  } else {
    int nv = 0, nw = 0;
    for (int i = 0; i < LPR; ++i) {
      const float a = row_lane<LPR>(v, i), b = row_lane<LPR>(w, i);
      nv += (a >= v) + (b >= v);
      nw += (a >= w) + (b >= w);
    }
    bound = reduce_lanes<LPR, OpMax>(__builtin_fmaxf(nv >= k + 1 ? v : -kInf, nw >= k + 1 ? w : -kInf));
  }
  return __builtin_fminf(__builtin_fmaxf(bound, -__FLT_MAX__), __FLT_MAX__);
}

// sum of the lanes before this one, inside groups of LPR lanes (row shifts by DPP, then whole rows of 16)
template <int kShift>
__device__ __forceinline__ int add_shifted(int v, int t) {
  const int up = __builtin_amdgcn_update_dpp(0, v, 0x110 + kShift, 0xf, 0xf, true);
  return v + (t >= kShift ? up : 0);
}
template <int LPR>
__device__ __forceinline__ int lanes_before(int v, int t) {
  int incl = add_shifted<1>(v, t & 15);
  incl = add_shifted<2>(incl, t & 15);
  incl = add_shifted<4>(incl, t & 15);
  if constexpr (LPR >= 16) incl = add_shifted<8>(incl, t & 15);
#pragma unroll
  for (int o = 16; o < LPR; o <<= 1) {
    const int up = __shfl(incl, (t & ~(o - 1)) - 1, LPR);  // (the end of the run of lanes before this one's)
    if (t & o) incl += up;
  }
  return incl - v;
}

// how many of the other 15 lanes of 16 hold a larger (hi, lo)
template <int kRor>
__device__ __forceinline__ int count_larger16(uint32_t hi, uint32_t lo) {
  if constexpr (kRor == 0) return 0;
  else {
    const uint64_t other = ((uint64_t)dpp32<0x120 + kRor>(hi) << 32) | dpp32<0x120 + kRor>(lo);
    return (other > (((uint64_t)hi << 32) | lo) ? 1 : 0) + count_larger16<kRor - 1>(hi, lo);
  }
}

// the hardware's exponential (1 ulp) of the argument rounded to base 2
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// IPL consecutive numbers of a row, as they are stored, in whole registers (of 16-bit ones a register each is taken otherwise)
template <typename T, int IPL>
struct Items {
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
  static constexpr int kPer = sizeof(T) == 4 || IPL == 1 ? 1 : 2, kWords = IPL / kPer;
  struct __attribute__((packed, aligned(sizeof(T)))) Stored { std::conditional_t<kPer == 2, uint32_t, Bits> w[kWords]; };
  uint32_t w[kWords];
  // from column `first`; `fill` behind the row's end
  __device__ __forceinline__ void load(const T* __restrict__ row, int first, int E, T fill) {
    if (first + IPL <= E) {
      const Stored s = *reinterpret_cast<const Stored*>(row + first);
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = s.w[i];
      return;
    }
    const Bits* in = reinterpret_cast<const Bits*>(row);
    const uint32_t none = __builtin_bit_cast(Bits, fill);
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      w[i] = first + i * kPer < E ? in[first + i * kPer] : none;
      if constexpr (kPer == 2) w[i] |= (first + i * 2 + 1 < E ? in[first + i * 2 + 1] : none) << 16;
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    return (float)__builtin_bit_cast(T, (Bits)(w[i / kPer] >> (kPer == 2 ? 16 * (i & 1) : 0)));
  }
};

template <typename T, int LPR, int IPL>
__global__ void __launch_bounds__(kThreads, resident(sizeof(T), LPR, IPL)) k_route_fwd(const RouteParams P) {
  constexpr int R = 64 / LPR, kRow = LPR * IPL;
  constexpr float kInf = __builtin_inff();
  __shared__ int hist[kRow];
  // a wave's candidates' values, row after row; also one row's keys in 64 bits
  __shared__ uint64_t store[kWaves][R * kRow / 2 > kRow ? R * kRow / 2 : kRow];
  __shared__ uint16_t lists[kWaves][R * kRow];  // candidates that reach the bound
  __shared__ uint64_t slot_store[kWaves][R * (LPR + 1)];
  __shared__ uint32_t redo_rows[kSteps * kWaves * R];
  __shared__ int redo_count[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / LPR, t = lane % LPR;
  float* vals = reinterpret_cast<float*>(store[wave]) + sub * kRow;
  uint16_t* list = lists[wave] + sub * kRow;
  uint64_t* slots = slot_store[wave] + sub * (LPR + 1);
  const int E = P.cands, first = t * IPL, k = P.top_k, G = P.groups, per = P.per_group;
  for (int e = threadIdx.x; e < E; e += kThreads) hist[e] = 0;
  if (threadIdx.x < 2) redo_count[threadIdx.x] = 0;
  __syncthreads();
  const bool group_scores = G > 1 && P.top2 && !P.bias;  // groups are compared by sums of scores, candidates by logits
  const bool need_scores = P.bias != nullptr || group_scores;
  const bool need_softmax = !P.sigmoid && (need_scores || !P.renormalize);
  // whole groups of lanes per group of candidates, a power of two of them: groups are formed in registers
  const int lanes_per = per / IPL;
  const bool whole = per % IPL == 0 && (lanes_per & (lanes_per - 1)) == 0;
  int share = LPR;  // else: lanes that scan one group in LDS
  while (share > 1 && LPR / share < G) share >>= 1;
  float bias[IPL];
#pragma unroll
  for (int i = 0; i < IPL; ++i) bias[i] = 0.0f;
  if (P.bias) {
    Items<float, IPL> b;
    b.load(P.bias, first, E, 0.0f);
#pragma unroll
    for (int i = 0; i < IPL; ++i) bias[i] = b[i];
  }

  bool odd_bias = false;  // infinities or NaN among the biases
#pragma unroll
  for (int i = 0; i < IPL; ++i) odd_bias |= !(fabsf(bias[i]) < kInf);
  odd_bias = __any(odd_bias);

  const uint32_t last = (uint32_t)P.rows - 1, per_step = kWaves * R, row_groups = last / per_step + 1;
  const auto row_at = [&](uint32_t row) { return static_cast<const T*>(P.logits) + (uint64_t)row * (uint64_t)P.stride; };
  uint32_t row = min(blockIdx.x * per_step + wave * R + sub, last);
  constexpr T kNone = (T)-__builtin_inff();
  Items<T, IPL> ahead;
  ahead.load(row_at(row), first, E, kNone);
  int flip = 0;
  for (uint32_t rg0 = blockIdx.x; rg0 < row_groups; rg0 += kSteps * gridDim.x) {
    for (uint32_t rg = rg0; rg < min(rg0 + kSteps * gridDim.x, row_groups); rg += gridDim.x) {
      const uint32_t want = rg * per_step + wave * R + sub;
      const bool mine = want <= last;
      row = min(want, last);
      const T* src = row_at(row);
      float c[IPL];  // logits, then what the candidates are compared by; -inf: not eligible
      float probe = 0.0f;
#pragma unroll
      for (int i = 0; i < IPL; ++i) {
        c[i] = ahead[i];
        probe = __builtin_fmaf(c[i], 0.0f, probe);  // NaN as soon as one logit is not finite
      }
      const bool odd = odd_bias || __any(probe != probe);  // (E not a multiple of IPL: the places behind the end are -inf)
      ahead.load(row_at(min((rg + gridDim.x) * per_step + wave * R + sub, last)), first, E, kNone);

      // err: bound of two scores' errors.  sigmoid: s (1 - s) (|l| 2^-23.4 + 2^-23) of the exponential, 2^-23 of the
      // reciprocal, 2^-24 of the sum: below 2^-22 each.  softmax, relative to its largest score 1 / z: as much of the
      // exponential and up to 30 roundings of z, below 2^-19 each.  Of the two together twice as much is taken in either case.
      float m = 0.0f, z = 1.0f, inv_z = 1.0f, err = 0x1p-20f;
      if (need_softmax) {
        float mf = c[0];
#pragma unroll
        for (int i = 1; i < IPL; ++i) mf = __builtin_fmaxf(mf, c[i]);
        mf = reduce_lanes<LPR, OpMax>(mf);
        m = mf == -kInf ? 0.0f : mf;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < IPL; ++i) sum += fast_exp(c[i] - m);
        z = reduce_lanes<LPR, OpSum>(sum);
        if (z == 0.0f) z = 1.0f;
        inv_z = 1.0f / z;
        err = 0x1p-17f * inv_z;
      }
      float a = -kInf, b = -kInf;  // the two largest of this lane's part of its group
      if (need_scores) {
        float s[IPL];
        if (P.sigmoid) {
#pragma unroll
          for (int i = 0; i < IPL; ++i) s[i] = __builtin_amdgcn_rcpf(1.0f + fast_exp(-c[i]));
        } else {
#pragma unroll
          for (int i = 0; i < IPL; ++i) s[i] = fast_exp(c[i] - m) * inv_z;
        }
        if (P.bias) {
#pragma unroll
          for (int i = 0; i < IPL; ++i) s[i] += bias[i];
          if (odd) {  // (a NaN score does not take a ruling out back)
#pragma unroll
            for (int i = 0; i < IPL; ++i) s[i] = c[i] == -kInf || bias[i] == -kInf ? -kInf : s[i];
          }
#pragma unroll
          for (int i = 0; i < IPL; ++i) c[i] = s[i];
        } else {  // the groups' values are of the scores
#pragma unroll
          for (int i = 0; i < IPL; ++i) {
            s[i] = c[i] == -kInf ? -kInf : s[i] != s[i] ? kInf : s[i];
            if (!whole) vals[first + i] = s[i];
            const float lo = __builtin_fminf(a, s[i]);
            a = __builtin_fmaxf(a, s[i]);
            b = __builtin_fmaxf(b, lo);
          }
        }
      }
      if (odd) {
#pragma unroll
        for (int i = 0; i < IPL; ++i) c[i] = c[i] != c[i] ? kInf : c[i];
      }

      bool close = false;  // fp32 cannot tell
      bool in_group = true;  // (whole groups of lanes) this lane's group is taken
      if (G > 1) {
        if (!group_scores) {
          if (whole && !P.top2) {
#pragma unroll
            for (int i = 0; i < IPL; ++i) a = __builtin_fmaxf(a, c[i]);
          } else if (whole) {
#pragma unroll
            for (int i = 0; i < IPL; ++i) {
              const float lo = __builtin_fminf(a, c[i]);
              a = __builtin_fmaxf(a, c[i]);
              b = __builtin_fmaxf(b, lo);
            }
          } else {
            wave_lds_handoff();
#pragma unroll
            for (int i = 0; i < IPL; ++i) vals[first + i] = c[i];
          }
        }
        const int width = whole ? lanes_per : share;  // lanes that hold the same group
        if (!whole) {
          wave_lds_handoff();
          const int g = t / share;
          a = b = -kInf;
          if (g < G)
            for (int i = t % share; i < per; i += share) {
              const float v = vals[g * per + i], lo = __builtin_fminf(a, v);
              a = __builtin_fmaxf(a, v);
              b = __builtin_fmaxf(b, lo);
            }
        }
        for (int o = 1; o < width; o <<= 1) {
          const float a2 = __shfl_xor(a, o), b2 = __shfl_xor(b, o);
          b = __builtin_fmaxf(__builtin_fminf(a, a2), __builtin_fmaxf(b, b2));
          a = __builtin_fmaxf(a, a2);
        }
        // (two biases of the lowest number stay above a group that nothing is eligible of)
        const float g = P.top2 && b != -kInf ? __builtin_fmaxf(a + b, -__FLT_MAX__) : a;
        const int my_group = t / width;
        // by (value, lower index): a group's rank is the number of groups before it
        const uint32_t hi = order_key(g), lo = (uint32_t)(kMaxGroups - my_group);
        int rank = 0;
        for (int o = 0; o < G; o += 4) {
          uint32_t other[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) other[i] = (uint32_t)__shfl((int)hi, min(o + i, G - 1) * width, LPR);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint64_t mine_key = ((uint64_t)hi << 32) | lo;
            rank += o + i < G && (((uint64_t)other[i] << 32) | (uint32_t)(kMaxGroups - o - i)) > mine_key;
          }
        }
        const bool taken = my_group < G && rank < P.top_groups;
        if (need_scores && P.top_groups < G) {  // the last group taken against the first one left
          const uint64_t at_last = __ballot(my_group < G && rank == P.top_groups - 1) >> (sub * LPR);
          const float worst = __shfl(g, __builtin_ctzll(at_last), LPR);
          if (my_group < G && rank == P.top_groups && g != -kInf)
            close = !(worst - g > 2.0f * err + 0x1p-21f * (fabsf(worst) + fabsf(g)));  // (inf - inf: cannot tell)
        }
        if (whole) {
          in_group = taken;
        } else {
          const uint64_t kept = (__ballot(taken) >> (sub * LPR));  // bit t: lane t's group is taken
          int from = first;
          asm("" : "+v"(from));  // (or the 16 places' groups are worked out before the loop over rows, and registers run out)
          int at = from / per, in = from % per;
#pragma unroll
          for (int i = 0; i < IPL; ++i) {
            if (at >= G || !((kept >> (at * share)) & 1)) c[i] = -kInf;
            if (++in == per) {
              in = 0;
              ++at;
            }
          }
        }
      }

      // the candidates that can be among the k + 1 largest: their places in a list, their values in LDS
      float bound = -__FLT_MAX__;
      if constexpr (IPL > 1) {
        float v = c[0], w = c[IPL / 2];
#pragma unroll
        for (int i = 1; i < IPL / 2; ++i) {
          v = __builtin_fmaxf(v, c[i]);
          w = __builtin_fmaxf(w, c[IPL / 2 + i]);
        }
        bound = prune_bound<LPR>(in_group ? v : -kInf, in_group ? w : -kInf, k);
      }
      // by the signs of the differences: no comparison, no carry to wait for.  A bound of 0 is made -0, from which neither 0 nor
      // -0 leaves -0.
      if (bound == 0.0f) bound = -0.0f;
      uint32_t below = 0;
#pragma unroll
      for (int i = IPL - 1; i >= 0; --i) below = __builtin_amdgcn_alignbit(below, __float_as_uint(c[i] - bound), 31);
      uint32_t reach = in_group ? ~below & ((1u << IPL) - 1) : 0;
      wave_lds_handoff();
#pragma unroll
      for (int i = 0; i < IPL; ++i) vals[first + i] = c[i];
      int before = lanes_before<LPR>(__popc(reach), t);
      int n = __shfl(before + __popc(reach), LPR - 1, LPR);
      if (__any(n > 2 * LPR)) {  // many equal values: of those at the bound the first k + 1 will do
        uint32_t larger = 0;
#pragma unroll
        for (int i = IPL - 1; i >= 0; --i) larger = 2 * larger + (c[i] > bound);
        larger &= reach;
        uint32_t equal = reach & ~larger, kept = 0;
        int left = k + 1 - lanes_before<LPR>(__popc(equal), t);
        for (; equal && left > 0; --left, equal &= equal - 1) kept |= equal & (0u - equal);
        reach = larger | kept;
        before = lanes_before<LPR>(__popc(reach), t);
        n = __shfl(before + __popc(reach), LPR - 1, LPR);
      }
      for (; reach; reach &= reach - 1) list[before++] = (uint16_t)(first + __builtin_ctz(reach));
      for (int j = t; j <= k; j += LPR) slots[j] = 0;
      wave_lds_handoff();
      const auto entry = [&](int j) {
        const int e = list[j];
        return ((uint64_t)order_key(vals[e]) << 32) | (uint32_t)(kMaxCands - e);  // (of equal values the lower index is larger)
      };
      uint64_t own = t < n ? entry(t) : 0;
      int n_max = n;
      if constexpr (R > 1) n_max = (int)reduce_lanes<64, OpMax>((float)n);
      constexpr int kPer = IPL < 8 ? (IPL > 1 ? IPL / 2 : 1) : 4;  // entries a lane that fit over the values
      if (n_max <= LPR) {
        int rank = 0;
        if constexpr (LPR == 16) {
          rank = count_larger16<15>((uint32_t)(own >> 32), (uint32_t)own);
        } else {
          const float hi = __uint_as_float((uint32_t)(own >> 32)), lo = __uint_as_float((uint32_t)own);
          for (int i = 0; i < n_max; ++i)
            rank += (((uint64_t)__float_as_uint(row_lane<LPR>(hi, i)) << 32) | __float_as_uint(row_lane<LPR>(lo, i))) > own;
        }
        if (own && rank <= k) slots[rank] = own;
      } else if (n_max <= kPer * LPR) {
        uint64_t mine_all[kPer];
#pragma unroll
        for (int q = 0; q < kPer; ++q) mine_all[q] = t + q * LPR < n ? entry(t + q * LPR) : 0;
        wave_lds_handoff();
        uint64_t* entries = store[wave] + sub * (kPer * LPR);
#pragma unroll
        for (int q = 0; q < kPer; ++q) entries[t + q * LPR] = mine_all[q];
        wave_lds_handoff();
        int rank[kPer] = {};
#pragma unroll 2
        for (int i = 0; i < n_max; ++i) {
          const uint64_t other = entries[i];
#pragma unroll
          for (int q = 0; q < kPer; ++q) rank[q] += other > mine_all[q];
        }
#pragma unroll
        for (int q = 0; q < kPer; ++q)
          if (mine_all[q] && rank[q] <= k) slots[rank[q]] = mine_all[q];
      } else {
        for (int j = t; j < n; j += LPR) {
          own = entry(j);
          int rank = 0;
          for (int i = 0; i < n; ++i) rank += entry(i) > own;
          if (rank <= k) slots[rank] = own;
        }
      }
      wave_lds_handoff();

      const uint64_t got = t < k ? slots[t] : 0;
      const int at = got ? kMaxCands - (int)(uint32_t)got : -1;
      // Neighbours of the order that fp32 cannot tell, unless they are one (logit, bias) twice.  Where the last one taken and the
      // first one left are one pair, this pair says nothing of what comes behind it: every candidate is looked at, also those
      // that the bound or the cut of equal values kept off the list.  (Larger values are in slots before, where each has been held
      // against its neighbour.)
      if (P.bias) {
        bool cut_same = false;
        const float v = key_value((uint32_t)(got >> 32));
        if (got) {
          const uint64_t next = slots[t + 1];
          const float v2 = key_value((uint32_t)(next >> 32));
          if (next && v - v2 <= err + 0x1p-22f * (fabsf(v) + fabsf(v2))) {
            const int at2 = kMaxCands - (int)(uint32_t)next;
            const bool same = (float)src[at] == (float)src[at2] && P.bias[at] == P.bias[at2];
            close |= !same;
            cut_same = same && t == k - 1;
          }
        }
        if (__any(cut_same)) {
          const float worst = __shfl(v, k - 1, LPR);
          const int at_cut = __shfl(cut_same ? at : -1, k - 1, LPR);
          // from here up to `worst` fp32 cannot tell: the tolerance above with both values taken for the larger, and a little more
          const float least = __builtin_fmaxf(worst - (err + 0x1.4p-21f * fabsf(worst)) * 1.0001f, -__FLT_MAX__);
          uint32_t near = 0;
#pragma unroll
          for (int i = 0; i < IPL; ++i) near |= c[i] >= least && c[i] <= worst ? 1u << i : 0;
          if (at_cut < 0 || !in_group) near = 0;
          for (; near; near &= near - 1) {
            const int e = first + __builtin_ctz(near);
            close |= !((float)src[e] == (float)src[at_cut] && P.bias[e] == P.bias[at_cut]);
          }
        }
      }
      const uint64_t all_close = __ballot(close && mine);
      const bool redo = R == 1 ? all_close != 0 : ((all_close >> (sub * LPR)) & ((1ull << (LPR & 63)) - 1)) != 0;
      if (redo && t == 0) redo_rows[atomicAdd(&redo_count[flip], 1)] = row;

      const Chosen ch = chosen_share<LPR>(P.sigmoid, P.renormalize, at >= 0 ? (float)src[at] : 0.0f, at >= 0, m, z);
      if (mine && t < k && !redo) {
        const uint64_t out = (uint64_t)row * (uint32_t)k + t;
        P.weights[out] = z != z ? z : P.scale * ch.share;  // (a NaN in a softmax is in every score)
        P.indices[out] = at;
        if (at >= 0) atomicAdd(&hist[at], 1);
      }
    }
    // the rows that fp32 could not tell, a wave each
    if (!need_scores) continue;
    __syncthreads();
    const int n_redo = redo_count[flip];
    flip ^= 1;
    if (threadIdx.x == 0) redo_count[flip] = 0;
    for (int i = wave; i < n_redo; i += kWaves) {
      const uint32_t again = redo_rows[i];
      const T* src = row_at(again);
      const int at = choose_wide<T>(P, src, store[wave]);
      float m = 0.0f, z = 1.0f;
      if (!P.sigmoid) row_softmax<T, 64>(src, E, lane, m, z);
      const Chosen ch = chosen_share<64>(P.sigmoid, P.renormalize, at >= 0 ? (float)src[at] : 0.0f, at >= 0, m, z);
      if (lane < k) {
        const uint64_t out = (uint64_t)again * (uint32_t)k + lane;
        P.weights[out] = z != z ? z : P.scale * ch.share;
        P.indices[out] = at;
        if (at >= 0) atomicAdd(&hist[at], 1);
      }
    }
    __syncthreads();
  }
  __syncthreads();
  int32_t* out = P.parts > 1 ? P.ws + (int64_t)blockIdx.x * E : P.counts;
  for (int e = threadIdx.x; e < E; e += kThreads) out[e] = hist[e];
}

// counts = the sums of the workgroups' counts: 32 candidates a workgroup, 32 groups of threads over the partial rows (1024 of
// them: 4.6 us, the latency of 32 loads and of the sums after them; 257: 1.9 us).  Nothing has to be cleared beforehand.
__global__ void __launch_bounds__(1024) k_route_counts(const RouteParams P) {
  __shared__ int acc[32][33];
  const int c = threadIdx.x & 31, grp = threadIdx.x >> 5, e = blockIdx.x * 32 + c;
  int s = 0;
  if (e < P.cands) {
#pragma unroll 8
    for (int p = grp; p < P.parts; p += 32) s += P.ws[(int64_t)p * P.cands + e];
  }
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
// A row of gradients is put together in LDS (zeros and the k chosen) and stored in 16-byte pieces: 131072 x 256 bf16, top 8,
// 21 to 24 us, bound by its 67 MB of stores.
template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads) k_route_bwd(const RouteParams P) {
  constexpr int R = 64 / LPR, kRow = LPR * 16, N = Elem<T>::kN;
  __shared__ __align__(16) float rows[kWaves][R * kRow];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / LPR, t = lane % LPR;
  float* acc = rows[wave] + sub * kRow;
  const int64_t want = ((P.block0 + blockIdx.x) * kWaves + wave) * R + sub;
  const bool mine = want < P.rows;
  const int64_t row = mine ? want : P.rows - 1;
  const T* l = static_cast<const T*>(P.logits) + row * P.stride;
  const int64_t slot = t < P.top_k ? P.indices[row * P.top_k + t] : -1;
  const bool filled = slot >= 0 && slot < P.cands;
  const int at = filled ? (int)slot : -1;
  const float dw = filled ? P.grad_w[row * P.top_k + t] : 0.0f;
  const bool dense = !P.sigmoid && !P.renormalize;
  // a NaN in a softmax is in every score: the forward left it in every weight of the row
  const float first = P.weights[row * P.top_k];
  const float base = !P.sigmoid && first != first ? first : 0.0f;
  for (int e = 4 * t; e < P.cands; e += 4 * LPR) *reinterpret_cast<f32x4_lds*>(acc + e) = f32x4_lds{base, base, base, base};
  float m = 0.0f, z = 1.0f;
  if (dense) row_softmax<T, LPR>(l, P.cands, t, m, z);
  const Chosen c = chosen_share<LPR>(P.sigmoid, P.renormalize, filled ? (float)l[at] : 0.0f, filled, m, z);
  float g;
  if (P.renormalize) {
    float d = 0.0f;
    for (int i = 0; i < P.top_k; ++i) {
      const float wi = __shfl(c.share, i, LPR), di = __shfl(dw, i, LPR);
      d = __builtin_fmaf(wi, dw - di, d);
    }
    g = P.scale * c.share * d * c.comp;
  } else {
    g = P.scale * dw * (dense ? 1.0f : c.share * c.comp);
  }
  const float dot = dense ? reduce_lanes<LPR, OpSum>(filled ? g * c.share : 0.0f) : 0.0f;
  wave_lds_handoff();
  if (filled) acc[at] = base + g;
  wave_lds_handoff();
  if (!mine) return;
  T* out = static_cast<T*>(P.grad) + row * P.cands;
  for (int e = t * N; e < P.cands; e += LPR * N) {
    typename Elem<T>::Vec o;
    if (dense) {
      const auto v = load16<T>(l, e, P.cands, (T)-__builtin_inff());
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = (T)(expf((float)v[j] - m) / z * (acc[e + j] - dot));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = (T)acc[e + j];
    }
    store16<T>(out, e, P.cands, o);
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

// Lanes a row and candidates a lane: the fewest lanes that hold the row 16 a lane, one choice and one group a lane (8 lanes:
// rows of at most 8 candidates) -- lane exchanges cost the same for one row as for eight.  Where a lane holds several
// candidates there is one lane more than choices, or prune_bound has nothing to go by.
struct RouteShape { int lpr, ipl; };
RouteShape route_shape(int cands, int top_k, int groups) {
  const int need = std::max(top_k, groups);
  RouteShape s{64, 1};
  if (cands <= 8) s.lpr = 8;
  else if (cands <= 256 && need <= (cands <= 16 ? 16 : 15)) s.lpr = 16;
  else if (cands <= 512 && need <= (cands <= 32 ? 32 : 31)) s.lpr = 32;
  while (s.lpr * s.ipl < cands) s.ipl *= 2;
  if (s.lpr > 16) s.ipl = s.ipl == 2 ? 4 : s.ipl == 8 ? 16 : s.ipl;  // (1, 4 and 16 only: these rows are rare)
  return s;
}

int route_parts(int64_t rows, int lpr, int most) { return (int)std::min<int64_t>(ceil_div(rows, kWaves * (64 / lpr)), kCus * most); }

template <typename T>
void launch_fwd(const RouteParams& P, RouteShape s, hipStream_t st) {
#define UR_ROUTE(L, I) \
  if (s.lpr == L && s.ipl == I) k_route_fwd<T, L, I><<<P.parts, kThreads, 0, st>>>(P);
  UR_ROUTE(8, 1) UR_ROUTE(16, 1) UR_ROUTE(16, 2) UR_ROUTE(16, 4) UR_ROUTE(16, 8) UR_ROUTE(16, 16)
  UR_ROUTE(32, 1) UR_ROUTE(32, 4) UR_ROUTE(32, 16) UR_ROUTE(64, 1) UR_ROUTE(64, 4) UR_ROUTE(64, 16)
#undef UR_ROUTE
}

template <typename T>
void launch_bwd(const RouteParams& P, int lpr, hipStream_t st) {
  in_pieces(ceil_div(P.rows, kWaves * (64 / lpr)), kThreads, [&](int64_t first, unsigned grid) {
    RouteParams Q = P;
    Q.block0 = first;
    if (lpr == 8) k_route_bwd<T, 8><<<grid, kThreads, 0, st>>>(Q);
    else if (lpr == 16) k_route_bwd<T, 16><<<grid, kThreads, 0, st>>>(Q);
    else if (lpr == 32) k_route_bwd<T, 32><<<grid, kThreads, 0, st>>>(Q);
    else k_route_bwd<T, 64><<<grid, kThreads, 0, st>>>(Q);
  });
}

}  // namespace

extern "C" {

int64_t ur_route_workspace_bytes(int64_t rows, int cands) {
  if (rows <= 0 || cands <= 0 || rows > 0x7fffffff || cands > kMaxCands)
    return set_error(UR_ERR_INVALID_ARG, "bad rows or cands");
  const int parts = route_parts(rows, 64, 4);  // (the most any shape needs)
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
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  RouteParams P{};
  P.logits = logits; P.stride = row_stride; P.bias = bias; P.rows = rows; P.cands = cands; P.top_k = top_k;
  P.groups = groups; P.per_group = cands / groups; P.top_groups = top_groups;
  P.sigmoid = score == UR_SCORE_SIGMOID; P.top2 = group_score == UR_GROUP_TOP2; P.renormalize = renormalize != 0;
  P.scale = scale; P.weights = weights; P.indices = indices; P.counts = counts;
  const RouteShape shape = route_shape(cands, top_k, groups);
  P.ws = static_cast<int32_t*>(workspace); P.parts = route_parts(rows, shape.lpr, resident(dtype_bytes(dtype), shape.lpr, shape.ipl));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UR_F32) launch_fwd<float>(P, shape, st);
  else if (dtype == UR_F16) launch_fwd<_Float16>(P, shape, st);
  else launch_fwd<__bf16>(P, shape, st);
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
  const int lpr = cands <= 8 ? 8 : cands <= 256 && top_k <= 16 ? 16 : cands <= 512 && top_k <= 32 ? 32 : 64;
  if (dtype == UR_F32) launch_bwd<float>(P, lpr, st);
  else if (dtype == UR_F16) launch_bwd<_Float16>(P, lpr, st);
  else launch_bwd<__bf16>(P, lpr, st);
  return launch_status("ur_route_backward");
}

}  // extern "C"
