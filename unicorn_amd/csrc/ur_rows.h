// Building blocks of the row-wise operators (ur_layer_norm.hip, ur_route.hip, ur_distill.hip): element types,
// 16-byte row accesses, reductions over groups of lanes and over a workgroup.  gfx950 only, wave64.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/unicorn_render.h"
#include "ur_status.h"

namespace ur {

// ---- element types: storage type, elements per 16-byte access ------------------------------------------------------
// The vector types are declared with the alignment of ONE element: rows of odd length or stride start anywhere, and the
// hardware's unaligned global accesses (the default mode of the target) take a 16-byte access at any such address.
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8), aligned(2)));

template <typename T> struct Elem;
template <> struct Elem<float> { using Vec = f32x4; static constexpr int kN = 4; };
template <> struct Elem<_Float16> { using Vec = f16x8; static constexpr int kN = 8; };
template <> struct Elem<__bf16> { using Vec = bf16x8; static constexpr int kN = 8; };

// kN elements from column `col` of a row of `cols`; what lies behind the row's end reads as `fill`
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec load16(const T* __restrict__ row, int64_t col, int64_t cols, T fill) {
  constexpr int N = Elem<T>::kN;
  if (col + N <= cols) return *reinterpret_cast<const typename Elem<T>::Vec*>(row + col);
  typename Elem<T>::Vec v;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = (col + j < cols) ? row[col + j] : fill;
  return v;
}

// stores the part of `v` that lies inside the row
template <typename T>
__device__ __forceinline__ void store16(T* __restrict__ row, int64_t col, int64_t cols, typename Elem<T>::Vec v) {
  constexpr int N = Elem<T>::kN;
  if (col + N <= cols) {
    *reinterpret_cast<typename Elem<T>::Vec*>(row + col) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (col + j < cols) row[col + j] = v[j];
}

// the same for a result that nobody reads soon, past the caches, which keep something better
template <typename T>
__device__ __forceinline__ void store16_past(T* __restrict__ row, int64_t col, int64_t cols, typename Elem<T>::Vec v) {
  if (col + Elem<T>::kN <= cols) __builtin_nontemporal_store(v, reinterpret_cast<typename Elem<T>::Vec*>(row + col));
  else store16<T>(row, col, cols, v);
}

// one element of a tensor whose type is known at run time only (parameters, small side inputs)
__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
  if (dtype == UR_F32) return static_cast<const float*>(p)[i];
  if (dtype == UR_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}

__device__ __forceinline__ void store_from_float(void* p, int dtype, int64_t i, float v) {
  if (dtype == UR_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == UR_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
  else static_cast<__bf16*>(p)[i] = (__bf16)v;
}

// ---- reductions over L consecutive lanes (L = 4, 8, 16, 32 or 64); every lane of the group gets the result ----------
// All lanes of the wave have to be active.  Up to 16 lanes by DPP (one VALU instruction a step); a mirrored row stands in
// for the exchange of two halves because the halves are uniform by then.  Beyond, the two row-swap instructions.
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kCtrl, 0xf, 0xf, true);  // (every lane has a source: nothing is left as it was)
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

struct OpSum {
  static __device__ __forceinline__ float f(float a, float b) { return a + b; }
};
struct OpMax {
  static __device__ __forceinline__ float f(float a, float b) { return __builtin_fmaxf(a, b); }
};

template <int kCtrl, typename Op>
__device__ __forceinline__ float dpp_step(float v) {
  return Op::f(v, __uint_as_float(dpp32<kCtrl>(__float_as_uint(v))));
}

template <int L, typename Op>
__device__ __forceinline__ float reduce_lanes(float v) {
  if constexpr (L >= 2) v = dpp_step<kDppXor1, Op>(v);
  if constexpr (L >= 4) v = dpp_step<kDppXor2, Op>(v);
  if constexpr (L >= 8) v = dpp_step<kDppHalfMirror, Op>(v);
  if constexpr (L >= 16) v = dpp_step<kDppMirror, Op>(v);
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = Op::f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = Op::f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// What step kStep (lanes 1, 2, 4, 8, 16, 32 apart, or the mirror that stands in for it) of such a reduction combines a lane's
// value with.
template <int kStep>
__device__ __forceinline__ uint32_t other_lane(uint32_t v) {
  if constexpr (kStep < 4) {
    constexpr int kCtrl[4] = {kDppXor1, kDppXor2, kDppHalfMirror, kDppMirror};
    return dpp32<kCtrl[kStep]>(v);
  } else if constexpr (kStep == 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return r[0] ^ r[1] ^ v;  // (one of the two is the lane's own)
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return r[0] ^ r[1] ^ v;
  }
}

// sum of 64-bit numbers over L consecutive lanes
template <int L, int kStep = 0>
__device__ __forceinline__ double sum_lanes(double v) {
  if constexpr ((1 << kStep) < L) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint64_t o = ((uint64_t)other_lane<kStep>((uint32_t)(b >> 32)) << 32) | other_lane<kStep>((uint32_t)b);
    return sum_lanes<L, kStep + 1>(v + __longlong_as_double((long long)o));
  } else {
    return v;
  }
}

// Sums over TPR threads: a group of lanes (TPR <= 64), or the whole workgroup through LDS (`part`: kN floats per
// wave; the partial sums are added in wave order, so the result does not depend on timing).  The caller puts a barrier
// between two uses of the same `part`.
template <int TPR, int kN>
__device__ __forceinline__ void sum_threads(float (&v)[kN], float* part) {
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = reduce_lanes<(TPR < 64 ? TPR : 64), OpSum>(v[i]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < kN; ++i) part[wave * kN + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += part[w * kN + i];
      v[i] = s;
    }
  }
}

// A wave hands values to its own lanes through LDS: the compiler must not move the accesses across this point.
__device__ __forceinline__ void wave_lds_handoff() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A launch holds less than 2^32 threads (2^29 rows of 8 lanes are more): larger grids go out in pieces, launch(first
// workgroup, workgroups).
template <typename F>
void in_pieces(int64_t blocks, int threads, const F& launch) {
  const int64_t most = 0xffffffffll / threads;
  for (int64_t b = 0; b < blocks; b += most) launch(b, (unsigned)(blocks - b < most ? blocks - b : most));
}
inline bool known_dtype(int d) { return d == UR_F32 || d == UR_F16 || d == UR_BF16; }
inline int dtype_bytes(int d) { return d == UR_F32 ? 4 : 2; }

}  // namespace ur
