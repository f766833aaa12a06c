// Row-wise training kernels (LayerNorm, rotary head norm): element types, sums over the lanes of a row, and the
// reduction of the parameters' gradients from the partial rows of work-groups.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace saf3r {

template <int N>
using Int = std::integral_constant<int, N>;

// VE elements of T at p (16-byte aligned for VE > 1) as floats.
template <int VE, typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[VE]) {
  typedef T vec __attribute__((ext_vector_type(VE)));
  if constexpr (VE == 1) {
    x[0] = (float)p[0];
  } else {
    const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = (float)v[e];
  }
}

template <int VE, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[VE]) {
  typedef T vec __attribute__((ext_vector_type(VE)));
  if constexpr (VE == 1) {
    p[0] = (T)x[0];
  } else {
    vec v;
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = (T)x[e];
    *reinterpret_cast<vec*>(p) = v;
  }
}

// The first `n` of VE elements at p, which is aligned to its elements only; zeros behind them. A whole vector is one load
// (global memory takes any dword, and here any element, alignment).
template <int VE, typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&x)[VE]) {
  typedef T vec __attribute__((ext_vector_type(VE)));
  typedef vec any __attribute__((aligned(sizeof(T))));
  if (n >= VE) {
    const vec v = *reinterpret_cast<const any*>(p);
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = e < n ? (float)p[e] : 0.f;
  }
}

template <int VE, typename T>
__device__ __forceinline__ void store_some(T* p, int n, const float (&x)[VE]) {
  typedef T vec __attribute__((ext_vector_type(VE)));
  typedef vec any __attribute__((aligned(sizeof(T))));
  if (n >= VE) {
    vec v;
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = (T)x[e];
    *reinterpret_cast<any*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (e < n) p[e] = (T)x[e];
  }
}

// VE parameters from element c of a tensor, or `none` where there is no tensor. (The element type is a template
// argument: a branch on a run-time type around these loads was compiled so that one arm left the column of the
// store behind it unset.)
template <int VE, typename TP>
__device__ __forceinline__ void load_param(const void* p, int64_t c, float none, float (&x)[VE]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = none;
  } else {
    load_vec<VE>((const TP*)p + c, x);
  }
}

// Sum over groups of W consecutive lanes (a power of two up to 64), in every lane of the group: within rows of 16
// lanes by DPP, then row pairs and halves by the permlane swaps.
template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
  if constexpr (W >= 2) x += dpp_mov<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  if constexpr (W >= 4) x += dpp_mov<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  if constexpr (W >= 8) x += dpp_mov<0x141>(x);  // row_half_mirror
  if constexpr (W >= 16) x += dpp_mov<0x140>(x); // row_mirror
  if constexpr (W >= 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  if constexpr (W >= 64) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  return x;
}

// 1 / sqrt(x) to fp32 accuracy: the hardware's estimate (1 ulp) with one Newton step; inf for 0.
__device__ __forceinline__ float inv_sqrt(float x) {
  const float r = __builtin_amdgcn_rsqf(x);
  const float n = r * (1.5f - 0.5f * x * r * r);
  return x > 1e-37f && x < 1e37f ? n : r;
}

// Sum over the lanes of a wave that have the same place in their group of W lanes, in each of them: rotations within
// rows of 16 lanes, then row pairs and halves.
template <int W>
__device__ __forceinline__ float groups_sum(float x) {
  if constexpr (W <= 2) x += dpp_mov<0x122>(x);  // row_ror:2
  if constexpr (W <= 4) x += dpp_mov<0x124>(x);  // row_ror:4
  if constexpr (W <= 8) x += dpp_mov<0x128>(x);  // row_ror:8
  if constexpr (W <= 16) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  if constexpr (W <= 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  return x;
}

// Adds the VE values of every lane over the groups of W lanes of a work-group of 256 (waves first, then four waves
// through LDS); the sums end in the first group. lds: 4 * 64 * VE floats (not used where there is one group).
template <int VE, int W>
__device__ __forceinline__ void add_slots(float (&x)[VE], float* lds) {
  if constexpr (W < 256) {
    constexpr int kLanes = W < 64 ? W : 64;
    const int lane = tid_x() & 63, wave = tid_x() >> 6;
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = groups_sum<kLanes>(x[e]);
    __syncthreads();
    if (lane < kLanes) {
#pragma unroll
      for (int e = 0; e < VE; ++e) lds[(e * 4 + wave) * kLanes + lane] = x[e];
    }
    __syncthreads();
    if (tid_x() < kLanes) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float* at = lds + e * 4 * kLanes + lane;
        x[e] = (at[0] + at[kLanes]) + (at[2 * kLanes] + at[3 * kLanes]);
      }
    }
  }
}

// Parameters are fp32, or of the rows' 16-bit type (`half`: the 16-bit one of the row types, or fp32).
inline int param_check(const char* who, int param_type, int half) {
  if (param_type != SAF3R_FP32 && param_type != half)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: parameters of type %d: fp32 or the rows' 16-bit type", who, param_type);
  return SAF3R_OK;
}

// dweight / dbias (each may be null) of n columns from `parts` partial rows [part][2][n], in part order per slice.
int sum_parts(const char* who, const float* part, int64_t parts, int n, void* dweight, void* dbias, int type,
              hipStream_t stream);

// A row tensor's pointer and stride (elements) as the row kernels need them; written rows do not overlap.
inline int row_check(const char* who, const void* ptr, int64_t stride, int dim, int type, bool written) {
  if ((uintptr_t)ptr % (type == SAF3R_FP32 ? 4 : 2))
    return fail(SAF3R_ERR_INVALID, "%s: rows must be aligned to their elements", who);
  if (stride < 0 || (written && stride < dim))
    return fail(SAF3R_ERR_INVALID, "%s: row stride %lld for rows of %d", who, (long long)stride, dim);
  return SAF3R_OK;
}

}  // namespace saf3r
