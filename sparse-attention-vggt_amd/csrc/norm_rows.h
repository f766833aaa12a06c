// Rows that lie in the registers of the lanes that own them: a part of a wave, a wave or a work-group a row (LayerNorm, gated
// residual with norm).
#pragma once

#include "row_ops.h"

namespace saf3r {

// Sum over the TPR lanes of a row (TPR 256: the work-group, through LDS).
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* lds) {
  if constexpr (TPR <= 64) {
    return lanes_sum<TPR>(x);
  } else {
    x = lanes_sum<64>(x);
    const int wave = tid_x() >> 6;
    __syncthreads();
    if ((tid_x() & 63) == 0) lds[wave] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
}

// Vectors of a row: whole and aligned, or (SOME) aligned to their elements, the last one of a row shorter.
template <bool SOME, int VE, typename T>
__device__ __forceinline__ void get(const T* p, int n, float (&x)[VE]) {
  if constexpr (SOME)
    load_some<VE>(p, n, x);
  else
    load_vec<VE>(p, x);
}
template <bool SOME, int VE, typename T>
__device__ __forceinline__ void put(T* p, int n, const float (&x)[VE]) {
  if constexpr (SOME)
    store_some<VE>(p, n, x);
  else
    store_vec<VE>(p, x);
}
template <bool SOME, int VE, typename TP>
__device__ __forceinline__ void get_param(const void* p, int c, int n, float none, float (&x)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) x[e] = none;
  if (p) get<SOME, VE>((const TP*)p + c, n, x);
}

constexpr int kVe = 8;  // elements of a vector

constexpr int kLnMaxDim = 8192;

inline int ln_check(const char* who, int64_t rows, int dim, int x_type, int y_type, int param_type) {
  if (rows < 0 || dim <= 0) return fail(SAF3R_ERR_INVALID, "%s: invalid sizes: %lld rows of %d", who, (long long)rows, dim);
  if (dim > kLnMaxDim) return fail(SAF3R_ERR_UNSUPPORTED, "%s: rows of %d (at most %d)", who, dim, kLnMaxDim);
  if (rows > (int64_t)1 << 38) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many rows", who);
  for (int t : {x_type, y_type, param_type})
    if (t < SAF3R_FP32 || t > SAF3R_FP16) return fail(SAF3R_ERR_INVALID, "%s: unknown element type %d", who, t);
  if (y_type != x_type && x_type != SAF3R_FP32)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: 16-bit rows keep their type (types %d and %d)", who, x_type, y_type);
  return param_check(who, param_type, y_type);
}

// rows of `type` that eight-element vectors can read
inline bool ln_vec(const void* ptr, int64_t stride, int type) {
  const int size = type == SAF3R_FP32 ? 4 : 2;
  return (uintptr_t)ptr % 16 == 0 && stride * size % 16 == 0;
}

template <typename F>
inline int ln_types(int x_type, int y_type, int param_type, F f) {
  const bool p32 = param_type == SAF3R_FP32;
  auto rows = [&](auto tx, auto ty) { return p32 ? f(tx, ty, float()) : f(tx, ty, ty); };
  if (x_type == SAF3R_BF16) return rows(__bf16(), __bf16());
  if (x_type == SAF3R_FP16) return rows(_Float16(), _Float16());
  if (y_type == SAF3R_BF16) return rows(float(), __bf16());
  if (y_type == SAF3R_FP16) return rows(float(), _Float16());
  return f(float(), float(), float());
}

}  // namespace saf3r
