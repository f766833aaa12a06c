// Products with an epilogue (linear layers): element types, activations and the epilogue of eight columns of a row, shared by
// the tile kernel, the kernel for few rows, the join of split reductions and the gradient before the products.
#pragma once

#include "dropout.h"
#include "row_ops.h"

namespace saf3r {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Half;  // a 16-bit type's vector and matrix products
template <>
struct Half<__bf16> {
  typedef bf16x8 vec8;
  static __device__ __forceinline__ f32x16 mma32(vec8 a, vec8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16(vec8 a, vec8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Half<_Float16> {
  typedef f16x8 vec8;
  static __device__ __forceinline__ f32x16 mma32(vec8 a, vec8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16(vec8 a, vec8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Both GELUs are z times a share s(z) in (0, 1); the derivative is s + z s'.
//   exact: s is the normal distribution function by its complement, q = 1 - s(|z|) = t (c1 + t (c2 + ...)) exp(-z^2 / 2) / 2,
//   t = 1 / (1 + 0.3275911 |z| / sqrt 2) (Abramowitz and Stegun, 7.1.26: within 7.5e-8), so that z s = max(z, 0) - |z| q; s' is
//   the density, whose exponential is the same. A library erf costs about three times as many instructions.
//   tanh form: s = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (z + 0.044715 z^3); s' = 2 s (1 - s) u'.
// Behind |z| = 15 s is 0 or 1 in fp32: z is held there in its products with q, s and s' (an infinity times zero would be a NaN).
// A NaN stays one.
__device__ __forceinline__ float gelu_tail(float z, float* e) {  // q
  const float t = __builtin_amdgcn_rcpf(1.f + 0.23164189f * fabsf(z));
  *e = __builtin_amdgcn_exp2f(-0.72134752f * z * z);
  float q = t * (1.061405429f * 0.5f) + (-1.453152027f * 0.5f);
  q = q * t + 1.421413741f * 0.5f;
  q = q * t + -0.284496736f * 0.5f;
  q = q * t + 0.254829592f * 0.5f;
  return q * t * *e;
}

__device__ __forceinline__ float tanh_share(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-2.3022082f * z * (1.f + 0.044715f * z * z)));
}

// z within [low, high], one instruction (fminf makes a NaN quiet first: sums over rows of the exact GELU's gradient, 87936 x 4096
// in bf16 without a dz, 300 us in place of 291 to 297; bound by HBM with a dz, the same). A NaN's is some number.
__device__ __forceinline__ float clamp(float z, float low, float high) { return __builtin_amdgcn_fmed3f(z, low, high); }

__device__ __forceinline__ float gelu_of(float z, float q) { return fmaxf(z, 0.f) - clamp(fabsf(z), 0.f, 15.f) * q; }

__device__ __forceinline__ float act_value(int act, float z) {
  if (act == SAF3R_NO_ACTIVATION) return z;
  if (act == SAF3R_GELU) {
    float e;
    const float q = gelu_tail(z, &e);
    return gelu_of(z, q);
  }
  return fmaxf(z, -15.f) * tanh_share(z);
}

// act(z) and act'(z)
__device__ __forceinline__ float act_slope(int act, float z, float* value) {
  if (act == SAF3R_NO_ACTIVATION) {
    *value = z;
    return 1.f;
  }
  const float low = fmaxf(z, -15.f), b = clamp(z, -15.f, 15.f);
  if (act == SAF3R_GELU) {
    float e;
    const float q = gelu_tail(z, &e);
    *value = gelu_of(z, q);
    return (z < 0.f ? q : 1.f - q) + b * (0.39894228f * e);
  }
  const float s = tanh_share(z);
  *value = low * s;
  return s + b * (s * (1.f - s) * (1.5957691f * (1.f + 0.134145f * b * b)));
}

// y = res + gate drop(act(z + bias)); kept = z + bias. Rows of n columns; `vec`: every row can be read and written in
// vectors of eight (n % 8 == 0, 16-byte aligned).
struct EpiParams {
  const void* bias;
  const void* gate;
  const void* res;  // of y's type
  void* y;
  void* kept;  // of the operands' type
  int64_t ld_res, ld_y, ld_kept;
  DropParams drop;
  int act, n;
  bool param32, y32, vec;
};

template <typename T>
__device__ __forceinline__ void epi_load(const void* p, bool f32, bool vec, int64_t at, int cnt, float (&x)[8]) {
  if (f32) {
    if (vec)
      load_vec<8>((const float*)p + at, x);
    else
      load_some<8>((const float*)p + at, cnt, x);
  } else {
    if (vec)
      load_vec<8>((const T*)p + at, x);
    else
      load_some<8>((const T*)p + at, cnt, x);
  }
}

template <typename T>
__device__ __forceinline__ void epi_store(void* p, bool f32, bool vec, int64_t at, int cnt, const float (&x)[8]) {
  if (f32) {
    if (vec)
      store_vec<8>((float*)p + at, x);
    else
      store_some<8>((float*)p + at, cnt, x);
  } else {
    if (vec)
      store_vec<8>((T*)p + at, x);
    else
      store_some<8>((T*)p + at, cnt, x);
  }
}

// The parameters of columns col .. col + 7 (col % 8 == 0, col < n).
template <typename T>
struct EpiCols {
  float bias[8], gate[8];
  __device__ __forceinline__ void load(const EpiParams& e, int col) {
    if (e.bias) epi_load<T>(e.bias, e.param32, e.vec, col, e.n - col, bias);
    if (e.gate) epi_load<T>(e.gate, e.param32, e.vec, col, e.n - col, gate);
  }
};

// The elements at which eight columns of a row start.
struct EpiPlace {
  int64_t res, y, kept;
  __device__ __forceinline__ void init(const EpiParams& e, int64_t row, int col) {
    res = row * e.ld_res + col;
    y = row * e.ld_y + col;
    kept = row * e.ld_kept + col;
  }
  __device__ __forceinline__ void down(const EpiParams& e, int rows) {
    res += rows * e.ld_res;
    y += rows * e.ld_y;
    kept += rows * e.ld_kept;
  }
};

// The epilogue of columns col .. col + 7 of a row that is there; r: the residual's.
template <typename T>
__device__ __forceinline__ void epilogue8(const EpiParams& e, const DropKey& key, const EpiCols<T>& c, const EpiPlace& at,
                                          int64_t row, int col, const float (&r)[8], float (&x)[8]) {
  const int cnt = e.n - col;
  if (e.bias) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] += c.bias[j];
  }
  if (e.kept) epi_store<T>(e.kept, false, e.vec, at.kept, cnt, x);
  if (e.act != SAF3R_NO_ACTIVATION) {
    if (e.act == SAF3R_GELU) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = act_value(SAF3R_GELU, x[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = act_value(SAF3R_GELU_TANH, x[j]);
    }
  }
  if (e.drop.limit) drop8(key, e.drop.limit, e.drop.scale, (uint32_t)col >> 3, (uint64_t)row, x);
  if (e.gate) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= c.gate[j];
  }
  if (e.res) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] += r[j];
  }
  epi_store<T>(e.y, e.y32, e.vec, at.y, cnt, x);
}

template <typename T>
__device__ __forceinline__ void epilogue8(const EpiParams& e, const DropKey& key, int64_t row, int col, float (&x)[8]) {
  EpiCols<T> c;
  EpiPlace at;
  float r[8];
  c.load(e, col);
  at.init(e, row, col);
  if (e.res) epi_load<T>(e.res, e.y32, e.vec, at.res, e.n - col, r);
  epilogue8<T>(e, key, c, at, row, col, r, x);
}

// First step of a backward pass (linear_grad.hip): dz = dy gate keep/(1-p) act'(kept), rounded to the operands' type, and the
// partial sums over rows of dy drop(act(kept)) (the gate's gradient) and dz (the bias's).
struct LinearGradParams {
  const void* dy;
  const void* kept;
  const void* gate;
  void* dz;     // null: sums only; columns n .. n8 - 1 are zeros
  float* part;  // null: no sums; [parts][2][n], the gate's where it is asked for
  int64_t ld_dy, ld_kept, ld_dz, rows, part_rows;
  void* dgate;  // where one work-group has all rows (direct): the sums themselves, each may be null
  void* dbias;
  DropParams drop;
  int act, n;
  bool param32, direct;
};
int64_t linear_grad_parts(int64_t rows, int n);
int linear_grad(const char* who, const LinearGradParams& p, int type, bool dy32, bool vec, bool dgate, int64_t parts,
                hipStream_t stream);

}  // namespace saf3r
