// LayerNorm over rows of any width up to 8192 with its backward pass: y = (x - mean) rstd w + b, and from dy
//   g = dy w,  xh = (x - mean) rstd,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum dy xh,  db = sum dy.
// fp32, bf16 or fp16 rows; all arithmetic and every sum is fp32, each result is rounded once.
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx, each once. A row lies in the
// registers of the lanes that own it (a part of a wave, a wave, or a work-group for wide rows), so the mean, the
// centred squares and the result need one read. The parameters' gradients are sums over rows: each lane keeps the
// sums of its columns in registers while its work-group walks its rows, one work-group writes one partial row, and a
// second kernel adds the partial rows in a fixed order (no atomics: equal inputs give equal bits). A lane reads eight
// elements at a time, also where a row is not aligned to that or ends inside them.
// Measured: 87936 rows of 1024, fp32 to bf16: forward 94 us for 540 MB (5.7 TB/s), backward 156 us for 900 MB (5.8
// TB/s) and 5 us for the sums (a 4 GiB copy, read and written: 4.8 TB/s); 4097 rows of 1027, fp32: 10 and 15 us (16 and 28
// with single elements).
#include "norm_rows.h"

namespace saf3r {

struct LnParams {
  const void* x;
  const void* dy;
  void* y;  // forward: y; backward: dx
  const void* w;
  const void* b;
  float* mean;
  float* rstd;
  float* part;  // backward: [work-groups][2][dim]
  int64_t x_stride, dy_stride, y_stride;
  int64_t rows;
  int64_t step;  // backward: rows of all work-groups' steps (the grid's size comes from host memory in a kernel: slow)
  int dim;
  float eps;
};

template <typename TX, typename TY, typename TP, bool SOME, int NV, int TPR>
__global__ void __launch_bounds__(256) layer_norm_fwd_kernel(const LnParams p) {
  __shared__ float lds[4];
  const int lane = tid_x() % TPR;
  constexpr int kRows = 256 / TPR;
  const int64_t row = (int64_t)bid_x() * kRows + tid_x() / TPR;
  const bool there = row < p.rows;
  const TX* xp = (const TX*)p.x + (there ? row : 0) * p.x_stride;
  float x[NV][kVe], w[NV][kVe], b[NV][kVe];
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
    if (c < p.dim) get<SOME, kVe>(xp + c, p.dim - c, x[j]);
  }
  // (the parameters are on their way while the statistics are summed)
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
    if (c < p.dim) {
      get_param<SOME, kVe, TP>(p.w, c, p.dim - c, 1.f, w[j]);
      get_param<SOME, kVe, TP>(p.b, c, p.dim - c, 0.f, b[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if ((j * TPR + lane) * kVe < p.dim) {
#pragma unroll
      for (int e = 0; e < kVe; ++e) s += x[j][e];
    }
  const float inv_n = 1.f / (float)p.dim;
  const float mean = row_sum<TPR>(s, lds) * inv_n;
  s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
    if (c < p.dim) {
#pragma unroll
      for (int e = 0; e < kVe; ++e) {
        x[j][e] -= mean;
        s += !SOME || c + e < p.dim ? x[j][e] * x[j][e] : 0.f;
      }
    }
  }
  const float rstd = inv_sqrt(row_sum<TPR>(s, lds) * inv_n + p.eps);
  if (!there) return;
  TY* yp = (TY*)p.y + row * p.y_stride;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
    if (c < p.dim) {
#pragma unroll
      for (int e = 0; e < kVe; ++e) x[j][e] = x[j][e] * rstd * w[j][e] + b[j][e];
      put<SOME, kVe>(yp + c, p.dim - c, x[j]);
    }
  }
  if (lane == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
}

template <typename TX, typename TY, typename TP, bool SOME, int NV, int TPR, bool PARAMS>
__global__ void __launch_bounds__(256) layer_norm_bwd_kernel(const LnParams p) {
  constexpr int kRows = 256 / TPR;
  __shared__ float lds[4];
  __shared__ float sums[PARAMS && kRows > 1 ? 256 * kVe : 1];
  const int lane = tid_x() % TPR, slot = tid_x() / TPR;
  float w[NV][kVe], dw[PARAMS ? NV : 1][kVe], db[PARAMS ? NV : 1][kVe];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
#pragma unroll
    for (int e = 0; e < kVe; ++e) w[j][e] = 0.f;
    if (c < p.dim) get_param<SOME, kVe, TP>(p.w, c, p.dim - c, 1.f, w[j]);
  }
  if constexpr (PARAMS) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < kVe; ++e) dw[j][e] = db[j][e] = 0.f;
  }
  const float inv_n = 1.f / (float)p.dim;
  for (int64_t row0 = (int64_t)bid_x() * kRows; row0 < p.rows; row0 += p.step) {
    const int64_t row = row0 + slot;
    const bool there = row < p.rows;  // (a wave's rows end together with the loop: sums cross its lanes)
    const TX* xp = (const TX*)p.x + (there ? row : 0) * p.x_stride;
    const TY* gp = (const TY*)p.dy + (there ? row : 0) * p.dy_stride;
    const float mean = there ? p.mean[row] : 0.f, rstd = there ? p.rstd[row] : 0.f;
    float x[NV][kVe], g[NV][kVe];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + lane) * kVe;
#pragma unroll
      for (int e = 0; e < kVe; ++e) x[j][e] = g[j][e] = 0.f;
      if (there && c < p.dim) {
        get<SOME, kVe>(xp + c, p.dim - c, x[j]);
        get<SOME, kVe>(gp + c, p.dim - c, g[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < kVe; ++e) {  // (behind the row's end g is zero)
        const float xh = (x[j][e] - mean) * rstd;
        if constexpr (PARAMS) {
          dw[j][e] += g[j][e] * xh;
          db[j][e] += g[j][e];
        }
        x[j][e] = xh;
        g[j][e] *= w[j][e];
        s1 += g[j][e];
        s2 += g[j][e] * xh;
      }
    const float m1 = row_sum<TPR>(s1, lds) * inv_n, m2 = row_sum<TPR>(s2, lds) * inv_n;
    if (there) {
      TX* op = (TX*)p.y + row * p.y_stride;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + lane) * kVe;
        if (c < p.dim) {
#pragma unroll
          for (int e = 0; e < kVe; ++e) x[j][e] = rstd * (g[j][e] - m1 - x[j][e] * m2);
          put<SOME, kVe>(op + c, p.dim - c, x[j]);
        }
      }
    }
  }
  if constexpr (PARAMS) {
    float* part = p.part + (int64_t)bid_x() * 2 * p.dim;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + lane) * kVe;
      add_slots<kVe, TPR>(dw[j], sums);
      if (slot == 0 && c < p.dim) put<SOME, kVe>(part + c, p.dim - c, dw[j]);
      add_slots<kVe, TPR>(db[j], sums);
      if (slot == 0 && c < p.dim) put<SOME, kVe>(part + p.dim + c, p.dim - c, db[j]);
    }
  }
}

// Lanes of a row and vectors of a lane for a width: at most 32 values a lane, so that the backward pass keeps x, dy, w
// and both sums in registers.
template <typename F>
static int ln_dispatch(int dim, bool some, F f) {
  auto lanes = [&](auto part) {
    const int n = (dim + kVe - 1) / kVe;
    if (n <= 8) return f(part, Int<1>(), Int<8>());
    if (n <= 16) return f(part, Int<1>(), Int<16>());
    if (n <= 32) return f(part, Int<1>(), Int<32>());
    if (n <= 64) return f(part, Int<1>(), Int<64>());
    if (n <= 128) return f(part, Int<2>(), Int<64>());
    if (n <= 192) return f(part, Int<3>(), Int<64>());
    if (n <= 256) return f(part, Int<4>(), Int<64>());
    if (n <= 512) return f(part, Int<2>(), Int<256>());
    return f(part, Int<4>(), Int<256>());
  };
  return some ? lanes(std::true_type()) : lanes(std::false_type());
}

// Work-groups of the backward pass: two a compute unit, which all run at once at any width, with at least eight rows each,
// so that the partial rows they write are a small part of the rows they read. (Backward and sums, 87936 rows of 1024 and
// 10408 of 1536: 161 and 29 us; with one a compute unit 189 and 41, with three 167 and 28, with four 169 and 32.)
static int64_t ln_parts(int64_t rows, int rows_per_step) {
  return std::max<int64_t>(1, std::min<int64_t>(512, rows / (rows_per_step > 8 ? rows_per_step : 8)));
}

}  // namespace saf3r

using namespace saf3r;

extern "C" int saf3r_layer_norm_fwd(const void* x, int64_t x_stride, int x_type, int64_t rows, int dim,
                                    const void* weight, const void* bias, int param_type, float eps, void* y,
                                    int64_t y_stride, int y_type, float* mean, float* rstd, void* stream) {
  const char* who = "saf3r_layer_norm_fwd";
  if (int e = injected(who)) return e;
  if (int e = ln_check(who, rows, dim, x_type, y_type, param_type)) return e;
  if (!(eps >= 0.f && eps < 3.0e38f)) return fail(SAF3R_ERR_INVALID, "%s: eps must be finite and not negative", who);
  if (rows == 0) return SAF3R_OK;
  if (!x || !y || !mean || !rstd) return fail(SAF3R_ERR_INVALID, "%s: null pointer", who);
  if (int e = row_check(who, x, x_stride, dim, x_type, false)) return e;
  if (int e = row_check(who, y, y_stride, dim, y_type, true)) return e;
  LnParams p{};
  p.x = x;
  p.y = y;
  p.w = weight;
  p.b = bias;
  p.mean = mean;
  p.rstd = rstd;
  p.x_stride = x_stride;
  p.y_stride = y_stride;
  p.rows = rows;
  p.dim = dim;
  p.eps = eps;
  const bool vec = dim % 8 == 0 && ln_vec(x, x_stride, x_type) && ln_vec(y, y_stride, y_type) &&
                   ln_vec(weight, 0, param_type) && ln_vec(bias, 0, param_type);
  return ln_dispatch(dim, !vec, [&](auto some, auto nv, auto tpr) {
    return ln_types(x_type, y_type, param_type, [&](auto tx, auto ty, auto tp) {
      constexpr int kTpr = decltype(tpr)::value;
      const int64_t grid = (rows + 256 / kTpr - 1) / (256 / kTpr);
      // (a launch counts its threads in 32 bits)
      if (grid > 0xffffffffll / 256) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many rows for one launch", who);
      hipLaunchKernelGGL(
          (layer_norm_fwd_kernel<decltype(tx), decltype(ty), decltype(tp), decltype(some)::value, decltype(nv)::value,
                                 kTpr>),
          dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, p);
      return check_launch(who);
    });
  });
}

extern "C" int64_t saf3r_layer_norm_bwd_workspace_bytes(int64_t rows, int dim) {
  const char* who = "saf3r_layer_norm_bwd_workspace_bytes";
  if (ln_check(who, rows, dim, SAF3R_FP32, SAF3R_FP32, SAF3R_FP32)) return -1;
  return ln_parts(rows, 1) * 2 * dim * 4;
}

extern "C" int saf3r_layer_norm_bwd(const void* dy, int64_t dy_stride, int y_type, const void* x, int64_t x_stride,
                                    int x_type, int64_t rows, int dim, const float* mean, const float* rstd,
                                    const void* weight, int param_type, void* dx, int64_t dx_stride, void* dweight,
                                    void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "saf3r_layer_norm_bwd";
  if (int e = injected(who)) return e;
  if (int e = ln_check(who, rows, dim, x_type, y_type, param_type)) return e;
  const bool params = dweight || dbias;
  if (rows > 0) {
    if (!dy || !x || !mean || !rstd || !dx) return fail(SAF3R_ERR_INVALID, "%s: null pointer", who);
    if (int e = row_check(who, x, x_stride, dim, x_type, false)) return e;
    if (int e = row_check(who, dx, dx_stride, dim, x_type, true)) return e;
    if (int e = row_check(who, dy, dy_stride, dim, y_type, false)) return e;
  }
  const int64_t need = params ? saf3r_layer_norm_bwd_workspace_bytes(rows, dim) : 0;
  if (workspace_bytes < need || (need > 0 && (!workspace || (uintptr_t)workspace % 16)))
    return fail(SAF3R_ERR_INVALID, "%s: workspace of %lld bytes: %lld, 16-byte aligned, are needed", who,
                (long long)workspace_bytes, (long long)need);
  LnParams p{};
  p.x = x;
  p.dy = dy;
  p.y = dx;
  p.w = weight;
  p.mean = const_cast<float*>(mean);
  p.rstd = const_cast<float*>(rstd);
  p.part = (float*)workspace;
  p.x_stride = x_stride;
  p.dy_stride = dy_stride;
  p.y_stride = dx_stride;
  p.rows = rows;
  p.dim = dim;
  const bool vec = dim % 8 == 0 && ln_vec(x, x_stride, x_type) && ln_vec(dx, dx_stride, x_type) &&
                   ln_vec(dy, dy_stride, y_type) && ln_vec(weight, 0, param_type);
  int64_t parts = 0;
  int rc = SAF3R_OK;
  if (rows > 0)
    rc = ln_dispatch(dim, !vec, [&](auto some, auto nv, auto tpr) {
      return ln_types(x_type, y_type, param_type, [&](auto tx, auto ty, auto tp) {
        constexpr int kTpr = decltype(tpr)::value;
        parts = ln_parts(rows, 256 / kTpr);
        p.step = parts * (256 / kTpr);
        if (params)
          hipLaunchKernelGGL((layer_norm_bwd_kernel<decltype(tx), decltype(ty), decltype(tp), decltype(some)::value,
                                                    decltype(nv)::value, kTpr, true>),
                             dim3((uint32_t)parts), dim3(256), 0, (hipStream_t)stream, p);
        else
          hipLaunchKernelGGL((layer_norm_bwd_kernel<decltype(tx), decltype(ty), decltype(tp), decltype(some)::value,
                                                    decltype(nv)::value, kTpr, false>),
                             dim3((uint32_t)parts), dim3(256), 0, (hipStream_t)stream, p);
        return check_launch(who);
      });
    });
  if (rc != SAF3R_OK || !params) return rc;
  return sum_parts(who, (const float*)workspace, parts, dim, dweight, dbias, param_type, (hipStream_t)stream);
}
