// The end of a branch and the norm before the next one, in one pass over the residual stream:
//   h = x + gate d,  d = branch keep / (1 - p),  y = (h - mean) rstd w + b
// h is rounded to the stream's type first: the norm reads the stream as every later reader does. Backward, from dh (of the
// stream) and dy (of the norm), with g = dy w, xh = (h - mean) rstd:
//   dH = dh + rstd (g - mean(g) - xh mean(g xh)),  dx = dH,  dbranch = gate keep / (1 - p) dH,
//   dgate = sum dH d,  dw = sum dy xh,  db = sum dy
// fp32, bf16 or fp16 stream, branch and y of one type; all arithmetic and every sum is fp32, each result is rounded once.
//
// Bound by HBM: forward reads x and branch and writes h and y, backward reads dh, dy, h and branch and writes dx and dbranch,
// each once (apart, with a product by the gate, a sum and a norm of their own, the same step moves 1.5 to 2 times the bytes).
// 87936 x 1024, fp32 stream, bf16 branch: 207 us forward (5.2 TB/s), 295 backward (5.5 TB/s) and 5 for the sums; 1041 x 1024 in
// bf16 4.8 forward.
// A row lies in the registers of the lanes that own it; the keep mask is computed again, never stored; the parameters'
// gradients go by partial rows, summed in a fixed order.
#include "dropout.h"
#include "norm_rows.h"

namespace saf3r {

struct RnParams {
  const void* x;  // forward: x; backward: dh (or null)
  const void* branch;
  const void* dy;
  const void* gate;
  const void* w;
  const void* b;
  void* h;
  void* y;  // forward: y; backward: dx
  void* dbranch;
  float* mean;
  float* rstd;
  float* part;  // backward: [work-groups][3][dim]: gate, weight, bias
  int64_t x_stride, branch_stride, dy_stride, h_stride, y_stride, dbranch_stride;
  int64_t rows, step;
  DropParams drop;
  int dim;
  float eps;
};

template <typename TX, typename TY, typename TP, bool SOME, int NV, int TPR>
__global__ void __launch_bounds__(256) residual_norm_fwd_kernel(const RnParams p) {
  __shared__ float lds[4];
  const int lane = tid_x() % TPR;
  constexpr int kRows = 256 / TPR;
  const int64_t row = (int64_t)bid_x() * kRows + tid_x() / TPR;
  const bool there = row < p.rows;
  const int64_t at = there ? row : 0;
  const TX* xp = (const TX*)p.x + at * p.x_stride;
  const TY* bp = (const TY*)p.branch + at * p.branch_stride;
  float x[NV][kVe], d[NV][kVe], w[NV][kVe], b[NV][kVe];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
    if (c < p.dim) {
      get<SOME, kVe>(xp + c, p.dim - c, x[j]);
      get<SOME, kVe>(bp + c, p.dim - c, d[j]);
      get_param<SOME, kVe, TP>(p.gate, c, p.dim - c, 1.f, b[j]);
    }
  }
  DropKey key{};
  if (p.drop.limit) key = drop_key(p.drop);
  TX* hp = (TX*)p.h + at * p.h_stride;
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
    if (c < p.dim) {
      if (p.drop.limit) drop8(key, p.drop.limit, p.drop.scale, (uint32_t)c >> 3, (uint64_t)row, d[j]);
#pragma unroll
      for (int e = 0; e < kVe; ++e) x[j][e] = (float)(TX)(x[j][e] + b[j][e] * d[j][e]);
      if (there) put<SOME, kVe>(hp + c, p.dim - c, x[j]);
#pragma unroll
      for (int e = 0; e < kVe; ++e) s += !SOME || c + e < p.dim ? x[j][e] : 0.f;
      // (the parameters are on their way while the statistics are summed)
      get_param<SOME, kVe, TP>(p.w, c, p.dim - c, 1.f, w[j]);
      get_param<SOME, kVe, TP>(p.b, c, p.dim - c, 0.f, b[j]);
    }
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

template <typename TX, typename TY, typename TP, bool SOME, int NV, int TPR>
__global__ void __launch_bounds__(256) residual_norm_bwd_kernel(const RnParams p) {
  constexpr int kRows = 256 / TPR;
  __shared__ float lds[4];
  __shared__ float sums[kRows > 1 ? 256 * kVe : 1];
  const int lane = tid_x() % TPR, slot = tid_x() / TPR;
  float w[NV][kVe], gate[NV][kVe], dw[NV][kVe], db[NV][kVe], dg[NV][kVe];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
#pragma unroll
    for (int e = 0; e < kVe; ++e) w[j][e] = gate[j][e] = dw[j][e] = db[j][e] = dg[j][e] = 0.f;
    if (c < p.dim) {
      get_param<SOME, kVe, TP>(p.w, c, p.dim - c, 1.f, w[j]);
      get_param<SOME, kVe, TP>(p.gate, c, p.dim - c, 1.f, gate[j]);
    }
  }
  DropKey key{};
  if (p.drop.limit) key = drop_key(p.drop);
  const float inv_n = 1.f / (float)p.dim;
  for (int64_t row0 = (int64_t)bid_x() * kRows; row0 < p.rows; row0 += p.step) {
    const int64_t row = row0 + slot;
    const bool there = row < p.rows;  // (a wave's rows end together with the loop: sums cross its lanes)
    const int64_t at = there ? row : 0;
    const float mean = there ? p.mean[at] : 0.f, rstd = there ? p.rstd[at] : 0.f;
    float x[NV][kVe], g[NV][kVe], up[NV][kVe], d[NV][kVe];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + lane) * kVe;
#pragma unroll
      for (int e = 0; e < kVe; ++e) x[j][e] = g[j][e] = up[j][e] = d[j][e] = 0.f;
      if (there && c < p.dim) {
        get<SOME, kVe>((const TX*)p.h + at * p.h_stride + c, p.dim - c, x[j]);
        get<SOME, kVe>((const TY*)p.dy + at * p.dy_stride + c, p.dim - c, g[j]);
        if (p.x) get<SOME, kVe>((const TX*)p.x + at * p.x_stride + c, p.dim - c, up[j]);
        if (p.branch) get<SOME, kVe>((const TY*)p.branch + at * p.branch_stride + c, p.dim - c, d[j]);
      }
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < kVe; ++e) {  // (behind the row's end g is zero)
        const float xh = (x[j][e] - mean) * rstd;
        dw[j][e] += g[j][e] * xh;
        db[j][e] += g[j][e];
        x[j][e] = xh;
        g[j][e] *= w[j][e];
        s1 += g[j][e];
        s2 += g[j][e] * xh;
      }
    const float m1 = row_sum<TPR>(s1, lds) * inv_n, m2 = row_sum<TPR>(s2, lds) * inv_n;
    if (there) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + lane) * kVe;
        if (c < p.dim) {
          float f[kVe];
#pragma unroll
          for (int e = 0; e < kVe; ++e) {
            g[j][e] = up[j][e] + rstd * (g[j][e] - m1 - x[j][e] * m2);
            f[e] = g[j][e];
          }
          put<SOME, kVe>((TX*)p.y + row * p.y_stride + c, p.dim - c, g[j]);
          if (p.drop.limit) drop8(key, p.drop.limit, p.drop.scale, (uint32_t)c >> 3, (uint64_t)row, f, d[j]);
#pragma unroll
          for (int e = 0; e < kVe; ++e) {
            dg[j][e] += f[e] * d[j][e];
            f[e] *= gate[j][e];
          }
          if (p.dbranch) put<SOME, kVe>((TY*)p.dbranch + row * p.dbranch_stride + c, p.dim - c, f);
        }
      }
    }
  }
  if (!p.part) return;
  float* part = p.part + (int64_t)bid_x() * 3 * p.dim;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * kVe;
    add_slots<kVe, TPR>(dg[j], sums);
    if (slot == 0 && c < p.dim) put<SOME, kVe>(part + c, p.dim - c, dg[j]);
    add_slots<kVe, TPR>(dw[j], sums);
    if (slot == 0 && c < p.dim) put<SOME, kVe>(part + p.dim + c, p.dim - c, dw[j]);
    add_slots<kVe, TPR>(db[j], sums);
    if (slot == 0 && c < p.dim) put<SOME, kVe>(part + 2 * p.dim + c, p.dim - c, db[j]);
  }
}

// Lanes of a row and vectors of a lane for a width: at most 16 values a lane up to rows of 4096, so that the backward pass
// keeps four rows, two parameters and three sums in registers.
template <typename F>
static int rn_dispatch(int dim, bool some, F f) {
  auto lanes = [&](auto part) {
    const int n = (dim + kVe - 1) / kVe;
    if (n <= 8) return f(part, Int<1>(), Int<8>());
    if (n <= 32) return f(part, Int<1>(), Int<32>());
    if (n <= 64) return f(part, Int<1>(), Int<64>());
    if (n <= 128) return f(part, Int<2>(), Int<64>());
    if (n <= 256) return f(part, Int<1>(), Int<256>());
    if (n <= 512) return f(part, Int<2>(), Int<256>());
    return f(part, Int<4>(), Int<256>());
  };
  return some ? lanes(std::true_type()) : lanes(std::false_type());
}

// Work-groups of the backward pass: two a compute unit, three where one has a row of at most 2048 in its registers at a time,
// with eight rows each at least, so that the partial rows they write are a small part of the rows they read. (10408 rows of 1536
// with dropout, with their sums: 51 us with two, 47 with three, 48 with four; 5000 of 4096: 79 with two, 94 with four.)
static int64_t rn_parts(int64_t rows, int dim) {
  return std::max<int64_t>(1, std::min<int64_t>(dim > 1024 && dim <= 2048 ? 768 : 512, rows / (dim <= 64 ? 32 : 8)));
}

}  // namespace saf3r

using namespace saf3r;

extern "C" int saf3r_residual_norm_fwd(const void* x, int64_t x_stride, int x_type, const void* branch,
                                       int64_t branch_stride, int y_type, int64_t rows, int dim, const void* gate,
                                       const void* weight, const void* bias, int param_type, int drop,
                                       const int64_t* state, float eps, void* h, int64_t h_stride, void* y,
                                       int64_t y_stride, float* mean, float* rstd, void* stream) {
  const char* who = "saf3r_residual_norm_fwd";
  if (int e = injected(who)) return e;
  if (int e = ln_check(who, rows, dim, x_type, y_type, param_type)) return e;
  if (!(eps >= 0.f && eps < 3.0e38f)) return fail(SAF3R_ERR_INVALID, "%s: eps must be finite and not negative", who);
  RnParams p{};
  if (int e = drop_check(who, drop, state, &p.drop)) return e;
  if (rows == 0) return SAF3R_OK;
  if (!x || !branch || !h || !y || !mean || !rstd) return fail(SAF3R_ERR_INVALID, "%s: null pointer", who);
  if (int e = row_check(who, x, x_stride, dim, x_type, false)) return e;
  if (int e = row_check(who, branch, branch_stride, dim, y_type, false)) return e;
  if (int e = row_check(who, h, h_stride, dim, x_type, true)) return e;
  if (int e = row_check(who, y, y_stride, dim, y_type, true)) return e;
  p.x = x;
  p.branch = branch;
  p.gate = gate;
  p.w = weight;
  p.b = bias;
  p.h = h;
  p.y = y;
  p.mean = mean;
  p.rstd = rstd;
  p.x_stride = x_stride;
  p.branch_stride = branch_stride;
  p.h_stride = h_stride;
  p.y_stride = y_stride;
  p.rows = rows;
  p.dim = dim;
  p.eps = eps;
  const bool vec = dim % 8 == 0 && ln_vec(x, x_stride, x_type) && ln_vec(branch, branch_stride, y_type) &&
                   ln_vec(h, h_stride, x_type) && ln_vec(y, y_stride, y_type) && ln_vec(gate, 0, param_type) &&
                   ln_vec(weight, 0, param_type) && ln_vec(bias, 0, param_type);
  return rn_dispatch(dim, !vec, [&](auto some, auto nv, auto tpr) {
    return ln_types(x_type, y_type, param_type, [&](auto tx, auto ty, auto tp) {
      constexpr int kTpr = decltype(tpr)::value;
      const int64_t grid = (rows + 256 / kTpr - 1) / (256 / kTpr);
      if (grid > 0xffffffffll / 256) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many rows for one launch", who);
      hipLaunchKernelGGL((residual_norm_fwd_kernel<decltype(tx), decltype(ty), decltype(tp), decltype(some)::value,
                                                   decltype(nv)::value, kTpr>),
                         dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, p);
      return check_launch(who);
    });
  });
}

extern "C" int64_t saf3r_residual_norm_bwd_workspace_bytes(int64_t rows, int dim) {
  const char* who = "saf3r_residual_norm_bwd_workspace_bytes";
  if (ln_check(who, rows, dim, SAF3R_FP32, SAF3R_FP32, SAF3R_FP32)) return -1;
  return rn_parts(rows, dim) * 3 * dim * 4;
}

extern "C" int saf3r_residual_norm_bwd(const void* dh, int64_t dh_stride, const void* dy, int64_t dy_stride, int y_type,
                                       const void* h, int64_t h_stride, int x_type, const void* branch,
                                       int64_t branch_stride, int64_t rows, int dim, const float* mean,
                                       const float* rstd, const void* gate, const void* weight, int param_type,
                                       int drop, const int64_t* state, void* dx, int64_t dx_stride, void* dbranch,
                                       int64_t dbranch_stride, void* dgate, void* dweight, void* dbias, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  const char* who = "saf3r_residual_norm_bwd";
  if (int e = injected(who)) return e;
  if (int e = ln_check(who, rows, dim, x_type, y_type, param_type)) return e;
  RnParams p{};
  if (int e = drop_check(who, drop, state, &p.drop)) return e;
  const bool params = dgate || dweight || dbias;
  if (rows > 0) {
    if (!dy || !h || !mean || !rstd || !dx) return fail(SAF3R_ERR_INVALID, "%s: null pointer", who);
    if (dgate && !branch) return fail(SAF3R_ERR_INVALID, "%s: the gate's gradient needs the branch", who);
    if (int e = row_check(who, dy, dy_stride, dim, y_type, false)) return e;
    if (int e = row_check(who, h, h_stride, dim, x_type, false)) return e;
    if (int e = row_check(who, dx, dx_stride, dim, x_type, true)) return e;
    if (dh)
      if (int e = row_check(who, dh, dh_stride, dim, x_type, false)) return e;
    if (dgate)
      if (int e = row_check(who, branch, branch_stride, dim, y_type, false)) return e;
    if (dbranch)
      if (int e = row_check(who, dbranch, dbranch_stride, dim, y_type, true)) return e;
  }
  const int64_t need = params ? saf3r_residual_norm_bwd_workspace_bytes(rows, dim) : 0;
  if (workspace_bytes < need || (need > 0 && (!workspace || (uintptr_t)workspace % 16)))
    return fail(SAF3R_ERR_INVALID, "%s: workspace of %lld bytes: %lld, 16-byte aligned, are needed", who,
                (long long)workspace_bytes, (long long)need);
  p.x = dh;
  p.dy = dy;
  p.branch = dgate ? branch : nullptr;
  p.gate = gate;
  p.w = weight;
  p.h = const_cast<void*>(h);
  p.y = dx;
  p.dbranch = dbranch;
  p.mean = const_cast<float*>(mean);
  p.rstd = const_cast<float*>(rstd);
  p.part = params ? (float*)workspace : nullptr;
  p.x_stride = dh_stride;
  p.dy_stride = dy_stride;
  p.branch_stride = branch_stride;
  p.h_stride = h_stride;
  p.y_stride = dx_stride;
  p.dbranch_stride = dbranch_stride;
  p.rows = rows;
  p.dim = dim;
  const bool vec = dim % 8 == 0 && (!dh || ln_vec(dh, dh_stride, x_type)) && ln_vec(dy, dy_stride, y_type) &&
                   ln_vec(h, h_stride, x_type) && (!dgate || ln_vec(branch, branch_stride, y_type)) &&
                   ln_vec(dx, dx_stride, x_type) && (!dbranch || ln_vec(dbranch, dbranch_stride, y_type)) &&
                   ln_vec(gate, 0, param_type) && ln_vec(weight, 0, param_type);
  int64_t parts = 0;
  int rc = SAF3R_OK;
  if (rows > 0)
    rc = rn_dispatch(dim, !vec, [&](auto some, auto nv, auto tpr) {
      return ln_types(x_type, y_type, param_type, [&](auto tx, auto ty, auto tp) {
        constexpr int kTpr = decltype(tpr)::value;
        parts = rn_parts(rows, dim);
        p.step = parts * (256 / kTpr);
        hipLaunchKernelGGL((residual_norm_bwd_kernel<decltype(tx), decltype(ty), decltype(tp), decltype(some)::value,
                                                     decltype(nv)::value, kTpr>),
                           dim3((uint32_t)parts), dim3(256), 0, (hipStream_t)stream, p);
        return check_launch(who);
      });
    });
  if (rc != SAF3R_OK || !params) return rc;
  return sum_parts3(who, (const float*)workspace, parts, dim, dgate, dweight, dbias, param_type, (hipStream_t)stream);
}
