// Dropout by itself: y = x keep / (1 - p), the mask of dropout.h. Its gradient is the same function of dy.
//
// Bound by HBM: x is read and y written once, and no mask (87936 x 1024 in bf16: 61 to 67 us, 5.4 to 5.9 TB/s). A block of the
// generator (ten rounds of two 32-bit products, at a quarter of the vector rate) serves a vector of eight elements.
#include "dropout.h"
#include "row_ops.h"

namespace saf3r {

struct DropoutParams {
  const void* x;
  void* y;
  int64_t x_stride, y_stride, count;  // count: vectors of all rows
  int64_t step_rows, groups;          // a step of the grid: step_rows rows and step_groups vectors
  int64_t step_groups;
  int dim;
  DropParams drop;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutParams p) {
  int64_t at = (int64_t)bid_x() * 256 + tid_x();
  if (at >= p.count) return;
  const DropKey key = drop_key(p.drop);
  int64_t row = at / p.groups, group = at - row * p.groups;
  const int64_t step = p.step_rows * p.groups + p.step_groups;
  for (; at < p.count; at += step) {
    const int64_t c = group * 8;
    const int cnt = (int)(p.dim - c);
    float x[8];
    if constexpr (VEC)
      load_vec<8>((const T*)p.x + row * p.x_stride + c, x);
    else
      load_some<8>((const T*)p.x + row * p.x_stride + c, cnt, x);
    drop8(key, p.drop.limit, p.drop.scale, (uint32_t)group, (uint64_t)row, x);
    if constexpr (VEC)
      store_vec<8>((T*)p.y + row * p.y_stride + c, x);
    else
      store_some<8>((T*)p.y + row * p.y_stride + c, cnt, x);
    row += p.step_rows;
    group += p.step_groups;
    if (group >= p.groups) {
      group -= p.groups;
      ++row;
    }
  }
}

}  // namespace saf3r

using namespace saf3r;

extern "C" int saf3r_dropout(const void* x, int64_t x_stride, int type, int64_t rows, int dim, int drop,
                             const int64_t* state, void* y, int64_t y_stride, void* stream) {
  const char* who = "saf3r_dropout";
  if (int e = injected(who)) return e;
  if (rows < 0 || dim <= 0)
    return fail(SAF3R_ERR_INVALID, "%s: invalid sizes: %lld rows of %d", who, (long long)rows, dim);
  if (rows > (int64_t)1 << 38) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many rows", who);
  if (type < SAF3R_FP32 || type > SAF3R_FP16) return fail(SAF3R_ERR_INVALID, "%s: unknown element type %d", who, type);
  DropoutParams p{};
  if (int e = drop_check(who, drop, state, &p.drop)) return e;
  if (!state || (uintptr_t)state % 8) return fail(SAF3R_ERR_INVALID, "%s: dropout needs its state (two int64)", who);
  p.drop.state = state;
  if (rows == 0) return SAF3R_OK;
  if (!x || !y) return fail(SAF3R_ERR_INVALID, "%s: null pointer", who);
  if (int e = row_check(who, x, x_stride, dim, type, false)) return e;
  if (int e = row_check(who, y, y_stride, dim, type, true)) return e;
  const int size = type == SAF3R_FP32 ? 4 : 2;
  auto aligned = [&](const void* q, int64_t stride) { return (uintptr_t)q % 16 == 0 && stride * size % 16 == 0; };
  const bool vec = dim % 8 == 0 && aligned(x, x_stride) && aligned(y, y_stride);
  p.x = x;
  p.y = y;
  p.x_stride = x_stride;
  p.y_stride = y_stride;
  p.dim = dim;
  p.groups = ((int64_t)dim + 7) / 8;
  p.count = rows * p.groups;
  // eight work-groups a compute unit
  const int64_t grid = std::min<int64_t>(2048, (p.count + 255) / 256);
  p.step_rows = grid * 256 / p.groups;
  p.step_groups = grid * 256 % p.groups;
  auto go = [&](auto t) {
    if (vec)
      hipLaunchKernelGGL((dropout_kernel<decltype(t), true>), dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, p);
    else
      hipLaunchKernelGGL((dropout_kernel<decltype(t), false>), dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, p);
    return check_launch(who);
  };
  return type == SAF3R_FP32 ? go(float()) : type == SAF3R_BF16 ? go(__bf16()) : go(_Float16());
}
