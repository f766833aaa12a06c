// Second step of the parameters' gradients: adds the partial rows that the work-groups of a row kernel wrote.
#include "row_ops.h"

namespace saf3r {

struct PartParams {
  const float* part;  // [parts][2][n]
  int64_t parts;
  int n;
  void* out[2];
  int type;
};

// A work-group adds 32 columns: eight slices of the partial rows side by side, then the slices in order. Small next to
// the pass that wrote the partial rows (8 MB of them at most for 1024 columns).
__global__ void __launch_bounds__(256) sum_parts_kernel(const PartParams p) {
  __shared__ float lds[8][32];
  const int col = tid_x() & 31, slice = tid_x() >> 5;
  const int64_t c = (int64_t)bid_x() * 32 + col;  // column of [2][n]
  float s = 0.f;
  if (c < 2 * (int64_t)p.n)
    for (int64_t k = slice; k < p.parts; k += 8) s += p.part[k * 2 * p.n + c];
  lds[slice][col] = s;
  __syncthreads();
  if (slice || c >= 2 * (int64_t)p.n) return;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += lds[k][col];
  const int which = c >= p.n;
  void* out = p.out[which];
  if (!out) return;
  const int64_t at = c - (which ? p.n : 0);
  if (p.type == SAF3R_FP32)
    ((float*)out)[at] = s;
  else if (p.type == SAF3R_BF16)
    ((__bf16*)out)[at] = (__bf16)s;
  else
    ((_Float16*)out)[at] = (_Float16)s;
}

int sum_parts(const char* who, const float* part, int64_t parts, int n, void* dweight, void* dbias, int type,
              hipStream_t stream) {
  const PartParams p = {part, parts, n, {dweight, dbias}, type};
  hipLaunchKernelGGL(sum_parts_kernel, dim3((uint32_t)((2 * (int64_t)n + 31) / 32)), dim3(256), 0, stream, p);
  return check_launch(who);
}

}  // namespace saf3r
