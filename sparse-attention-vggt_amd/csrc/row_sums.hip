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

// A work-group of 1024 adds 16 columns: 64 slices of the partial rows side by side, four loads in flight each, then the
// slices in order. One wave reads four lines of 64 bytes; 128 work-groups for 1024 columns.
constexpr int kSumCols = 16, kSumSlices = 64;

__global__ void __launch_bounds__(kSumCols* kSumSlices) sum_parts_kernel(const PartParams p) {
  __shared__ float lds[kSumSlices][kSumCols + 1];
  const int col = tid_x() % kSumCols, slice = tid_x() / kSumCols;
  const int64_t n2 = 2 * (int64_t)p.n, c = (int64_t)bid_x() * kSumCols + col;  // column of [2][n]
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < n2) {
    const float* at = p.part + c;
    int64_t k = slice;
    for (; k + 3 * kSumSlices < p.parts; k += 4 * kSumSlices)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += at[(k + j * kSumSlices) * n2];
    for (; k < p.parts; k += kSumSlices) s[0] += at[k * n2];
  }
  lds[slice][col] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  // four threads a column, then one
  if (slice < 4) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kSumSlices / 4; ++k) t += lds[slice * (kSumSlices / 4) + k][col];
    s[0] = t;
  }
  __syncthreads();
  if (slice < 4) lds[slice][col] = s[0];
  __syncthreads();
  if (slice || c >= n2) return;
  s[0] = (lds[0][col] + lds[1][col]) + (lds[2][col] + lds[3][col]);
  const int which = c >= p.n;
  void* out = p.out[which];
  if (!out) return;
  const int64_t at = c - (which ? p.n : 0);
  if (p.type == SAF3R_FP32)
    ((float*)out)[at] = s[0];
  else if (p.type == SAF3R_BF16)
    ((__bf16*)out)[at] = (__bf16)s[0];
  else
    ((_Float16*)out)[at] = (_Float16)s[0];
}

int sum_parts(const char* who, const float* part, int64_t parts, int n, void* dweight, void* dbias, int type,
              hipStream_t stream) {
  const PartParams p = {part, parts, n, {dweight, dbias}, type};
  hipLaunchKernelGGL(sum_parts_kernel, dim3((uint32_t)((2 * (int64_t)n + kSumCols - 1) / kSumCols)),
                     dim3(kSumCols * kSumSlices), 0, stream, p);
  return check_launch(who);
}

}  // namespace saf3r
