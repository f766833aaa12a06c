// Before the products of a linear layer's backward pass: the gradient behind the epilogue, and its sums over rows.
//   dz = dy gate keep/(1-p) act'(kept),  dbias = sum dz,  dgate = sum dy keep/(1-p) act(kept)
// dz is rounded to the operands' type, which the matrix products read; the sums take it unrounded. kept is of that type too, so
// that act and act' are those of a z that is off by half a step: in fp32 it would be written and read at twice the bytes
// (87936 x 4096: 720 MB more in either pass, about 150 us each). Relative distance from 64 bits, bf16, 1041 x 1024 to 4096
// with GELU: dx 2.41e-3, dW 2.29e-3, nearly all of it dz's rounding and their own; 1.66e-3 with fp32 throughout. Products of
// a dz in two parts would take dz's away for the time of the products again.
//
// Bound by HBM: dy and kept are read and dz is written once (87936 x 4096 with GELU and its sums: 460 to 475 us, 4.6 TB/s). A
// work-group of 256 owns 256 columns of a range of rows, eight rows at a time; a lane keeps the sums of its eight columns,
// and every work-group writes one partial row (summed in a fixed order by sum_parts: equal inputs give equal bits).
#include "linear.h"

namespace saf3r {

template <typename T, typename TY, bool VEC, bool DGATE>
__global__ void __launch_bounds__(256) linear_grad_kernel(const LinearGradParams p) {
  __shared__ float lds[256 * 8];
  const int lane = tid_x() & 31, slot = tid_x() >> 5;
  const int col = (bid_x() * 32 + lane) * 8, cnt = p.n - col;
  const int64_t begin = bid_y() * p.part_rows, end = begin + p.part_rows < p.rows ? begin + p.part_rows : p.rows;
  float db[8], dg[8], gate[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    db[e] = dg[e] = 0.f;
    gate[e] = 1.f;
  }
  DropKey key{};
  if (p.drop.limit) key = drop_key(p.drop);
  if (col < p.n) {
    if (p.gate) epi_load<T>(p.gate, p.param32, VEC, col, cnt, gate);
#pragma unroll 2
    for (int64_t row = begin + slot; row < end; row += 8) {
      float g[8], z[8] = {};
      if constexpr (VEC)
        load_vec<8>((const TY*)p.dy + row * p.ld_dy + col, g);
      else
        load_some<8>((const TY*)p.dy + row * p.ld_dy + col, cnt, g);
      if (p.kept) epi_load<T>(p.kept, false, VEC, row * p.ld_kept + col, cnt, z);
      if (p.drop.limit) drop8(key, p.drop.limit, p.drop.scale, (uint32_t)col >> 3, (uint64_t)row, g, z);
      if (p.kept) {
        auto slopes = [&](int act) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float a;
            const float d = act_slope(act, z[e], &a);
            if constexpr (DGATE) dg[e] += g[e] * a;
            g[e] *= d;
          }
        };
        if (p.act == SAF3R_GELU) {
          slopes(SAF3R_GELU);
        } else if (p.act == SAF3R_GELU_TANH) {
          slopes(SAF3R_GELU_TANH);
        } else if constexpr (DGATE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) dg[e] += g[e] * z[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] *= gate[e];
        db[e] += g[e];
      }
      if (p.dz) store_vec<8>((T*)p.dz + row * p.ld_dz + col, g);
    }
  }
  if (!p.part) return;
  if constexpr (DGATE) add_slots<8, 32>(dg, lds);
  add_slots<8, 32>(db, lds);
  if (tid_x() < 32 && col < p.n && p.direct) {
    if (DGATE && p.dgate) epi_store<T>(p.dgate, p.param32, false, col, cnt, dg);
    if (p.dbias) epi_store<T>(p.dbias, p.param32, false, col, cnt, db);
  } else if (tid_x() < 32 && col < p.n) {
    float* to = p.part + (int64_t)bid_y() * 2 * p.n + col;
    if constexpr (VEC) {
      if constexpr (DGATE) store_vec<8>(to, dg);
      store_vec<8>(to + p.n, db);
    } else {
      if constexpr (DGATE) store_some<8>(to, cnt, dg);
      store_some<8>(to + p.n, cnt, db);
    }
  }
}

// Partial rows: work-groups for four on a compute unit, with at least sixteen rows each (with eight, the backward pass of 261 x 64
// to 4096 takes 17.3 us in place of 16.7, of 777 x 64 to 515 14.7 in place of 14.2); up to 32 rows one work-group has them all
// and writes the sums itself, which saves the launch of their second step.
int64_t linear_grad_parts(int64_t rows, int n) {
  const int64_t strips = (n + 255) / 256;
  return rows <= 32 ? 1 : std::max<int64_t>(1, std::min<int64_t>((1024 + strips - 1) / strips, rows / 16));
}

int linear_grad(const char* who, const LinearGradParams& p, int type, bool dy32, bool vec, bool dgate, int64_t parts,
                hipStream_t stream) {
  const dim3 grid((uint32_t)((p.n + 255) / 256), (uint32_t)parts);
  auto one = [&](auto t, auto ty, auto v, auto dg) {
    hipLaunchKernelGGL((linear_grad_kernel<decltype(t), decltype(ty), decltype(v)::value, decltype(dg)::value>), grid,
                       dim3(256), 0, stream, p);
    return check_launch(who);
  };
  auto go = [&](auto t, auto ty) {
    if (dgate) return vec ? one(t, ty, Int<1>(), Int<1>()) : one(t, ty, Int<0>(), Int<1>());
    return vec ? one(t, ty, Int<1>(), Int<0>()) : one(t, ty, Int<0>(), Int<0>());
  };
  if (type == SAF3R_BF16) return dy32 ? go(__bf16(), float()) : go(__bf16(), __bf16());
  return dy32 ? go(_Float16(), float()) : go(_Float16(), _Float16());
}

}  // namespace saf3r
