// Linear layers with their epilogue, and the products of their backward pass:
//   forward  y  = res + gate drop(act(x W^T + bias))   x [rows][in], W [out][in]
//   backward dx = dz W,  dW = dz^T x                   dz [rows][out] from linear_grad.hip
// All three are one product C[m][n] = sum_k A B whose operands lie with the reduction along a row (ROWS: x, W and dz of the
// first two) or across rows (COLS: W of the second, both of the third). bf16 or fp16 operands, fp32 sums.
//
// Bound by the matrix cores (and, in the largest products, by the clock that the card's power leaves them: 2.2 GHz falls to 1.6
// under 8192^3) for a few hundred rows or more, by the bytes of W below. Measured, bf16, launches in a graph:
//   8192^3                  800 to 825 us (1330 to 1380 TFLOP/s)
//   87936 x 1024 to 4096    690 to 720, with GELU and the kept values 860 to 900; dx 641, dW 555 to 580
//   10992 x 4096 to 1024    90, with gate, dropout and an fp32 residual 119; dx 93, dW 87
//   1041 x 1024 to 4096     19.5, with GELU and the kept values 23; dx 20.5, dW 15, both together 26
//   4 x 1024 to 4096        4.6
// A library product of the same sizes, without an epilogue: 8192^3 787; 87936 x 1024 to 4096 588, dx 663, dW 864; 10992 x 4096
// to 1024 72, dx 106, dW 118; 1041 x 1024 to 4096 19, dx 29, dW 22. The forward pass is behind at short reductions and where a
// round of tiles is not full: a tile's epilogue lies behind its products, and nothing of the next tile is copied meanwhile.
#include "linear.h"

#include <cmath>

namespace saf3r {

// What DMA lanes without an element of their own read: zeros.
__device__ const uint4 kZeros = {0, 0, 0, 0};

struct GemmParams {
  const char* a;
  const char* b;
  int64_t lda, ldb;  // bytes
  int m, n, k;
  int steps;         // steps of 64 of the whole reduction
  int split_steps;   // steps of a split
  int splits, tiles_m, tiles_n;
  int group;         // rows of tiles that are taken together
  float* part;       // splits > 1: [split][m][ldp]
  int64_t ldp;
  EpiParams epi;
};

// Unit of an operand: R rows (or columns), 128 or 64, by 64 of the reduction.
constexpr int unit_bytes(int r) { return r * 128; }

// How a wave copies its quarter of a unit: R / 32 instructions of 1 KB. ROWS: instruction j of wave w takes rows 8 (4 j + w)
// .. + 7 of 128 bytes; COLS: of the reduction's 64 rows of 2 R bytes the 1 KB from 4 j + w on. The 16-byte chunks of a row
// are swizzled by the row (the lanes' sources are, the LDS side of such a copy is linear).
// Swizzles: ROWS: swz8. COLS: a transposed read takes 64 bytes of four reduction rows for either half of the wave: those fall on
// 64 different banks when rows of 256 bytes differ in bits 2 and 3 of the chunk, rows of 128 bytes two apart in bit 2.
template <int R>
__device__ __forceinline__ int swz_cols(int kr) {
  return R == 128 ? (kr & 3) << 2 : ((kr >> 1) & 1) << 2;
}

template <bool COLS, int R>
struct Copy {
  static constexpr int kCount = R / 32, kRowChunks = R / 8, kKRows = 512 / R;  // COLS: chunks of a row, rows of 1 KB
  const char* base;      // the unit's first row or column, step 0
  uint32_t off[kCount];  // byte offset of the lane's chunk
  int at;            // its place along the reduction: element (ROWS) or row (COLS, instruction 0)

  // unit u of an operand of `count` rows (columns) from `first` (a unit behind the last one reads the first one's)
  __device__ __forceinline__ void init(int wave, int lane, const char* operand, int first, int count, int64_t ld) {
    first = first < count ? first : 0;
    base = operand + (COLS ? (int64_t)first * 2 : first * ld);
    if constexpr (COLS) {
      const int kr = kKRows * wave + lane / kRowChunks, chunk = (lane % kRowChunks) ^ swz_cols<R>(kr);
      // columns behind the last are the last chunk's: their results are not stored
      const int last = (count - 1) / 8 * 8 - first;
      const int c = chunk * 8 < last ? chunk * 8 : last;
      at = kr;
#pragma unroll
      for (int j = 0; j < kCount; ++j) off[j] = (uint32_t)((4 * kKRows * j + kr) * ld + c * 2);
    } else {
      const int r = 8 * wave + (lane >> 3), chunk = (lane & 7) ^ swz8(r), last = count - 1 - first;
      at = chunk * 8;
#pragma unroll
      for (int j = 0; j < kCount; ++j) {
        const int row = r + 32 * j < last ? r + 32 * j : last;
        off[j] = (uint32_t)(row * ld + chunk * 16);
      }
    }
  }

  // instruction J of step * its bytes to `lds`; with ANY only the first `left` elements (rows) of the step are there, zeros
  // in place of the others
  template <int J, bool ANY>
  __device__ __forceinline__ void issue(int64_t step_bytes, uint32_t lds, int left) const {
    if constexpr (ANY) {
      const bool there = at + (COLS ? 4 * kKRows * J : 0) < left;
      dma16(there ? base + step_bytes + off[J] : (const char*)&kZeros, lds + J * 4096);
    } else {
      dma16s(base + step_bytes, off[J], lds + J * 4096);
    }
  }
};

// The copies of a work-group of four waves: units 0 .. UB - 1 of a step are B's, the next UA are A's. With ANY a step may be
// the last one, of which `left` of 64 is there.
template <bool ACOLS, bool BCOLS, int UA, int UB, int SLOTS, int R = 128>
struct Feed {
  static constexpr int kUnit = unit_bytes(R);
  Copy<ACOLS, R> a[UA];
  Copy<BCOLS, R> b[UB];
  int64_t astep, bstep;
  uint32_t lds0;
  int s0, s1, left, tail;

  __device__ __forceinline__ void init(const GemmParams& p, int split, int m0, int n0, int wave, int lane, const char* lds) {
#pragma unroll
    for (int u = 0; u < UA; ++u) a[u].init(wave, lane, p.a, m0 + u * R, p.m, p.lda);
#pragma unroll
    for (int u = 0; u < UB; ++u) b[u].init(wave, lane, p.b, n0 + u * R, p.n, p.ldb);
    astep = ACOLS ? 64 * p.lda : 128;
    bstep = BCOLS ? 64 * p.ldb : 128;
    lds0 = lds_addr(lds) + wave * 1024;
    s0 = split * p.split_steps;
    s1 = s0 + p.split_steps < p.steps ? s0 + p.split_steps : p.steps;
    left = p.k - (p.steps - 1) * 64;                       // elements of the last step
    tail = left < 64 && s1 == p.steps ? p.steps - 1 : -1;  // the step with fewer than 64
  }
  // steps of this split whose 64 elements are there
  __device__ __forceinline__ int whole() const { return tail < 0 ? s1 : s1 - 1; }
  static __device__ __forceinline__ int after(int slot, int n) { return slot + n >= SLOTS ? slot + n - SLOTS : slot + n; }

  template <int U, int J, bool ANY>
  __device__ __forceinline__ void one(int step, int slot) const {
    const uint32_t to = lds0 + slot * kUnit;
    const int there = ANY && step == tail ? left : 64;
    if constexpr (U < UB)
      b[U].template issue<J, ANY>(step * bstep, to, there);
    else
      a[U - UB].template issue<J, ANY>(step * astep, to, there);
  }
  template <int U>
  __device__ __forceinline__ void unit(int step, int slot) const {
    if (step >= s1) return;
    one<U, 0, true>(step, slot);
    one<U, 1, true>(step, slot);
    if constexpr (R == 128) {
      one<U, 2, true>(step, slot);
      one<U, 3, true>(step, slot);
    }
  }
};

// Fragments of a wave's half of a unit (R / 64 blocks of 32 rows or columns) for the 32x32x16 products: lane l holds row l % 32
// of a block, elements 16 ks + 8 (l / 32) .. + 7 of the reduction.
template <bool COLS, typename T, int R = 128>
struct Frags {
  typedef typename Half<T>::vec8 vec8;
  static constexpr int kBlocks = R / 64;
  int addr[COLS ? kBlocks : 4];

  __device__ __forceinline__ void init(int lane, int part) {
    const int h = lane >> 5;
    if constexpr (COLS) {
      const int i = lane & 15, kr = 8 * h + (i >> 2), s = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        addr[b] = kr * 2 * R + ((4 * (kBlocks * part + b) + s) ^ swz_cols<R>(kr)) * 16 + 8 * (i & 1);
    } else {
      const int r = lane & 31;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) addr[ks] = (R / 2 * part + r) * 128 + (((2 * ks + h) ^ swz8(r)) << 4);
    }
  }

  __device__ __forceinline__ vec8 get(const char* unit, int block, int ks) const {
    if constexpr (COLS) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const char* p = unit + addr[block] + ks * 32 * R;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * R));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      return __builtin_bit_cast(vec8, u32x4{x[0], x[1], y[0], y[1]});
    } else {
      return *reinterpret_cast<const vec8*>(unit + addr[ks] + block * 4096);
    }
  }
};

// Work-groups go to the eight XCDs in turn: each XCD takes a contiguous range of the tiles, which go by groups of some
// rows of tiles (group_of), so that the work-groups of an XCD share operand rows in its L2.
struct Place {
  int tm, tn, split;
};
__device__ __forceinline__ Place place_of(const GemmParams& p, int id) {
  const int tiles = p.tiles_m * p.tiles_n, all = tiles * p.splits;
  const int q = all / 8, r = all % 8, x = id % 8;
  id = x * q + (x < r ? x : r) + id / 8;
  Place at;
  at.split = p.splits > 1 ? id / tiles : 0;
  id -= at.split * tiles;
  const int per = p.group * p.tiles_n, g = id / per, in = id - g * per, left = p.tiles_m - p.group * g;
  const int rows = left < p.group ? left : p.group;
  at.tn = in / rows;
  at.tm = p.group * g + in - at.tn * rows;
  return at;
}

// Results of 32 rows by 32 NB columns of a wave, blocks x[0], x[1] (a lane holds row l % 32, columns 8 q + 4 (l / 32) + e in
// element 4 q + e), through the wave's own part of LDS: read back, 4 NB lanes hold a row, each eight columns, so that every
// load and store of the epilogue takes whole lines. (Eight columns a lane of 32 rows, straight from the registers: four
// requests a line, and 87936 x 1024 to 4096 took an eighth longer, 840 us in place of 740 with the copies and tiles of
// the time.)
constexpr int turn_row(int nb) { return 32 * nb + 4; }           // floats: 16-byte places of 16 rows are distinct banks
constexpr int turn_bytes(int nb) { return 32 * turn_row(nb) * 4; }  // of a wave

template <typename T, int NB>
__device__ __forceinline__ void finish_rows(const GemmParams& p, const DropKey& key, const EpiCols<T>& cols, int split,
                                            int row0, int col0, float* turn, const f32x16 (&x)[NB]) {
  constexpr int kLanes = 4 * NB, kRows = 64 / kLanes, kPasses = 32 / kRows;  // lanes of a row, rows of a pass
  const int lane = tid_x() & 63, col = col0 + 8 * (lane % kLanes);
  int row = row0 + lane / kLanes;
  EpiPlace at;
  at.init(p.epi, row, col);
  // (the residual is on its way while the rows turn)
  float res[kPasses][8];
  if (p.epi.res && p.splits == 1) {
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass)
      if (row + kRows * pass < p.m && col < p.n)
        epi_load<T>(p.epi.res, p.epi.y32, p.epi.vec, at.res + kRows * pass * p.epi.ld_res, p.epi.n - col, res[pass]);
  }
  float* to = turn + (lane & 31) * turn_row(NB) + 4 * (lane >> 5);
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(to + 32 * b + 8 * q) = f32x4{x[b][4 * q], x[b][4 * q + 1], x[b][4 * q + 2], x[b][4 * q + 3]};
  asm volatile("" ::: "memory");  // (a wave's LDS accesses stay in their order)
  const float* from = turn + lane / kLanes * turn_row(NB) + 8 * (lane % kLanes);
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    float v[8];
    load_vec<8>(from + pass * kRows * turn_row(NB), v);
    if (row < p.m && col < p.n) {
      if (p.splits > 1)
        store_vec<8>(p.part + ((int64_t)split * p.m + row) * p.ldp + col, v);
      else
        epilogue8<T>(p.epi, key, cols, at, row, col, res[pass], v);
    }
    row += kRows;
    at.down(p.epi, kRows);
  }
  asm volatile("" ::: "memory");
}

// Nothing moves across: the order of products, LDS reads and copies is the one written down.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// This wave's copies but the last N are there and all that it read from LDS has come back; then every wave's.
template <int N>
__device__ __forceinline__ void arrive() {
  wait_vm<N>();
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  barrier_only();
}

// Before the first step, behind the wait for its copies: scalar loads have come back too, and the epilogue's flags are loaded
// (flags_there) before. Left to the compiler they are loaded ahead of the steps' loop, and with a scalar load under way at its
// start every step waits for all of its LDS reads before its first product.
__device__ __forceinline__ void flags_there(const GemmParams& p) {
  asm volatile("" ::"s"((int)p.epi.y32), "s"((int)p.epi.vec), "s"((int)p.epi.param32));
}
__device__ __forceinline__ void start() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  barrier_only();
}

// f(Int<0>()), f(Int<1>()), .., f(Int<N - 1>())
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F f) {
  if constexpr (I < N) {
    f(Int<I>());
    each<N, I + 1>(f);
  }
}

// 256 x 128 tile of four waves in two rows of two, each 64 x 64 of either unit of A; 80 KB of LDS and two work-groups a compute
// unit, so that one's epilogue lies under the other's products. Units go through a ring of five LDS slots. A step of 64 is four
// groups of products (16 of the reduction each) of A0, then A1; fragments are read into the registers that the groups before
// have done with:
//   group    0          1     |    2        3      4      5     |   6           7
//   reads    B A0 k3          |  A1 k0 k1  A1 k2  A1 k3         | B A0 k0' k1'  B A0 k2'     (': of the next step)
//   copies   A0'        A0'   |  A1'       A1'    A1' B" B"     | B"            A0"
// The first barrier waits for A1 of this step and frees B A0, the second waits for B A0 of the next step and frees A1. The copies
// are spread (all behind the barriers, 87936 x 4096 to 1024 takes 729 us in place of 690).
template <typename T, bool ACOLS, bool BCOLS>
__global__ void __launch_bounds__(256, 2) gemm_pair_kernel(const GemmParams p) {
  typedef typename Half<T>::vec8 vec8;
  typedef Feed<ACOLS, BCOLS, 2, 1, 5> F;
  constexpr int kUnit = F::kUnit;
  __shared__ __attribute__((aligned(16))) char lds[5 * kUnit];
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const Place at = place_of(p, bid_x());
  const int m0 = at.tm * 256, n0 = at.tn * 128;
  F feed;
  feed.init(p, at.split, m0, n0, wave, lane, lds);
  Frags<ACOLS, T> fa;
  Frags<BCOLS, T> fb;
  fa.init(lane, wm);
  fb.init(lane, wn);
  f32x16 acc[2][2][2];  // [unit][row block][column block]
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[u][i][j][e] = 0.f;
  vec8 af[2][4], bf[2][4];
  auto read_a = [&](int slot, int i, int ks) { af[i][ks] = fa.get(lds + slot * kUnit, i, ks); };
  auto read_b = [&](int slot, int j, int ks) { bf[j][ks] = fb.get(lds + slot * kUnit, j, ks); };
  // read n of B and A of ks
  auto read_ba = [&](int n, int b_slot, int a_slot, int ks) {
    if (n < 2)
      read_b(b_slot, n, ks);
    else if (n < 4)
      read_a(a_slot, n - 2, ks);
  };
  // the products of ks of a unit, hook(n) behind the n-th of four
  auto products = [&](auto which, auto at_k, auto hook) {
    constexpr int u = decltype(which)::value, ks = decltype(at_k)::value;
    each<4>([&](auto n) {
      constexpr int i = decltype(n)::value / 2, j = decltype(n)::value % 2;
      acc[u][i][j] = Half<T>::mma32(bf[j][ks], af[i][ks], acc[u][i][j]);
      hook(n);
      fence();
    });
  };

  flags_there(p);
  int s = feed.s0, slot = 0;  // slot: of B of this step
  const int s1 = feed.s1, whole = feed.whole();
      feed.template unit<0>(s, 0);
      feed.template unit<1>(s, 1);
      feed.template unit<2>(s, 2);
      feed.template unit<0>(s + 1, 3);
      if (s + 1 < s1)
        wait_vm<8>();
      else
        wait_vm<4>();
      start();
#pragma unroll
      for (int ks = 0; ks < 3; ++ks)
#pragma unroll
        for (int n = 0; n < 4; ++n) read_ba(n, 0, 1, ks);
      fence();
      // Copies of a step: NEXT: of the next one, LATER: of the one behind it (2: with the check for the last step).
      auto step = [&](auto next, auto later, int s) {
        constexpr int kNext = decltype(next)::value, kLater = decltype(later)::value;
        const int a0 = F::after(slot, 1), a1 = F::after(slot, 2), b_next = F::after(slot, 3), a0_next = F::after(slot, 4);
        auto copy_next = [&](auto unit, auto j, int to) {
          if constexpr (kNext != 0) feed.template one<decltype(unit)::value, decltype(j)::value, kNext == 2>(s + 1, to);
        };
        auto copy_later = [&](auto unit, auto j, int to) {
          if constexpr (kLater != 0) feed.template one<decltype(unit)::value, decltype(j)::value, kLater == 2>(s + 2, to);
        };
        products(Int<0>(), Int<0>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          read_ba(m, slot, a0, 3);
          if constexpr (m == 1) copy_next(Int<1>(), Int<1>(), a0_next);
        });
        products(Int<0>(), Int<1>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          if constexpr (m == 0) copy_next(Int<1>(), Int<2>(), a0_next);
          if constexpr (m == 2) copy_next(Int<1>(), Int<3>(), a0_next);
        });
        arrive<kNext ? 8 : 0>();  // (behind A1: B and A0 of the next step)
        products(Int<0>(), Int<2>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          read_a(a1, m % 2, m / 2);
          if constexpr (m == 2) copy_next(Int<2>(), Int<0>(), slot);
        });
        products(Int<0>(), Int<3>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          if constexpr (m % 2 == 1) read_a(a1, m / 2, 2);
          if constexpr (m == 0) copy_next(Int<2>(), Int<1>(), slot);
          if constexpr (m == 2) copy_next(Int<2>(), Int<2>(), slot);
        });
        products(Int<1>(), Int<0>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          if constexpr (m % 2 == 1) read_a(a1, m / 2, 3);
          if constexpr (m == 0) copy_next(Int<2>(), Int<3>(), slot);
          if constexpr (m == 2) copy_later(Int<0>(), Int<0>(), a0);
        });
        products(Int<1>(), Int<1>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          if constexpr (m == 0) copy_later(Int<0>(), Int<1>(), a0);
          if constexpr (m == 2) copy_later(Int<0>(), Int<2>(), a0);
        });
        // (behind A0 of the next step: its A1 and three instructions of B behind it)
        if constexpr (kNext != 0) arrive<kLater ? 7 : 4>();
        products(Int<1>(), Int<2>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          if constexpr (kNext != 0) {
            read_ba(m, b_next, a0_next, 0);
            read_ba(m, b_next, a0_next, 1);
          }
          if constexpr (m == 2) copy_later(Int<0>(), Int<3>(), a0);
        });
        products(Int<1>(), Int<3>(), [&](auto n) {
          constexpr int m = decltype(n)::value;
          if constexpr (kNext != 0) read_ba(m, b_next, a0_next, 2);
          if constexpr (m == 1) copy_later(Int<1>(), Int<0>(), a1);
        });
        slot = b_next;
      };
      // (A0 of the second step, whose first instruction belongs to the step before)
      if (s + 1 < s1) feed.template one<1, 0, true>(s + 1, 4);
#pragma unroll 1
      for (; s + 2 < whole; ++s) step(Int<1>(), Int<1>(), s);
      if (s + 2 < s1) step(Int<1>(), Int<2>(), s++);
      if (s + 1 < s1) step(Int<2>(), Int<0>(), s++);
      step(Int<0>(), Int<0>(), s);

  __syncthreads();  // (the slots are read to their end)
  float* turn = reinterpret_cast<float*>(lds + wave * turn_bytes(2));
  DropKey key{};
  if (p.epi.drop.limit) key = drop_key(p.epi.drop);
  EpiCols<T> cols;
  const int col0 = n0 + 64 * wn, col = col0 + 8 * (lane & 7);
  if (p.splits == 1 && col < p.n) cols.load(p.epi, col);
#pragma unroll 1
  for (int blk = 0; blk < 4; ++blk) {
    f32x16 x[2];
    switch (blk) {
      case 0: x[0] = acc[0][0][0], x[1] = acc[0][0][1]; break;
      case 1: x[0] = acc[0][1][0], x[1] = acc[0][1][1]; break;
      case 2: x[0] = acc[1][0][0], x[1] = acc[1][0][1]; break;
      default: x[0] = acc[1][1][0], x[1] = acc[1][1][1]; break;
    }
    finish_rows<T, 2>(p, key, cols, at.split, m0 + 128 * (blk >> 1) + 64 * wm + 32 * (blk & 1), col0, turn, x);
  }
}

// Tiles of 128 x 128 (NB 2) and 64 x 64 (NB 1) for products with few of the larger ones: four waves in two rows of two, each NB x
// NB blocks. A step is bound by its copies (32 or 16 instructions of 28 cycles); a short product by its first copies' way and
// by the epilogue, which smaller tiles spread over more compute units. Units of both operands go through a ring of SLOTS. A step is
// four groups of NB x NB products; of 128 x 128, with the barrier behind the second product of group 1 (of 64 x 64 behind group 1):
//   group    0        1         2         3
//   reads    B A k3   | B A k0'  B A k1'   B A k2'     (': of the next step)
//   copies            |          B         A           (of the step whose place is free)
// Reads and copies are spread, one or two behind a product: the four waves read together behind a barrier, and eight reads at
// once hold up the products (dW of 10992 x 1024 to 4096 92.6 -> 87 us, 1041 x 4096 to 1024 21.2 -> 20.3).
template <typename T, bool ACOLS, bool BCOLS, int NB, int SLOTS>
__device__ __forceinline__ void small_tile(const GemmParams& p, int id, char* lds) {
  typedef typename Half<T>::vec8 vec8;
  constexpr int R = 64 * NB, kPer = R / 32;  // rows of a unit, a wave's instructions for it
  typedef Feed<ACOLS, BCOLS, 1, 1, SLOTS, R> F;
  constexpr int kUnit = F::kUnit;
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const Place at = place_of(p, id);
  const int m0 = at.tm * R, n0 = at.tn * R;
  F feed;
  feed.init(p, at.split, m0, n0, wave, lane, lds);
  Frags<ACOLS, T, R> fa;
  Frags<BCOLS, T, R> fb;
  fa.init(lane, wm);
  fb.init(lane, wn);
  f32x16 acc[NB][NB];  // [row block][column block]
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  vec8 af[NB][4], bf[NB][4];
  // the fragments of ks
  auto read = [&](int b_slot, int a_slot, int ks) {
#pragma unroll
    for (int j = 0; j < NB; ++j) bf[j][ks] = fb.get(lds + b_slot * kUnit, j, ks);
#pragma unroll
    for (int i = 0; i < NB; ++i) af[i][ks] = fa.get(lds + a_slot * kUnit, i, ks);
  };
  // the products of ks, hook(n) behind the n-th
  auto products = [&](auto at_k, auto hook) {
    constexpr int ks = decltype(at_k)::value;
    each<NB * NB>([&](auto n) {
      constexpr int i = decltype(n)::value / NB, j = decltype(n)::value % NB;
      acc[i][j] = Half<T>::mma32(bf[j][ks], af[i][ks], acc[i][j]);
      hook(at_k, n);
      fence();
    });
  };

  flags_there(p);
  int s = feed.s0, slot = 0;  // slot: of B of this step
  const int s1 = feed.s1, whole = feed.whole();
  constexpr int kAhead = SLOTS / 2;  // steps whose units have a place
  each<kAhead>([&](auto n) {
    constexpr int i = decltype(n)::value;
    feed.template unit<0>(s + i, 2 * i);
    feed.template unit<1>(s + i, 2 * i + 1);
  });
  if (s1 - s >= kAhead)
    wait_vm<2 * kPer * (kAhead - 1)>();
  else
    wait_vm<0>();
  start();
  read(0, 1, 0);
  read(0, 1, 1);
  read(0, 1, 2);
  fence();
  // behind: steps behind the next one whose copies are under way (-1: there is no next one); ahead: copies of step s + kAhead
  // (2: with the check for the last step)
  auto step = [&](auto behind, auto ahead, int s) {
    constexpr int kBehind = decltype(behind)::value, kCopy = decltype(ahead)::value;
    const int a0 = F::after(slot, 1), b_next = F::after(slot, 2), a_next = F::after(slot, 3);
    auto copy = [&](auto unit, auto n, int to) {
      constexpr int j = decltype(n)::value;
      if constexpr (kCopy != 0 && j < kPer) feed.template one<decltype(unit)::value, j, kCopy == 2>(s + kAhead, to);
    };
    // fragment f of ks: B's blocks, then A's
    auto read_one = [&](int f, int b_slot, int a_slot, int ks) {
      if (f < NB)
        bf[f][ks] = fb.get(lds + b_slot * kUnit, f, ks);
      else
        af[f - NB][ks] = fa.get(lds + a_slot * kUnit, f - NB, ks);
    };
    auto hook = [&](auto at_k, auto n) {
      constexpr int i = NB * NB * decltype(at_k)::value + decltype(n)::value;  // products of this step so far
      constexpr bool kNext = kBehind >= 0;
      if constexpr (NB == 1) {
        if constexpr (i == 0) read(slot, a0, 3);
        if constexpr (kNext && i == 2) read(b_next, a_next, 0);
        if constexpr (kNext && i == 2) read(b_next, a_next, 1);
        if constexpr (kNext && i == 3) read(b_next, a_next, 2);
        if constexpr (i >= 2) {
          copy(Int<i - 2>(), Int<0>(), i == 2 ? slot : a0);
          copy(Int<i - 2>(), Int<1>(), i == 2 ? slot : a0);
        }
      } else {
        if constexpr (i < 2) {
          read_one(2 * i, slot, a0, 3);
          read_one(2 * i + 1, slot, a0, 3);
        }
        if constexpr (kNext && i >= 6 && i < 8) {
          read_one(2 * i - 12, b_next, a_next, 0);
          read_one(2 * i - 11, b_next, a_next, 0);
        }
        if constexpr (kNext && i >= 8) read_one(i % 4, b_next, a_next, i / 4 - 1);
        if constexpr (i >= 8) copy(Int<i / 4 - 2>(), Int<i % 4>(), i < 12 ? slot : a0);
      }
      if constexpr (kNext && i == (NB == 1 ? 1 : 5)) arrive<2 * kPer * (kBehind > 0 ? kBehind : 0)>();
    };
    products(Int<0>(), hook);
    products(Int<1>(), hook);
    products(Int<2>(), hook);
    products(Int<3>(), hook);
    slot = b_next;
  };
#pragma unroll 1
  for (; s + kAhead < whole; ++s) step(Int<kAhead - 2>(), Int<1>(), s);
  if (s + kAhead < s1) step(Int<kAhead - 2>(), Int<2>(), s++);
  each<kAhead>([&](auto n) {  // the last kAhead steps
    constexpr int r = kAhead - decltype(n)::value;
    if (s1 - s == r) step(Int<r - 2>(), Int<0>(), s++);
  });

  __syncthreads();  // (the slots are read to their end)
  float* turn = reinterpret_cast<float*>(lds + wave * turn_bytes(NB));
  DropKey key{};
  if (p.epi.drop.limit) key = drop_key(p.epi.drop);
  EpiCols<T> cols;
  const int col0 = n0 + 32 * NB * wn, col = col0 + 8 * (lane % (4 * NB));
  if (p.splits == 1 && col < p.n) cols.load(p.epi, col);
#pragma unroll
  for (int i = 0; i < NB; ++i) finish_rows<T, NB>(p, key, cols, at.split, m0 + 32 * (NB * wm + i), col0, turn, acc[i]);
}

template <typename T, bool ACOLS, bool BCOLS, int NB, int SLOTS>
__global__ void __launch_bounds__(256, SLOTS * NB > 10 ? 1 : 2) gemm_small_kernel(const GemmParams p) {
  __shared__ __attribute__((aligned(16))) char lds[SLOTS * unit_bytes(64 * NB)];
  small_tile<T, ACOLS, BCOLS, NB, SLOTS>(p, bid_x(), lds);
}

// Both products of a small backward pass, dx in the first work-groups and dW in the rest: neither fills the card, and a launch
// is saved (1041 x 1024 to 4096: 37 -> 31 us, 64 x 1024 to 4096: 17 -> 13).
struct BothParams {
  GemmParams dx, dw;
  int first;  // work-groups of dx
};
template <typename T, int NB, int SLOTS>
__global__ void __launch_bounds__(256, SLOTS * NB > 10 ? 1 : 2) gemm_both_kernel(const BothParams p) {
  __shared__ __attribute__((aligned(16))) char lds[SLOTS * unit_bytes(64 * NB)];
  if (bid_x() < p.first)
    small_tile<T, false, true, NB, SLOTS>(p.dx, bid_x(), lds);
  else
    small_tile<T, true, true, NB, SLOTS>(p.dw, bid_x() - p.first, lds);
}

// 256 x 256 tile of four waves, one a SIMD: each owns 64 rows of both A units by a whole unit of B (128 x 128 in all, 256 sums a
// lane), which reads 32 KB of LDS for 128 products, a third less than two waves of 128 x 64, and copies a third less than
// tiles of 256 x 128. Every product is followed by at most a read and a copy, which issue under it (a 32x32x16 product
// holds the pipe for 32 cycles). A step is four groups of 16 products:
//   group    A0 k0 k1    |  A0 k2 k3    A1 k0 k1    A1 k2 k3
//   reads    B A0 k2 k3  |  A1 k0 k1    A1 k2 k3    B A0 k0' k1'     (': of the next step)
//   copies   B0"         |  B1"         A0"         A1"
// into the registers, and slots, that the groups before have done with. The barrier waits for A1 of this step and B0 B1 A0 of
// the next one; it frees B0 B1 A0 of this one and A1 of the last. The data path takes 28 cycles for an instruction of 1 KB
// at the hit rates of these products (15 from the L2, 40 to 50 from behind it), 64 of them a step of 2048 cycles of
// products: they are spread evenly (in a burst behind the barrier, 8192^3 takes 902 us in place of 820).
template <typename T, bool ACOLS, bool BCOLS>
__global__ void __launch_bounds__(256, 1) gemm_wide_kernel(const GemmParams p) {
  typedef typename Half<T>::vec8 vec8;
  typedef Feed<ACOLS, BCOLS, 2, 2, 10> F;
  constexpr int kUnit = F::kUnit;
  __shared__ __attribute__((aligned(16))) char lds[10 * kUnit];
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const Place at = place_of(p, bid_x());
  const int m0 = at.tm * 256, n0 = at.tn * 256;
  F feed;
  feed.init(p, at.split, m0, n0, wave, lane, lds);
  Frags<ACOLS, T> fa;
  Frags<BCOLS, T> fb[2];
  fa.init(lane, wm);
  fb[0].init(lane, 0);
  fb[1].init(lane, 1);
  f32x16 acc[2][2][4];  // [unit][row block][column block]
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[u][i][j][e] = 0.f;
  vec8 af[2][4], bf[4][4];
  auto read_a = [&](int slot, int i, int ks) { af[i][ks] = fa.get(lds + slot * kUnit, i, ks); };
  auto read_b = [&](int slot, int j, int ks) { bf[j][ks] = fb[j >> 1].get(lds + slot * kUnit, j & 1, ks); };
  // read n of B and A of ks and ks + 1
  auto read_ba = [&](int n, int b_slot, int a_slot, int ks) {
    if (n < 8)
      read_b(b_slot, n % 4, ks + n / 4);
    else if (n < 12)
      read_a(a_slot, n % 2, ks + (n - 8) / 2);
  };
  // the products of ks and ks + 1 of a unit, hook(n) behind the n-th of 16
  auto products = [&](auto which, auto first, auto hook) {
    constexpr int u = decltype(which)::value, k0 = decltype(first)::value;
    each<16>([&](auto n) {
      constexpr int m = decltype(n)::value, ks = k0 + m / 8, i = m / 4 % 2, j = m % 4;
      acc[u][i][j] = Half<T>::mma32(bf[j][ks], af[i][ks], acc[u][i][j]);
      hook(n);
      fence();
    });
  };

  flags_there(p);
  int s = feed.s0, slot = 0;  // slot: of B0 of this step
  each<2>([&](auto n) {
    constexpr int i = decltype(n)::value;
    feed.template unit<0>(s + i, 4 * i);
    feed.template unit<1>(s + i, 4 * i + 1);
    feed.template unit<2>(s + i, 4 * i + 2);
    feed.template unit<3>(s + i, 4 * i + 3);
  });
  if (s + 1 < feed.s1)
    wait_vm<20>();
  else
    wait_vm<4>();
  start();
#pragma unroll
  for (int n = 0; n < 12; ++n) read_ba(n, wn, 2, 0);
  fence();
  // ahead: copies of step s + 2 (2: with the check for the last step; 0: none, and all that is under way is waited for)
  auto step = [&](auto ahead, int s) {
    constexpr int kCopy = decltype(ahead)::value;
    auto copy = [&](auto unit, auto j, int to) {
      if constexpr (kCopy != 0) feed.template one<decltype(unit)::value, decltype(j)::value, kCopy == 2>(s + 2, to);
    };
    const int b_at = F::after(slot, wn), a0 = F::after(slot, 2), a1 = F::after(slot, 3);
    const int b_next = F::after(slot, 4 + wn), a0_next = F::after(slot, 6);
    const int to0 = F::after(slot, 8), to1 = F::after(slot, 9), to3 = F::after(slot, 1);
    products(Int<0>(), Int<0>(), [&](auto n) {
      constexpr int m = decltype(n)::value;
      read_ba(m, b_at, a0, 2);
      if constexpr (m % 4 == 1) copy(Int<0>(), Int<m / 4>(), to0);
    });
    arrive<kCopy ? 8 : 0>();  // (behind A0 of the next step: its A1 and B0 of the step after it)
    products(Int<0>(), Int<2>(), [&](auto n) {
      constexpr int m = decltype(n)::value;
      if constexpr (m % 4 == 0) read_a(a1, m / 4 % 2, m / 8);
      if constexpr (m % 4 == 1) copy(Int<1>(), Int<m / 4>(), to1);
    });
    products(Int<1>(), Int<0>(), [&](auto n) {
      constexpr int m = decltype(n)::value;
      if constexpr (m % 2 == 0 && m < 8) read_a(a1, m / 2 % 2, 2 + m / 4);
      if constexpr (m % 4 == 1) copy(Int<2>(), Int<m / 4>(), slot);
    });
    products(Int<1>(), Int<2>(), [&](auto n) {
      constexpr int m = decltype(n)::value;
      read_ba(m, b_next, a0_next, 0);
      if constexpr (m % 4 == 1) copy(Int<3>(), Int<m / 4>(), to3);
    });
    slot = F::after(slot, 4);
  };
  const int s1 = feed.s1, whole = feed.whole();
#pragma unroll 1
  for (; s + 2 < whole; ++s) step(Int<1>(), s);
#pragma unroll 1
  for (; s + 2 < s1; ++s) step(Int<2>(), s);  // (once at most)
#pragma unroll 1
  for (; s < s1; ++s) step(Int<0>(), s);
  __syncthreads();  // (the slots are read to their end)
  float* turn = reinterpret_cast<float*>(lds + wave * turn_bytes(2));
  DropKey key{};
  if (p.epi.drop.limit) key = drop_key(p.epi.drop);
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    EpiCols<T> cols;
    const int col0 = n0 + 128 * wn + 64 * part;
    if (p.splits == 1 && col0 + 8 * (lane & 7) < p.n) cols.load(p.epi, col0 + 8 * (lane & 7));
#pragma unroll 1
    for (int blk = 0; blk < 4; ++blk) {
      f32x16 x[2];
      switch (4 * part + blk) {
        case 0: x[0] = acc[0][0][0], x[1] = acc[0][0][1]; break;
        case 1: x[0] = acc[0][1][0], x[1] = acc[0][1][1]; break;
        case 2: x[0] = acc[1][0][0], x[1] = acc[1][0][1]; break;
        case 3: x[0] = acc[1][1][0], x[1] = acc[1][1][1]; break;
        case 4: x[0] = acc[0][0][2], x[1] = acc[0][0][3]; break;
        case 5: x[0] = acc[0][1][2], x[1] = acc[0][1][3]; break;
        case 6: x[0] = acc[1][0][2], x[1] = acc[1][0][3]; break;
        default: x[0] = acc[1][1][2], x[1] = acc[1][1][3]; break;
      }
      finish_rows<T, 2>(p, key, cols, at.split, m0 + 128 * (blk >> 1) + 64 * wm + 32 * (blk & 1), col0, turn, x);
    }
  }
}

// Few rows (16 MB at most): a work-group computes 16 columns; its eight waves take the reduction in turns of 64, straight from
// memory into the fragments of 16x16x32 products (a lane reads both halves of a 128-byte line of its row of W), and are
// joined in LDS. W is read once, by n / 16 work-groups with every load of a wave's share under way at once.
template <typename T, int MB>
__global__ void __launch_bounds__(512) few_rows_kernel(const GemmParams p) {
  typedef typename Half<T>::vec8 vec8;
  constexpr int kWaves = 8, kAhead = 4;  // turns of a wave whose loads are under way together
  __shared__ __attribute__((aligned(16))) float lds[kWaves][MB][16][20];
  const int lane = tid_x() & 63, wave = tid_x() >> 6;
  const int n0 = bid_x() * 16, i = lane & 15, at = (lane >> 4) * 8;
  const int nrow = n0 + i < p.n ? n0 + i : p.n - 1;
  const T* wp = (const T*)(p.b + nrow * p.ldb);
  const T* xp[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) xp[b] = (const T*)(p.a + (int64_t)(16 * b + i < p.m ? 16 * b + i : p.m - 1) * p.lda);
  f32x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[b][e] = 0.f;
  vec8 none;
#pragma unroll
  for (int e = 0; e < 8; ++e) none[e] = (T)0.f;
#pragma unroll 1
  for (int k0 = wave * 64; k0 < p.k; k0 += kWaves * 64 * kAhead) {
    vec8 w[kAhead][2], x[kAhead][2][MB];
#pragma unroll
    for (int t = 0; t < kAhead; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int k = k0 + t * kWaves * 64 + 32 * c + at;
        const bool there = k < p.k;  // (k is a multiple of 8)
        w[t][c] = there ? *reinterpret_cast<const vec8*>(wp + k) : none;
#pragma unroll
        for (int b = 0; b < MB; ++b) x[t][c][b] = there ? *reinterpret_cast<const vec8*>(xp[b] + k) : none;
      }
#pragma unroll
    for (int t = 0; t < kAhead; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[b] = Half<T>::mma16(w[t][c], x[t][c][b], acc[b]);
  }
  // element e of a lane: row l % 16 (of A), column 4 (l / 16) + e
#pragma unroll
  for (int b = 0; b < MB; ++b) *reinterpret_cast<f32x4*>(&lds[wave][b][i][(lane >> 4) * 4]) = acc[b];
  __syncthreads();
  if (tid_x() >= MB * 32) return;
  const int row = tid_x() >> 1, c8 = (tid_x() & 1) * 8;
  if (row >= p.m || n0 + c8 >= p.n) return;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v[e] += lds[w][row >> 4][row & 15][c8 + e];
  }
  DropKey key{};
  if (p.epi.drop.limit) key = drop_key(p.epi.drop);
  epilogue8<T>(p.epi, key, row, n0 + c8, v);
}

// Adds the splits of a reduction in their order and applies the epilogue; a thread owns eight columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const GemmParams p) {
  const int groups = (int)(p.ldp / 8);
  const int64_t at = (int64_t)bid_x() * 256 + tid_x();
  if (at >= (int64_t)p.m * groups) return;
  const int row = (int)(at / groups), col = (int)(at - (int64_t)row * groups) * 8;
  const float* from = p.part + (int64_t)row * p.ldp + col;
  float v[8];
  load_vec<8>(from, v);
#pragma unroll 4
  for (int s = 1; s < p.splits; ++s) {
    float x[8];
    load_vec<8>(from + s * (p.m * p.ldp), x);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x[e];
  }
  DropKey key{};
  if (p.epi.drop.limit) key = drop_key(p.epi.drop);
  epilogue8<T>(p.epi, key, row, col, v);
}

constexpr int kMaxSize = 1 << 21;         // widths of a layer (a unit's byte offsets stay in 32 bits)
constexpr int64_t kMaxRows = 0x7fffff00;  // rows of a layer

constexpr int64_t kMaxTiles = 0xffffffffll / 256;  // (a launch counts its threads in 32 bits)

// How a product runs: the kernel for few rows, or tiles of one kind and splits of the reduction.
enum Kind { kTiny, kSmall, kPair, kWide, kKinds };
constexpr int kTileM[kKinds] = {64, 128, 256, 256}, kTileN[kKinds] = {64, 128, 128, 256};
struct Plan {
  bool few;
  double time;
  int kind, splits, split_steps, steps, tiles_m, tiles_n;
};

// Microseconds of a product with `wgs` work-groups of one kind and `steps` steps each, from what single kinds took over 70 to
// 87936 rows, widths of 128 to 6144 and 1 to 16 splits: start and end; a step while every work-group has a compute unit of
// its own (few of them, and more with their number: the card's clock goes down under load); of two on a unit, a step of the
// slower and, with 512, of the whole card. A round behind the first costs half of one at least.
// `epilogue`: cycles of a value's activation, dropout and residual; the values of a lane are 16 to 256 a tile.
static double tile_time(int kind, int64_t wgs, int64_t steps, int epilogue) {
  constexpr struct {
    double ends, alone, shared, two, full;
    int places;
  } kTimes[kKinds] = {{5.5, 0.19, 0.06, 0.30, 0.45, 512},
                      {7.5, 0.31, 0.18, 0.72, 1.00, 512},
                      {10.0, 0.49, 0.44, 1.20, 1.75, 512},
                      {16.0, 0.97, 0.60, 1.57, 1.57, 256}};
  auto k = kTimes[kind];
  k.ends += (kTileM[kind] * kTileN[kind] / 256) * epilogue / 2100.0;
  const double x = (double)wgs / 256;
  if (wgs <= 256) return k.ends + (double)steps * (k.alone + k.shared * x * x);
  if (wgs <= k.places) return k.ends + (double)steps * (k.two + (k.full - k.two) * (x - 1));
  const int64_t halves = (2 * wgs + k.places - 1) / k.places;
  const double end = kind == kWide ? k.ends : 0.5 * k.ends;  // (of two on a unit, one ends under the other)
  return k.ends + 0.5 * (double)halves * (double)steps * k.full + 0.5 * (double)(halves - 2) * end;
}

// Cycles of a value's epilogue behind its conversion.
static int epilogue_cycles(int act, int drop) { return (act != SAF3R_NO_ACTIVATION ? 80 : 0) + (drop ? 70 : 0); }

// Tiles and splits of the least such time. There are two steps a split at least, but steps are shared out rounded up: the last
// split has what is left, which may be one step (19 steps in splits of 3). The join is a launch more, and writes and reads the
// partial sums once (5.5 TB/s). Against one kind and split for all sizes: 4096 x 1024 from 1041 rows 27.6 -> 16.3 us,
// 1024 x 1024 from 2748 rows 24 -> 15, 128 x 512 from 20000 rows 24.6 -> 18.9, 10992 x 1024 from 4096 105 -> 93.
static Plan plan_of(int64_t m, int n, int64_t k, bool rows_kind, int epilogue) {
  Plan r{};
  r.steps = (int)((k + 63) / 64);
  r.few = rows_kind && m <= 32;
  r.time = 1e300;
  for (int kind = 0; kind < kKinds; ++kind) {
    const int64_t tm = (m + kTileM[kind] - 1) / kTileM[kind], tn = ((int64_t)n + kTileN[kind] - 1) / kTileN[kind];
    if (kind != kWide && tm * tn > kMaxTiles) continue;
    for (int splits = 1; splits <= 64; splits += splits < 4 ? 1 : splits < 8 ? 2 : splits < 16 ? 4 : 8) {
      if (splits > 1 && (r.steps < 2 * splits || tm * tn * splits > 1024)) break;
      const int per = (r.steps + splits - 1) / splits, used = (r.steps + per - 1) / per;
      double t = tile_time(kind, tm * tn * used, per, used > 1 ? 0 : epilogue);
      if (used > 1) t += 2.5 + (double)used * (double)m * n * 8 / 5.5e6;
      if (t < r.time) {
        r.time = t;
        r.kind = kind;
        r.splits = used;
        r.split_steps = per;
        r.tiles_m = (int)tm;
        r.tiles_n = (int)tn;
      }
    }
  }
  return r;
}

// Rows of tiles of a group (place_of). An XCD runs so many consecutive tiles at a time, at best as square a part of C as they can
// make: its rows and columns of operands are what its L2 has to fetch. Whole rows where a row of tiles is shorter than that.
// (Against groups of eight rows everywhere: 87936 x 4096 to 1024 647 -> 634 us, its dx of 1024 columns 652 -> 641, 10992 x 4096
// to 1024 92.7 -> 91, 1041 x 4096 to 1024 21.7 -> 21.3; 8192^3 the same within 1%.)
static int group_of(int kind, int tiles_m, int tiles_n, int splits) {
  const int64_t all = (int64_t)tiles_m * tiles_n * splits, places = kind == kWide ? 32 : 64;
  const double at_once = (double)std::min<int64_t>(places, (all + 7) / 8);
  const double high = std::sqrt(at_once * kTileN[kind] / kTileM[kind]);
  if (at_once >= high * tiles_n) return 1;
  const int groups = std::max(1, (int)(tiles_m / high + 0.5));
  return (tiles_m + groups - 1) / groups;
}

static int64_t part_bytes(const Plan& r, int64_t m, int n) {
  return r.few || r.splits == 1 ? 0 : (int64_t)r.splits * m * ((n + 7) / 8 * 8) * 4;
}

// The operands, sizes and splits of a product C = A B; `part` holds part_bytes.
static GemmParams params_of(const Plan& r, const void* a, int64_t lda, const void* b, int64_t ldb, int64_t m, int n, int64_t k,
                            const EpiParams& epi, void* part) {
  GemmParams p{};
  p.a = (const char*)a;
  p.b = (const char*)b;
  p.lda = lda * 2;
  p.ldb = ldb * 2;
  p.m = (int)m;
  p.n = n;
  p.k = (int)k;
  p.epi = epi;
  p.steps = r.steps;
  p.split_steps = r.split_steps;
  p.splits = r.splits;
  p.tiles_m = r.tiles_m;
  p.tiles_n = r.tiles_n;
  p.group = group_of(r.kind, r.tiles_m, r.tiles_n, r.splits);
  p.part = (float*)part;
  p.ldp = (n + 7) / 8 * 8;
  return p;
}

template <typename T>
static int join(const char* who, const GemmParams& p, hipStream_t stream) {
  if (p.splits == 1) return SAF3R_OK;
  const int64_t threads = p.m * (p.ldp / 8);
  hipLaunchKernelGGL((join_kernel<T>), dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, stream, p);
  return check_launch(who);
}

// The product with the plan's kernels.
template <typename T, bool ACOLS, bool BCOLS>
static int product(const char* who, const Plan& r, const GemmParams& p, hipStream_t stream) {
  if constexpr (!ACOLS && !BCOLS) {
    if (r.few) {
      const dim3 grid((uint32_t)((p.n + 15) / 16));
      if (p.m <= 16)
        hipLaunchKernelGGL((few_rows_kernel<T, 1>), grid, dim3(512), 0, stream, p);
      else
        hipLaunchKernelGGL((few_rows_kernel<T, 2>), grid, dim3(512), 0, stream, p);
      return check_launch(who);
    }
  }
  const int64_t grid = (int64_t)r.tiles_m * r.tiles_n * r.splits;
  if (grid > kMaxTiles) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many tiles for one launch", who);
  const dim3 wgs((uint32_t)grid);
  if (r.kind == kWide)
    hipLaunchKernelGGL((gemm_wide_kernel<T, ACOLS, BCOLS>), wgs, dim3(256), 0, stream, p);
  else if (r.kind == kPair)
    hipLaunchKernelGGL((gemm_pair_kernel<T, ACOLS, BCOLS>), wgs, dim3(256), 0, stream, p);
  else if (r.kind == kTiny)
    hipLaunchKernelGGL((gemm_small_kernel<T, ACOLS, BCOLS, 1, 10>), wgs, dim3(256), 0, stream, p);
  else if (grid <= 256)  // (one a compute unit: twice the units on their way)
    hipLaunchKernelGGL((gemm_small_kernel<T, ACOLS, BCOLS, 2, 10>), wgs, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((gemm_small_kernel<T, ACOLS, BCOLS, 2, 4>), wgs, dim3(256), 0, stream, p);
  if (int e = check_launch(who)) return e;
  return join<T>(who, p, stream);
}

// Both products of a backward pass. Where both are small they run in one launch, with tiles of one kind and each with its own
// splits: the order of every sum, and so every bit, is that of the product by itself.
template <typename T>
static int both_products(const char* who, Plan rx, GemmParams dx, Plan rw, GemmParams dw, hipStream_t stream) {
  if (rx.kind <= kSmall && rw.kind <= kSmall) {
    int kind = -1;
    double best = rx.time + rw.time;
    for (int c : {kTiny, kSmall}) {
      const int64_t wgs = (int64_t)((dx.m + kTileM[c] - 1) / kTileM[c]) * ((dx.n + kTileN[c] - 1) / kTileN[c]) * dx.splits +
                          (int64_t)((dw.m + kTileM[c] - 1) / kTileM[c]) * ((dw.n + kTileN[c] - 1) / kTileN[c]) * dw.splits;
      if (wgs > 1024) continue;
      const double t = tile_time(c, wgs, std::max(dx.split_steps, dw.split_steps), 0) + (dx.splits > 1 ? 2.5 : 0) +
                       (dw.splits > 1 ? 2.5 : 0);
      if (t < best) {
        best = t;
        kind = c;
      }
    }
    if (kind >= 0) {
      BothParams p{dx, dw, 0};
      for (GemmParams* g : {&p.dx, &p.dw}) {
        g->tiles_m = (g->m + kTileM[kind] - 1) / kTileM[kind];
        g->tiles_n = (g->n + kTileN[kind] - 1) / kTileN[kind];
        g->group = group_of(kind, g->tiles_m, g->tiles_n, g->splits);
      }
      p.first = p.dx.tiles_m * p.dx.tiles_n * p.dx.splits;
      const int wgs = p.first + p.dw.tiles_m * p.dw.tiles_n * p.dw.splits;
      if (kind == kTiny)
        hipLaunchKernelGGL((gemm_both_kernel<T, 1, 10>), dim3((uint32_t)wgs), dim3(256), 0, stream, p);
      else if (wgs <= 256)
        hipLaunchKernelGGL((gemm_both_kernel<T, 2, 10>), dim3((uint32_t)wgs), dim3(256), 0, stream, p);
      else
        hipLaunchKernelGGL((gemm_both_kernel<T, 2, 4>), dim3((uint32_t)wgs), dim3(256), 0, stream, p);
      if (int e = check_launch(who)) return e;
      if (int e = join<T>(who, p.dx, stream)) return e;
      return join<T>(who, p.dw, stream);
    }
  }
  if (int e = product<T, false, true>(who, rx, dx, stream)) return e;
  return product<T, true, true>(who, rw, dw, stream);
}

// (`step`: threads of the grid)
template <typename T>
__global__ void __launch_bounds__(256) zero_rows_kernel(T* y, int64_t ld, int64_t count, int n, int64_t step) {
  for (int64_t at = (int64_t)bid_x() * 256 + tid_x(); at < count; at += step) y[at / n * ld + at % n] = (T)0.f;
}

// Up to two matrices as rows of width8 (the next multiple of eight) elements with zeros behind `width`: operands whose rows
// are not 16-byte aligned. A thread moves eight elements.
struct PadParams {
  const uint16_t* from[2];
  uint16_t* to[2];
  int64_t stride[2], rows[2];
  int64_t vectors;  // of both
  int width;
};
__global__ void __launch_bounds__(256) pad_rows_kernel(const PadParams p) {
  int64_t at = (int64_t)bid_x() * 256 + tid_x();
  if (at >= p.vectors) return;
  const int groups = (p.width + 7) / 8;
  const int which = at >= p.rows[0] * groups;
  if (which) at -= p.rows[0] * groups;
  const int64_t row = at / groups;
  const int c = (int)(at - row * groups) * 8, n = p.width - c;
  const uint16_t* from = p.from[which] + row * p.stride[which] + c;
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  typedef u16x8 any __attribute__((aligned(2)));
  u16x8 v;
  if (n >= 8) {
    v = *reinterpret_cast<const any*>(from);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? from[e] : (uint16_t)0;
  }
  *reinterpret_cast<u16x8*>(p.to[which] + (row * groups) * 8 + c) = v;
}

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
static int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
static int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

static int sizes_check(const char* who, int64_t rows, int in, int out) {
  if (rows < 0 || in <= 0 || out <= 0)
    return fail(SAF3R_ERR_INVALID, "%s: invalid sizes: %lld rows, %d to %d", who, (long long)rows, in, out);
  if (in > kMaxSize || out > kMaxSize)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: widths %d and %d (at most %d)", who, in, out, kMaxSize);
  if (rows > kMaxRows) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many rows", who);
  return SAF3R_OK;
}

static int types_check(const char* who, int type, int param_type, int y_type, int act) {
  if (type != SAF3R_BF16 && type != SAF3R_FP16)
    return type == SAF3R_FP32 ? fail(SAF3R_ERR_UNSUPPORTED, "%s: operands are bf16 or fp16", who)
                              : fail(SAF3R_ERR_INVALID, "%s: unknown element type %d", who, type);
  for (int t : {param_type, y_type})
    if (t < SAF3R_FP32 || t > SAF3R_FP16) return fail(SAF3R_ERR_INVALID, "%s: unknown element type %d", who, t);
  if (y_type != SAF3R_FP32 && y_type != type)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: results of type %d: fp32 or the operands' type", who, y_type);
  if (act < SAF3R_NO_ACTIVATION || act > SAF3R_GELU_TANH)
    return fail(SAF3R_ERR_INVALID, "%s: unknown activation %d", who, act);
  return param_check(who, param_type, type);
}

// An operand of the products, and whether they read it where it lies: rows at 16-byte alignment, of a multiple of eight.
static int operand_check(const char* who, const char* name, const void* p, int64_t stride) {
  if (!p) return fail(SAF3R_ERR_INVALID, "%s: null %s", who, name);
  if ((uintptr_t)p % 2) return fail(SAF3R_ERR_INVALID, "%s: rows of %s must be aligned to their elements", who, name);
  if (stride < 0) return fail(SAF3R_ERR_INVALID, "%s: row stride %lld of %s", who, (long long)stride, name);
  return SAF3R_OK;
}
static bool in_place(const void* p, int64_t stride, int width) {
  return aligned16(p) && stride % 8 == 0 && width % 8 == 0 && stride >= width && stride <= 2 * kMaxSize;
}
// bytes of an operand's copy
static int64_t pad_bytes(int64_t rows, int width) { return round256(rows * round8(width) * 2); }

// Copies the operands that are asked for to ws, one behind the other; their pointers and strides become the copies'.
static int pad_operands(const char* who, char* ws, int width, const void** x, int64_t* x_stride, int64_t x_rows, bool pad_x,
                        const void** w, int64_t* w_stride, int64_t w_rows, bool pad_w, hipStream_t stream) {
  if (!pad_x && !pad_w) return SAF3R_OK;
  PadParams p{};
  p.width = width;
  int n = 0;
  auto add = [&](const void** t, int64_t* stride, int64_t rows) {
    p.from[n] = (const uint16_t*)*t;
    p.to[n] = (uint16_t*)ws;
    p.stride[n] = *stride;
    p.rows[n] = rows;
    p.vectors += rows * (round8(width) / 8);
    *t = ws;
    *stride = round8(width);
    ws += pad_bytes(rows, width);
    ++n;
  };
  if (pad_x) add(x, x_stride, x_rows);
  if (pad_w) add(w, w_stride, w_rows);
  const int64_t grid = (p.vectors + 255) / 256;
  if (grid > 0xffffffffll / 256) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many rows for one launch", who);
  hipLaunchKernelGGL(pad_rows_kernel, dim3((uint32_t)grid), dim3(256), 0, stream, p);
  return check_launch(who);
}

// rows of n that eight-element vectors can read or write
static bool vec_rows(const void* p, int64_t stride) { return aligned16(p) && stride % 8 == 0; }

}  // namespace saf3r

using namespace saf3r;

extern "C" int64_t saf3r_linear_fwd_workspace_bytes(int64_t rows, int in, int out, int activation, int drop, int copies) {
  const char* who = "saf3r_linear_fwd_workspace_bytes";
  if (sizes_check(who, rows, in, out)) return -1;
  if (rows == 0) return 0;
  return part_bytes(plan_of(rows, out, in, true, epilogue_cycles(activation, drop)), rows, out) +
         (copies & 1 ? pad_bytes(rows, in) : 0) + (copies & 2 ? pad_bytes(out, in) : 0);
}

extern "C" int saf3r_linear_fwd(const void* x, int64_t x_stride, const void* w, int64_t w_stride, int type, int64_t rows,
                                int in, int out, const void* bias, const void* gate, int param_type, int activation,
                                int drop, const int64_t* state, const void* residual, int64_t res_stride, void* y,
                                int64_t y_stride, int y_type, void* kept, int64_t kept_stride, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  const char* who = "saf3r_linear_fwd";
  if (int e = injected(who)) return e;
  if (int e = sizes_check(who, rows, in, out)) return e;
  if (int e = types_check(who, type, param_type, y_type, activation)) return e;
  EpiParams epi{};
  if (int e = drop_check(who, drop, state, &epi.drop)) return e;
  if (rows == 0) return SAF3R_OK;
  if (int e = operand_check(who, "x", x, x_stride)) return e;
  if (int e = operand_check(who, "w", w, w_stride)) return e;
  if (!y) return fail(SAF3R_ERR_INVALID, "%s: null y", who);
  if (int e = row_check(who, y, y_stride, out, y_type, true)) return e;
  if (kept)
    if (int e = row_check(who, kept, kept_stride, out, type, true)) return e;
  if (residual)
    if (int e = row_check(who, residual, res_stride, out, y_type, false)) return e;
  for (const void* p : {bias, gate})
    if (p)
      if (int e = row_check(who, p, 0, out, param_type, false)) return e;
  const bool pad_x = !in_place(x, x_stride, in), pad_w = !in_place(w, w_stride, in);
  const int64_t need = saf3r_linear_fwd_workspace_bytes(rows, in, out, activation, drop, pad_x + 2 * pad_w);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace))))
    return fail(SAF3R_ERR_INVALID, "%s: workspace of %lld bytes: %lld, 16-byte aligned, are needed", who,
                (long long)workspace_bytes, (long long)need);
  epi.bias = bias;
  epi.gate = gate;
  epi.res = residual;
  epi.y = y;
  epi.kept = kept;
  epi.ld_res = res_stride;
  epi.ld_y = y_stride;
  epi.ld_kept = kept_stride;
  epi.act = activation;
  epi.n = out;
  epi.param32 = param_type == SAF3R_FP32;
  epi.y32 = y_type == SAF3R_FP32;
  epi.vec = out % 8 == 0 && vec_rows(y, y_stride) && aligned16(bias) && aligned16(gate) &&
            (!kept || vec_rows(kept, kept_stride)) && (!residual || vec_rows(residual, res_stride));
  const hipStream_t s = (hipStream_t)stream;
  const Plan plan = plan_of(rows, out, in, true, epilogue_cycles(activation, drop));
  char* copies = (char*)workspace + part_bytes(plan, rows, out);
  if (int e = pad_operands(who, copies, in, &x, &x_stride, rows, pad_x, &w, &w_stride, out, pad_w, s)) return e;
  // (zeros behind `in` in both)
  const GemmParams p = params_of(plan, x, x_stride, w, w_stride, rows, out, round8(in), epi, workspace);
  return type == SAF3R_BF16 ? product<__bf16, false, false>(who, plan, p, s) : product<_Float16, false, false>(who, plan, p, s);
}

// Workspace of a backward pass: dz, the partial sums over rows, copies of x and w, the splits of dx and of dW.
struct BwdSizes {
  int64_t dz, sums, copies, dx, dw;
  int64_t all() const { return dz + sums + copies + dx + dw; }
};
static BwdSizes bwd_sizes(int64_t rows, int in, int out, bool own_dz, bool pad_x, bool pad_w) {
  BwdSizes r{};
  if (rows == 0) return r;
  r.copies = (pad_x ? pad_bytes(rows, in) : 0) + (pad_w ? pad_bytes(out, in) : 0);
  r.dz = own_dz ? round256(rows * round8(out) * 2) : 0;
  r.sums = round256(linear_grad_parts(rows, out) * 2 * out * 4);
  r.dx = round256(part_bytes(plan_of(rows, in, out, false, 0), rows, in));
  r.dw = round256(part_bytes(plan_of(out, in, rows, false, 0), out, in));
  return r;
}

extern "C" int64_t saf3r_linear_bwd_workspace_bytes(int64_t rows, int in, int out, int copies) {
  const char* who = "saf3r_linear_bwd_workspace_bytes";
  if (sizes_check(who, rows, in, out)) return -1;
  return bwd_sizes(rows, in, out, copies & 4, copies & 1, copies & 2).all();
}

extern "C" int saf3r_linear_bwd(const void* dy, int64_t dy_stride, int y_type, const void* x, int64_t x_stride,
                                const void* w, int64_t w_stride, int type, int64_t rows, int in, int out,
                                const void* kept, int64_t kept_stride, const void* gate, int param_type, int activation,
                                int drop, const int64_t* state, void* dx, int64_t dx_stride, void* dw, int64_t dw_stride,
                                int dw_type, void* dbias, void* dgate, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  const char* who = "saf3r_linear_bwd";
  if (int e = injected(who)) return e;
  if (int e = sizes_check(who, rows, in, out)) return e;
  if (int e = types_check(who, type, param_type, y_type, activation)) return e;
  if (dw_type != SAF3R_FP32 && dw_type != type)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: dweight of type %d: fp32 or the operands' type", who, dw_type);
  LinearGradParams g{};
  if (int e = drop_check(who, drop, state, &g.drop)) return e;
  const hipStream_t s = (hipStream_t)stream;
  if (dw)
    if (int e = row_check(who, dw, dw_stride, in, dw_type, true)) return e;
  const bool sums = dbias || dgate;
  if (rows > 0) {
    if (!dy) return fail(SAF3R_ERR_INVALID, "%s: null dy", who);
    if (int e = row_check(who, dy, dy_stride, out, y_type, false)) return e;
    if (dw)
      if (int e = operand_check(who, "x", x, x_stride)) return e;
    if (dx) {
      if (int e = operand_check(who, "w", w, w_stride)) return e;
      if (int e = row_check(who, dx, dx_stride, in, type, true)) return e;
    }
    if ((activation != SAF3R_NO_ACTIVATION || dgate) && !kept)
      return fail(SAF3R_ERR_INVALID, "%s: the activation and the gate need what the forward pass kept", who);
    if (kept)
      if (int e = row_check(who, kept, kept_stride, out, type, false)) return e;
    if (gate)
      if (int e = row_check(who, gate, 0, out, param_type, false)) return e;
  }
  // dy itself is the products' operand where nothing lies between
  const bool own_dz = (dx || dw) && (activation != SAF3R_NO_ACTIVATION || gate || drop || y_type != type ||
                                     !in_place(dy, dy_stride, out));
  const bool pad_x = dw && !in_place(x, x_stride, in), pad_w = dx && !in_place(w, w_stride, in);
  const BwdSizes size = bwd_sizes(rows, in, out, own_dz, pad_x, pad_w);
  const int64_t need = size.all();
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace))))
    return fail(SAF3R_ERR_INVALID, "%s: workspace of %lld bytes: %lld, 16-byte aligned, are needed", who,
                (long long)workspace_bytes, (long long)need);
  if (rows == 0) {  // (no row: gradients of zeros)
    if (dw) {
      const int64_t count = (int64_t)out * in, grid = std::min<int64_t>(4096, (count + 255) / 256);
      if (dw_type == SAF3R_FP32)
        hipLaunchKernelGGL((zero_rows_kernel<float>), dim3((uint32_t)grid), dim3(256), 0, s, (float*)dw, dw_stride, count, in,
                           grid * 256);
      else
        hipLaunchKernelGGL((zero_rows_kernel<__bf16>), dim3((uint32_t)grid), dim3(256), 0, s, (__bf16*)dw, dw_stride, count,
                           in, grid * 256);
      if (int e = check_launch(who)) return e;
    }
    return sums ? sum_parts(who, nullptr, 0, out, dgate, dbias, param_type, s) : SAF3R_OK;
  }
  char* ws = (char*)workspace;
  const void* dz = dy;
  int64_t ld_dz = dy_stride;
  if (own_dz || sums) {
    const int64_t parts = linear_grad_parts(rows, out);
    g.dy = dy;
    g.kept = activation != SAF3R_NO_ACTIVATION || dgate ? kept : nullptr;
    g.gate = gate;
    g.dz = own_dz ? ws : nullptr;
    g.part = sums ? (float*)(ws + size.dz) : nullptr;
    g.ld_dy = dy_stride;
    g.ld_kept = kept_stride;
    g.ld_dz = round8(out);
    g.rows = rows;
    g.part_rows = (rows + parts - 1) / parts;
    g.dgate = dgate;
    g.dbias = dbias;
    g.direct = parts == 1;
    g.act = activation;
    g.n = out;
    g.param32 = param_type == SAF3R_FP32;
    const bool vec = out % 8 == 0 && vec_rows(dy, dy_stride) && aligned16(gate) && (!g.kept || vec_rows(kept, kept_stride));
    if (int e = linear_grad(who, g, type, y_type == SAF3R_FP32, vec, dgate != nullptr, parts, s)) return e;
    if (sums && !g.direct)
      if (int e = sum_parts(who, g.part, parts, out, dgate, dbias, param_type, s)) return e;
    if (own_dz) {
      dz = ws;
      ld_dz = g.ld_dz;
    }
  }
  if (int e = pad_operands(who, ws + size.dz + size.sums, in, &x, &x_stride, rows, pad_x, &w, &w_stride, out, pad_w, s))
    return e;
  char* part = ws + size.dz + size.sums + size.copies;
  auto plain = [&](void* y, int64_t ld, bool y32, int n) {
    EpiParams epi{};
    epi.y = y;
    epi.ld_y = ld;
    epi.n = n;
    epi.y32 = y32;
    epi.vec = n % 8 == 0 && vec_rows(y, ld);
    return epi;
  };
  const Plan rx = plan_of(rows, in, out, false, 0), rw = plan_of(out, in, rows, false, 0);
  const GemmParams px = params_of(rx, dz, ld_dz, w, w_stride, rows, in, out, plain(dx, dx_stride, false, in), part);
  const GemmParams pw =
      params_of(rw, dz, ld_dz, x, x_stride, out, in, rows, plain(dw, dw_stride, dw_type == SAF3R_FP32, in), part + size.dx);
  auto go = [&](auto t) {
    typedef decltype(t) T;
    if (dx && dw) return both_products<T>(who, rx, px, rw, pw, s);
    if (dx) return product<T, false, true>(who, rx, px, s);
    return dw ? product<T, true, true>(who, rw, pw, s) : (int)SAF3R_OK;
  };
  return type == SAF3R_BF16 ? go(__bf16()) : go(_Float16());
}
