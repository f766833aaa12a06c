// Linear layers with their epilogue, and the products of their backward pass:
//   forward  y  = res + gate drop(act(x W^T + bias))   x [rows][in], W [out][in]
//   backward dx = dz W,  dW = dz^T x                   dz [rows][out] from linear_grad.hip
// All three are one product C[m][n] = sum_k A B whose operands lie with the reduction along a row (ROWS: x, W and dz of the
// first two) or across rows (COLS: W of the second, both of the third). bf16 or fp16 operands, fp32 sums.
//
// Bound by the matrix cores for a few hundred rows or more, by the bytes of W below.
#include "linear.h"

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
  float* part;       // splits > 1: [split][m][ldp]
  int64_t ldp;
  EpiParams epi;
};

constexpr int kUnit = 16384;        // bytes of a unit: 128 rows (or columns) x 64 of the reduction
constexpr int kSlots = 5;           // units in LDS: 80 KB, two work-groups a compute unit
constexpr int kUnitRows = 128;

// How a wave copies its quarter of a unit: four instructions of 1 KB. ROWS: instruction j of wave w takes rows 8 (4 j + w)
// .. + 7 of 128 bytes; COLS: reduction rows 4 (4 j + w) .. + 3 of 256 bytes. The 16-byte chunks of a row are swizzled by the
// row (the lanes' sources are, the LDS side of such a copy is linear).
template <bool COLS>
struct Copy {
  uint32_t off[4];  // byte offset of the lane's chunk from the unit's base
  int at;           // its place along the reduction: element (ROWS) or row (COLS, instruction 0)

  __device__ __forceinline__ void init(int wave, int lane, int first, int count, int64_t ld) {
    if constexpr (COLS) {
      const int kr = 4 * wave + (lane >> 4), chunk = (lane & 15) ^ ((kr & 3) << 2);
      // columns behind the last are the last chunk's: their results are not stored
      const int last = (count - 1) / 8 * 8 - first;
      const int c = chunk * 8 < last ? chunk * 8 : (last > 0 ? last : 0);
      at = kr;
#pragma unroll
      for (int j = 0; j < 4; ++j) off[j] = (uint32_t)((16 * j + kr) * ld + c * 2);
    } else {
      const int r = 8 * wave + (lane >> 3);
      const int chunk = (lane & 7) ^ swz8(r);
      at = chunk * 8;
      const int last = count - 1 - first > 0 ? count - 1 - first : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = r + 32 * j < last ? r + 32 * j : last;
        off[j] = (uint32_t)(row * ld + chunk * 16);
      }
    }
  }

  __device__ __forceinline__ void issue(const char* base, uint32_t lds) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) dma16s(base, off[j], lds + j * 4096);
  }

  // the last step of a reduction that 64 does not divide: `left` elements or rows are there
  __device__ __forceinline__ void issue_tail(const char* base, uint32_t lds, int left) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool there = at + (COLS ? 16 * j : 0) < left;
      dma16(there ? base + off[j] : (const char*)&kZeros, lds + j * 4096);
    }
  }
};

// Fragments of a wave's 64 rows (columns) of a unit for the 32x32x16 products: lane l holds row l % 32 of a block of 32,
// elements 16 ks + 8 (l / 32) .. + 7 of the reduction.
template <bool COLS, typename T>
struct Frags {
  typedef typename Half<T>::vec8 vec8;
  int addr[COLS ? 2 : 4];

  __device__ __forceinline__ void init(int lane, int part) {
    const int h = lane >> 5;
    if constexpr (COLS) {
      const int i = lane & 15, kr = 8 * h + (i >> 2), s = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
      for (int b = 0; b < 2; ++b)
        addr[b] = kr * 256 + ((((2 * part + b) ^ (i >> 2)) << 2) + s) * 16 + 8 * (i & 1);
    } else {
      const int r = lane & 31;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) addr[ks] = (64 * part + r) * 128 + (((2 * ks + h) ^ swz8(r)) << 4);
    }
  }

  __device__ __forceinline__ vec8 get(const char* unit, int block, int ks) const {
    if constexpr (COLS) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const char* p = unit + addr[block] + ks * 4096;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 1024));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      return __builtin_bit_cast(vec8, u32x4{x[0], x[1], y[0], y[1]});
    } else {
      return *reinterpret_cast<const vec8*>(unit + addr[ks] + block * 4096);
    }
  }
};

// Tile of a work-group: 128 UA rows by 128 columns, four waves in two rows of two; each wave owns 64 x 64 of every 128 x 128.
// Units (128 x 64 of an operand) go through a ring of five LDS slots, in the order B, A0, (A1) of every step of 64: the
// fragments of B stay in registers for the step, so its slot and A0's are free again after the first half of it. A phase is
// the 16 products of one A unit: wait for its unit, one barrier, copies into the slots that the last phase freed, LDS reads,
// products. Copies are under way for two phases. Two work-groups share a compute unit, so that one's epilogue, waits and
// barriers lie under the other's products.
template <typename T, bool ACOLS, bool BCOLS, int UA>
__global__ void __launch_bounds__(256, 2) gemm_kernel(const GemmParams p) {
  typedef typename Half<T>::vec8 vec8;
  __shared__ __attribute__((aligned(16))) char lds[kSlots * kUnit];
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6);
  const int wm = wave >> 1, wn = wave & 1;

  // Work-groups go to the eight XCDs in turn: each XCD takes a contiguous range of the tiles, which go by groups of eight
  // rows of tiles, so that the work-groups of an XCD share operand rows in its L2.
  const int tiles = p.tiles_m * p.tiles_n;
  int id = bid_x(), split = 0;
  const int all = tiles * p.splits;
  {
    const int q = all / 8, r = all % 8, x = id % 8;
    id = x * q + (x < r ? x : r) + id / 8;
  }
  if (p.splits > 1) {
    split = id / tiles;
    id -= split * tiles;
  }
  int tm, tn;
  {
    const int per = 8 * p.tiles_n, g = id / per, in = id - g * per;
    const int rows = p.tiles_m - 8 * g < 8 ? p.tiles_m - 8 * g : 8;
    tn = in / rows;
    tm = 8 * g + in - tn * rows;
  }
  const int m0 = tm * (kUnitRows * UA), n0 = tn * kUnitRows;
  const int s0 = split * p.split_steps;
  const int s1 = s0 + p.split_steps < p.steps ? s0 + p.split_steps : p.steps;
  const int left = p.k - (p.steps - 1) * 64;           // elements of the last step
  const int tail = left < 64 && s1 == p.steps ? p.steps - 1 : -1;  // the step with fewer than 64

  Copy<ACOLS> ca[UA];
  Copy<BCOLS> cb;
  const char* abase[UA];
#pragma unroll
  for (int u = 0; u < UA; ++u) {
    const int first = m0 + u * kUnitRows < p.m ? m0 + u * kUnitRows : 0;  // (a unit without a row reads the first one's)
    ca[u].init(wave, lane, first, p.m, p.lda);
    abase[u] = p.a + (ACOLS ? (int64_t)first * 2 : first * p.lda);
  }
  cb.init(wave, lane, n0, p.n, p.ldb);
  const char* bbase = p.b + (BCOLS ? (int64_t)n0 * 2 : n0 * p.ldb);
  const int64_t astep = ACOLS ? 64 * p.lda : 128, bstep = BCOLS ? 64 * p.ldb : 128;
  const uint32_t lds0 = lds_addr(lds) + wave * 1024;

  int put = 0;  // slot of the next unit that is copied
  auto copy = [&](auto which, int step) {
    constexpr int u = decltype(which)::value;  // 0: B, 1 + a: unit a of A
    const uint32_t to = lds0 + put * kUnit;
    put = put == kSlots - 1 ? 0 : put + 1;
    if constexpr (u == 0) {
      const char* base = bbase + step * bstep;
      if (step == tail)
        cb.issue_tail(base, to, left);
      else
        cb.issue(base, to);
    } else {
      const char* base = abase[u - 1] + step * astep;
      if (step == tail)
        ca[u - 1].issue_tail(base, to, left);
      else
        ca[u - 1].issue(base, to);
    }
  };

  Frags<ACOLS, T> fa;
  Frags<BCOLS, T> fb;
  fa.init(lane, wm);
  fb.init(lane, wn);
  f32x16 acc[UA][2][2];  // [unit][row block][column block]
#pragma unroll
  for (int u = 0; u < UA; ++u)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[u][i][j][e] = 0.f;

  int got = 0;  // slot of the next unit that is read
  auto next = [&]() {
    const char* r = lds + got * kUnit;
    got = got == kSlots - 1 ? 0 : got + 1;
    return r;
  };
  // LDS reads of the last phase are done before the barrier that frees their slots
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    barrier_only();
  };
  vec8 bf[2][4];
  auto phase = [&](auto which, const char* ua) {
    constexpr int u = decltype(which)::value;
    vec8 af[2][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i) af[i][ks] = fa.get(ua, i, ks);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[u][i][j] = Half<T>::mma32(bf[j][ks], af[i][ks], acc[u][i][j]);
  };
  auto read_b = [&](const char* ub) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int j = 0; j < 2; ++j) bf[j][ks] = fb.get(ub, j, ks);
  };

  copy(Int<0>(), s0);
  copy(Int<1>(), s0);
  if constexpr (UA == 2) copy(Int<2>(), s0);
  if (s0 + 1 < s1) copy(Int<0>(), s0 + 1);
#pragma unroll 1
  for (int s = s0; s < s1 - 1; ++s) {
    // (copies behind the ones that are waited for: A1 of this step and B of the next, or B of the next)
    if constexpr (UA == 2)
      wait_vm<8>();
    else
      wait_vm<4>();
    arrive();
    copy(Int<1>(), s + 1);
    if constexpr (UA == 1) {
      if (s + 2 < s1) copy(Int<0>(), s + 2);
    }
    const char* ub = next();
    const char* ua = next();
    read_b(ub);
    phase(Int<0>(), ua);
    if constexpr (UA == 2) {
      wait_vm<8>();
      arrive();
      copy(Int<2>(), s + 1);
      if (s + 2 < s1) copy(Int<0>(), s + 2);
      phase(Int<1>(), next());
    }
  }
  if constexpr (UA == 2)
    wait_vm<4>();
  else
    wait_vm<0>();
  arrive();
  {
    const char* ub = next();
    const char* ua = next();
    read_b(ub);
    phase(Int<0>(), ua);
  }
  if constexpr (UA == 2) {
    wait_vm<0>();
    arrive();
    phase(Int<1>(), next());
  }

  // A lane holds row l % 32 of a block, columns 8 q + 4 (l / 32) + e in element 4 q + e. Exchanged between the halves of the
  // wave for pairs of q, it holds eight columns in a row: 16 (q / 2) + 8 (l / 32) .. + 7.
  const int h = lane >> 5;
  DropKey key{};
  if (p.epi.drop.limit) key = drop_key(p.epi.drop);
#pragma unroll 1
  for (int blk = 0; blk < UA * 4; ++blk) {
    f32x16 x;
    switch (blk) {
      case 0: x = acc[0][0][0]; break;
      case 1: x = acc[0][0][1]; break;
      case 2: x = acc[0][1][0]; break;
      case 3: x = acc[0][1][1]; break;
      case 4: x = acc[UA - 1][0][0]; break;
      case 5: x = acc[UA - 1][0][1]; break;
      case 6: x = acc[UA - 1][1][0]; break;
      default: x = acc[UA - 1][1][1]; break;
    }
    const int row = m0 + (blk >> 2) * kUnitRows + 64 * wm + 32 * ((blk >> 1) & 1) + (lane & 31);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int col = n0 + 64 * wn + 32 * (blk & 1) + 16 * half + 8 * h;
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (as scalars first: the bits of a vector's element were taken from its first one)
        const float lo = x[8 * half + e], hi = x[8 * half + 4 + e];
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi),
                                                        false, false);
        v[e] = __builtin_bit_cast(float, (uint32_t)r[0]);
        v[4 + e] = __builtin_bit_cast(float, (uint32_t)r[1]);
      }
      if (row < p.m && col < p.n) {
        if (p.splits > 1)
          store_vec<8>(p.part + ((int64_t)split * p.m + row) * p.ldp + col, v);
        else
          epilogue8<T>(p.epi, key, row, col, v);
      }
    }
  }
}

// Few rows (16 MB at most): a work-group computes 16 columns; its eight waves take the reduction in turns of 64, straight from
// memory into the fragments of 16x16x32 products (a lane reads both halves of a 128-byte line of its row of W), and are
// joined in LDS. W is read once, by n / 16 work-groups with every load of a wave's share under way at once.
template <typename T, int MB>
__global__ void __launch_bounds__(512) few_rows_kernel(const GemmParams p) {
  typedef typename Half<T>::vec8 vec8;
  constexpr int kWaves = 8, kAhead = MB >= 4 ? 2 : 4;  // turns of a wave whose loads are under way together
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

// How a product is split: tiles of 256 or 128 rows, splits of the reduction.
struct Plan {
  bool few;
  int ua, splits, split_steps, steps, tiles_m, tiles_n;
};

static Plan plan_of(int64_t m, int n, int64_t k, bool rows_kind) {
  Plan r{};
  r.steps = (int)((k + 63) / 64);
  r.few = rows_kind && m <= 64;
  r.tiles_n = (n + 127) / 128;
  const int64_t big = (m + 255) / 256 * r.tiles_n;
  r.ua = big >= 384 ? 2 : 1;
  r.tiles_m = (int)((m + 128 * r.ua - 1) / (128 * r.ua));
  const int64_t tiles = (int64_t)r.tiles_m * r.tiles_n;
  // splits of at least four steps that fill the 512 places
  int64_t splits = tiles >= 384 ? 1 : std::min<int64_t>(512 / tiles, r.steps / 4);
  if (splits < 1) splits = 1;
  r.split_steps = (int)((r.steps + splits - 1) / splits);
  r.splits = (r.steps + r.split_steps - 1) / r.split_steps;
  return r;
}

static int64_t part_bytes(const Plan& r, int64_t m, int n) {
  return r.few || r.splits == 1 ? 0 : (int64_t)r.splits * m * ((n + 7) / 8 * 8) * 4;
}

// C = A B with the plan's kernels; `part` holds part_bytes.
template <typename T, bool ACOLS, bool BCOLS>
static int product(const char* who, const void* a, int64_t lda, const void* b, int64_t ldb, int64_t m, int n, int64_t k,
                   const EpiParams& epi, void* part, hipStream_t stream) {
  const Plan r = plan_of(m, n, k, !ACOLS && !BCOLS);
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
  if constexpr (!ACOLS && !BCOLS) {
    if (r.few) {
      const dim3 grid((uint32_t)((n + 15) / 16));
      if (m <= 16)
        hipLaunchKernelGGL((few_rows_kernel<T, 1>), grid, dim3(512), 0, stream, p);
      else if (m <= 32)
        hipLaunchKernelGGL((few_rows_kernel<T, 2>), grid, dim3(512), 0, stream, p);
      else
        hipLaunchKernelGGL((few_rows_kernel<T, 4>), grid, dim3(512), 0, stream, p);
      return check_launch(who);
    }
  }
  p.split_steps = r.split_steps;
  p.splits = r.splits;
  p.tiles_m = r.tiles_m;
  p.tiles_n = r.tiles_n;
  p.part = (float*)part;
  p.ldp = (n + 7) / 8 * 8;
  const int64_t grid = (int64_t)r.tiles_m * r.tiles_n * r.splits;
  if (grid > 0xffffffffll / 256) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many tiles for one launch", who);
  if (r.ua == 2)
    hipLaunchKernelGGL((gemm_kernel<T, ACOLS, BCOLS, 2>), dim3((uint32_t)grid), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((gemm_kernel<T, ACOLS, BCOLS, 1>), dim3((uint32_t)grid), dim3(256), 0, stream, p);
  if (int e = check_launch(who)) return e;
  if (r.splits == 1) return SAF3R_OK;
  const int64_t threads = m * (p.ldp / 8);
  hipLaunchKernelGGL((join_kernel<T>), dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, stream, p);
  return check_launch(who);
}

// (`step`: threads of the grid)
template <typename T>
__global__ void __launch_bounds__(256) zero_rows_kernel(T* y, int64_t ld, int64_t count, int n, int64_t step) {
  for (int64_t at = (int64_t)bid_x() * 256 + tid_x(); at < count; at += step) y[at / n * ld + at % n] = (T)0.f;
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

// An operand of the products: `width` elements a row, read to the next multiple of eight.
static int operand_check(const char* who, const char* name, const void* p, int64_t stride, int64_t width) {
  if (!p) return fail(SAF3R_ERR_INVALID, "%s: null %s", who, name);
  if (!aligned16(p) || stride % 8) return fail(SAF3R_ERR_INVALID, "%s: rows of %s must be 16-byte aligned", who, name);
  if (stride < round8(width) || stride > 2 * kMaxSize)
    return fail(SAF3R_ERR_INVALID, "%s: row stride %lld of %s for rows of %lld", who, (long long)stride, name,
                (long long)width);
  return SAF3R_OK;
}

// rows of n that eight-element vectors can read or write
static bool vec_rows(const void* p, int64_t stride) { return aligned16(p) && stride % 8 == 0; }

}  // namespace saf3r

using namespace saf3r;

extern "C" int64_t saf3r_linear_fwd_workspace_bytes(int64_t rows, int in, int out) {
  const char* who = "saf3r_linear_fwd_workspace_bytes";
  if (sizes_check(who, rows, in, out)) return -1;
  return rows ? part_bytes(plan_of(rows, out, in, true), rows, out) : 0;
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
  if (in % 8) return fail(SAF3R_ERR_INVALID, "%s: rows of %d: the reduction must be a multiple of 8 (pad with zeros)", who, in);
  if (int e = operand_check(who, "x", x, x_stride, in)) return e;
  if (int e = operand_check(who, "w", w, w_stride, in)) return e;
  if (!y) return fail(SAF3R_ERR_INVALID, "%s: null y", who);
  if (int e = row_check(who, y, y_stride, out, y_type, true)) return e;
  if (kept)
    if (int e = row_check(who, kept, kept_stride, out, type, true)) return e;
  if (residual)
    if (int e = row_check(who, residual, res_stride, out, y_type, false)) return e;
  for (const void* p : {bias, gate})
    if (p)
      if (int e = row_check(who, p, 0, out, param_type, false)) return e;
  const int64_t need = saf3r_linear_fwd_workspace_bytes(rows, in, out);
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
  if (type == SAF3R_BF16)
    return product<__bf16, false, false>(who, x, x_stride, w, w_stride, rows, out, in, epi, workspace, s);
  return product<_Float16, false, false>(who, x, x_stride, w, w_stride, rows, out, in, epi, workspace, s);
}

// Workspace of a backward pass: dz, the partial sums over rows, the split products (one after the other).
struct BwdSizes {
  int64_t dz, sums, products;
};
static BwdSizes bwd_sizes(int64_t rows, int in, int out, bool own_dz) {
  BwdSizes r{};
  if (rows == 0) return r;
  r.dz = own_dz ? round256(rows * round8(out) * 2) : 0;
  r.sums = round256(linear_grad_parts(rows, out) * 2 * out * 4);
  r.products = std::max(part_bytes(plan_of(rows, in, out, false), rows, in), part_bytes(plan_of(out, in, rows, false), out, in));
  return r;
}

extern "C" int64_t saf3r_linear_bwd_workspace_bytes(int64_t rows, int in, int out, int own_dz) {
  const char* who = "saf3r_linear_bwd_workspace_bytes";
  if (sizes_check(who, rows, in, out)) return -1;
  const BwdSizes r = bwd_sizes(rows, in, out, own_dz);
  return r.dz + r.sums + r.products;
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
      if (int e = operand_check(who, "x", x, x_stride, in)) return e;
    if (dx) {
      if (int e = operand_check(who, "w", w, w_stride, in)) return e;
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
  const bool own_dz = (dx || dw) && (activation != SAF3R_NO_ACTIVATION || gate || drop || y_type != type || out % 8 ||
                                     !vec_rows(dy, dy_stride) || dy_stride < out || dy_stride > 2 * kMaxSize);
  const BwdSizes size = bwd_sizes(rows, in, out, own_dz);
  const int64_t need = size.dz + size.sums + size.products;
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
    g.act = activation;
    g.n = out;
    g.param32 = param_type == SAF3R_FP32;
    const bool vec = out % 8 == 0 && vec_rows(dy, dy_stride) && aligned16(gate) && (!g.kept || vec_rows(kept, kept_stride));
    if (int e = linear_grad(who, g, type, y_type == SAF3R_FP32, vec, parts, s)) return e;
    if (sums)
      if (int e = sum_parts(who, g.part, parts, out, dgate, dbias, param_type, s)) return e;
    if (own_dz) {
      dz = ws;
      ld_dz = g.ld_dz;
    }
  }
  void* part = ws + size.dz + size.sums;
  auto plain = [&](void* y, int64_t ld, bool y32, int n) {
    EpiParams epi{};
    epi.y = y;
    epi.ld_y = ld;
    epi.n = n;
    epi.y32 = y32;
    epi.vec = n % 8 == 0 && vec_rows(y, ld);
    return epi;
  };
  auto go = [&](auto t) {
    typedef decltype(t) T;
    if (dx)
      if (int e = product<T, false, true>(who, dz, ld_dz, w, w_stride, rows, in, out, plain(dx, dx_stride, false, in), part, s))
        return e;
    if (dw)
      return product<T, true, true>(who, dz, ld_dz, x, x_stride, out, in, rows, plain(dw, dw_stride, dw_type == SAF3R_FP32, in),
                                    part, s);
    return (int)SAF3R_OK;
  };
  return type == SAF3R_BF16 ? go(__bf16()) : go(_Float16());
}
