// Attention over the tokens of frames with its backward pass (head_dim 64, bf16, fp32 sums): the training
// form of the static head patterns (dense, frame-local, anchor + local, anchor, skip). It reads q, k and v
// where the projection left them ([clip][token][head][64] with any strides) and recomputes the
// probabilities in the backward pass from the row statistics lse of the forward pass.
//
//   S = scale q k^T over the keys a query may attend, L = log sum_j exp S_j, P = exp(S - L), O = P V
//   D = sum_d dO O,  dP = dO V^T,  dS = P (dP - D),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Every pattern gives a query tile (or, in the backward pass over keys, a key tile) at most two ranges of
// consecutive tokens on the other side: all, the first frame, the own frame. A work-group owns a tile of rows and walks
// the other side in tiles of tokens read from LDS (two buffers, the next tile copied by LDS-DMA while the current one is
// used); launches of few rows share the walk among more waves (see the modes below). Matrix products are
// v_mfma_f32_32x32x16_bf16 and none of their results crosses lanes: a product whose rows are summed over next (P, dS)
// leaves its 32x32 result with one column per lane and the rows 8 (i / 4) + 4 (lane / 32) + i % 4, and the other operand
// of the next product is read from LDS with the transposing read in that same row order (two groups of four rows per 16).
//
// The probabilities and dS are rounded to bf16 as operands of the second product, which is what the matrix
// cores take; everything else (S, dP, the statistics, all sums) is fp32.
//
// Backward without atomics: one kernel per side. The first owns query rows, computes D and dQ; the second owns
// key rows and computes dK and dV. Both recompute S and dP (7 products in place of 5), and the results do not
// depend on the order in which work-groups run.
//
// D cancels against dP, so an O that is rounded to bf16 would leave an error of its own in every dS of a row; the
// forward pass can store what the rounding of O took away (rest, bf16) for the sum that gives D.
//
// Tokens that the mask removes are no keys and their own rows come out as zeros (lse = -inf); their q, k, v and
// dO rows are replaced by zeros where they enter a product, so that whatever they hold stays out.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace saf3r {

template <int N>
using Int = std::integral_constant<int, N>;

// How the waves of a work-group share its rows and its walk (MODE):
//   kTogether: four waves, 32 rows each, walk together; a tile is 64 tokens, staged for all of them in two buffers;
//   kPairs:    two such groups of four waves own the same 128 rows, each walks every other tile (64 KB of buffers);
//   4 or 8:    so many waves own the same 32 rows, and each walks its share of tiles of 32 tokens in two buffers of its own
//              (64 or 128 KB).
// What the groups or waves found is joined at the end.
constexpr int kTile = 64;
constexpr int kTileElems = kTile * kHeadDim;
constexpr int kTogether = 0, kPairs = 2;
template <int MODE>
constexpr bool kAlone = MODE > kPairs;
template <int MODE>
constexpr int kTokens = kAlone<MODE> ? 32 : kTile;
template <int MODE>
constexpr int kThreads = kAlone<MODE> ? 64 * MODE : MODE == kPairs ? 512 : 256;
template <int MODE>
constexpr int kRows = kAlone<MODE> ? 32 : 128;  // of a work-group
template <int MODE>
constexpr int kBuffers = kAlone<MODE> ? 2 * MODE : MODE == kPairs ? 4 : 2;
constexpr int kFaClasses = 7;      // kinds of row tiles of a launch, see make_classes
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

enum Walk { kNone = 0, kAll = 1, kFirst = 2, kOwn = 3, kFirstOwn = 4 };

// Row tiles that walk alike: of the heads of a mask, head by head and clip by clip; per frame (from token tok0 on) or
// over the tokens tok0 .. tok1.
struct FaClass {
  int start;     // first work-group
  int per_clip;  // tiles of a clip of a head
  int nt;        // tiles of a frame (per-frame runs; 0: over tokens)
  int tok0, tok1;
  int walk;
  uint64_t heads;
};

struct FaTensor {
  __bf16* ptr;
  int64_t clip, token, head;  // strides in elements
};

struct FaParams {
  FaTensor q, k, v, o, rest, doo, dq, dk, dv;
  float* lse;            // [clip][head][token]
  float* delta;          // [clip][head][token]
  const uint8_t* mask;   // [clip][token], 0: not there (may be null)
  int N, T, H, clips;
  int wide;              // rows of a walk tile need 64-bit offsets
  float scale, c;        // softmax scale, scale * log2(e)
  FaClass cls[kFaClasses];
};

// What a work-group owns and walks.
struct FaItem {
  int head, clip;
  int row0, row_end;    // own rows: row0 .. min(row0 + tile, row_end)
  int a0, a1, b0, b1;   // walked ranges
};

// (The kernel's arguments lie in host memory, where a load that depends on another costs microseconds: all classes are
// read at once and chosen from in registers.)
__device__ inline FaItem fa_item(const FaParams& p, int rows) {
  const int bid = bid_x();
  FaClass s = p.cls[0];
#pragma unroll
  for (int i = 1; i < kFaClasses; ++i) {
    const FaClass x = p.cls[i];
    const bool in = x.start <= bid;  // (classes without tiles start behind every work-group)
    s.start = in ? x.start : s.start;
    s.per_clip = in ? x.per_clip : s.per_clip;
    s.nt = in ? x.nt : s.nt;
    s.tok0 = in ? x.tok0 : s.tok0;
    s.tok1 = in ? x.tok1 : s.tok1;
    s.walk = in ? x.walk : s.walk;
    s.heads = in ? x.heads : s.heads;
  }
  // Work-groups go to the eight XCDs in turn: eight runs (a head of a clip) side by side, so that a run's rows are read
  // through one L2. What eight do not divide comes behind. (60 clips of 120 tokens, 16 heads, forward / dQ / dK and dV: 22 /
  // 29 / 32 us, run by run 26 / 31 / 34; 8192 tokens: the same.)
  const int j = bid - s.start, even = (__builtin_popcountll(s.heads) * p.clips & ~7) * s.per_clip;
  const bool in_turn = j < even;
  const int k = in_turn ? j >> 3 : j - even, nth_run = k / s.per_clip, t = k - nth_run * s.per_clip;
  const int run = in_turn ? 8 * nth_run + (j & 7) : even / s.per_clip + nth_run;
  FaItem it;
  const int nth = run / p.clips;
  it.clip = run - nth * p.clips;
  uint64_t left = s.heads;  // the nth head of the mask
  for (int i = 0; i < nth; ++i) left &= left - 1;
  it.head = __builtin_ctzll(left);
  int frame0 = 0;
  if (s.nt > 0) {
    const int f = t / s.nt;
    frame0 = s.tok0 + f * p.T;
    it.row0 = frame0 + (t - f * s.nt) * rows;
    it.row_end = frame0 + p.T;
  } else {
    it.row0 = s.tok0 + t * rows;
    it.row_end = s.tok1;
  }
  it.a0 = it.a1 = it.b0 = it.b1 = 0;
  switch (s.walk) {
    case kAll: it.a1 = p.N; break;
    case kFirst: it.a1 = p.T; break;
    case kOwn: it.a0 = frame0; it.a1 = frame0 + p.T; break;
    case kFirstOwn:
      it.a1 = p.T;
      if (frame0 > 0) { it.b0 = frame0; it.b1 = frame0 + p.T; }
      break;
    default: break;
  }
  return it;
}

template <int TOKENS>
__host__ __device__ inline int tiles_of(int n) {
  return (n + TOKENS - 1) / TOKENS;
}

// Position of walk tile i: tokens start .. end of it (at most TOKENS).
template <int TOKENS>
__device__ inline void walk_tile(const FaItem& it, int na, int i, int* start, int* end) {
  if (i < na) {
    *start = it.a0 + i * TOKENS;
    *end = it.a1;
  } else {
    *start = it.b0 + (i - na) * TOKENS;
    *end = it.b1;
  }
}

// Chunk swizzle of the tiles (16-byte chunks of 128-byte rows, XOR with a function of the row). LDS serves 256 bytes a
// cycle: 16 lanes of a rows operand (16 rows, one chunk) and 32 lanes of a transposed one (4 rows, 4 chunks) fall on
// 64 different banks when the eight rows of one parity take eight values and rows two apart differ in bit 2. (With
// swz8, whose rows two apart stay in one half row, the transposed reads took twice their cycles.)
__device__ inline int swz_tile(int r) { return ((r & 2) << 1) | ((r >> 2) & 3); }

// LDS addresses of a lane's operand fragments in a [64][64] tile whose 16-byte chunks are swizzled by row.
struct FragAddr {
  int row[4];     // rows operand: row lane % 32, elements 16 ks + 8 (lane / 32) .. + 7
  int tr[2][2];   // transposed operand: [32-column half][row group 0 / 8], see tr_frag
};

__device__ inline FragAddr frag_addr(int lane) {
  FragAddr f;
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) f.row[ks] = r * 64 + (((2 * ks + h) ^ swz_tile(r)) << 3);
  // lane i of 16 addresses row i / 4, columns 4 (i % 4) .. + 3, and receives column i of those 4 x 16 elements
  const int tr = 4 * h + ((lane & 15) >> 2), cc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
  for (int dh = 0; dh < 2; ++dh)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int row = tr + 8 * g;
      f.tr[dh][g] = row * 64 + (((4 * dh + cc) ^ swz_tile(row)) << 3) + 4 * (lane & 1);
    }
  return f;
}

typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Rows operand: rows 32 half .. + 31 of the tile, k-step ks.
__device__ __forceinline__ bf16x8 row_frag(const __bf16* tile, const FragAddr& f, int half, int ks) {
  return *reinterpret_cast<const bf16x8*>(tile + half * 2048 + f.row[ks]);
}

// Transposed operand: columns 32 dh + lane % 32 of rows 16 step + {4 h .. 4 h + 3, 8 + 4 h ..} (h = lane / 32),
// the order in which a 32x32 product leaves its rows in a lane.
__device__ __forceinline__ bf16x8 tr_frag(const __bf16* tile, const FragAddr& f, int step, int dh) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + step * 1024 + f.tr[dh][0]));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + step * 1024 + f.tr[dh][1]));
  const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
  return __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
}

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Eight accumulator elements 8 st .. 8 st + 7 as a bf16 operand.
__device__ __forceinline__ bf16x8 pack8(const f32x16& x, int st) {
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (__bf16)x[8 * st + j];
  return r;
}

__device__ __forceinline__ float pair_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float pair_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Copies the rows of a walk tile of two tensors to LDS (LDS-DMA, no registers): a lane takes 16 bytes, swizzled by the
// choice of its source; a wave takes 16 rows of each tensor, or all 32 where it walks alone. Rows behind the range are
// copies of its last row: finite where the range is, and given probability zero by the caller. Whole tiles take a
// scalar base and the lane's own offsets, which fit 32 bits (`wide` where they do not); the last tile of a range takes an
// address a lane.
struct Stager {
  const __bf16 *x, *y;
  int64_t xs, ys;
  uint32_t xo[2], yo[2];  // byte offsets of the lane's two rows in 16
  int lane, row0;
  bool wide;
};

template <int MODE>
__device__ __forceinline__ Stager stager(const __bf16* x, int64_t xs, const __bf16* y, int64_t ys, bool wide, int wave,
                                         int lane) {
  Stager s;
  s.wide = wide;
  s.x = x;
  s.y = y;
  s.xs = xs;
  s.ys = ys;
  s.lane = lane;
  s.row0 = kAlone<MODE> ? 0 : (wave & 3) * 16;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = 8 * i + (lane >> 3), c = ((lane & 7) ^ swz_tile(row)) << 3;
    s.xo[i] = (uint32_t)(((s.row0 + row) * xs + c) * 2);
    s.yo[i] = (uint32_t)(((s.row0 + row) * ys + c) * 2);
  }
  return s;
}

template <int MODE>
__device__ __forceinline__ void stage(const Stager& s, int start, int end, const __bf16* xt, const __bf16* yt) {
  const uint32_t xl = lds_addr(xt) + s.row0 * 128, yl = lds_addr(yt) + s.row0 * 128;
  const bool whole = start + kTokens<MODE> <= end && !s.wide;
#pragma unroll
  for (int k = 0; k < (kAlone<MODE> ? 2 : 1); ++k) {
    if (whole) {
      const __bf16 *xb = s.x + (start + 16 * k) * s.xs, *yb = s.y + (start + 16 * k) * s.ys;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        dma16s(xb, s.xo[i], xl + k * 2048 + i * 1024);
        dma16s(yb, s.yo[i], yl + k * 2048 + i * 1024);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 8 * i + (s.lane >> 3), c = ((s.lane & 7) ^ swz_tile(row)) << 3;
        const int tok = min(start + s.row0 + 16 * k + row, end - 1);
        dma16(s.x + tok * s.xs + c, xl + k * 2048 + i * 1024);
        dma16(s.y + tok * s.ys + c, yl + k * 2048 + i * 1024);
      }
    }
  }
}

// Every LDS access of the wave is done.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Bits of a whole tile.
template <int MODE>
constexpr uint64_t kAllRows = kAlone<MODE> ? 0xFFFFFFFFull : ~0ull;

// Rows that are not there (bits) become zeros, so that what they hold stays out of every product. A wave clears what it
// copied itself.
template <int MODE>
__device__ __forceinline__ void clear_rows(const Stager& s, __bf16* xt, __bf16* yt, uint64_t bits) {
  if (bits == kAllRows<MODE>) return;
#pragma unroll
  for (int i = 0; i < (kAlone<MODE> ? 4 : 2); ++i) {
    const int row = s.row0 + i * 8 + (s.lane >> 3);
    if (!((bits >> row) & 1)) {
      *reinterpret_cast<u32x4*>(xt + row * 64 + (s.lane & 7) * 8) = u32x4{};
      *reinterpret_cast<u32x4*>(yt + row * 64 + (s.lane & 7) * 8) = u32x4{};
    }
  }
}

// The tiles of a walk that hold a token which is there, in order. Whether 64 tiles hold one is found at once, a tile a lane
// (a tile that its range cuts off counts without a look).
template <bool MASK, int MODE>
struct Tiles {
  const FaItem& it;
  const uint8_t* mask;
  int na, nw, base;
  uint64_t some;  // of the tiles base .. base + 63

  __device__ Tiles(const FaItem& item, const uint8_t* m) : it(item), mask(m), base(0), some(0) {
    na = tiles_of<kTokens<MODE>>(it.a1 - it.a0);
    nw = na + tiles_of<kTokens<MODE>>(it.b1 - it.b0);
    if constexpr (MASK) look(0);
  }

  __device__ void look(int first) {
    base = first;
    const int i = first + (int)(tid_x() & 63);
    bool any = false;
    if (i < nw) {
      int start, end;
      walk_tile<kTokens<MODE>>(it, na, i, &start, &end);
      any = start + kTokens<MODE> > end;
      if (!any) {
        typedef u32x4 bytes __attribute__((aligned(1)));
        u32x4 x{};
#pragma unroll
        for (int c = 0; c < kTokens<MODE>; c += 16) x |= *reinterpret_cast<const bytes*>(mask + start + c);
        any = (x[0] | x[1] | x[2] | x[3]) != 0;
      }
    }
    some = __ballot(any);
  }

  // The n-th tile behind tile i that holds one, nw behind the last.
  __device__ int after(int i, int n) {
    if constexpr (!MASK) return min(i + n, nw);
    while (true) {
      const int at = i + 1 - base;
      const uint64_t left = at < 64 ? some >> at : 0;
      if (left) {
        i += 1 + __builtin_ctzll(left);
        if (--n == 0) return i;
      } else {
        i = base + 63;
        if (i + 1 >= nw) return nw;
        look(i + 1);
      }
    }
  }
};

// The walk of a work-group over its ranges. Together: the four waves of a group use each of its tiles, staged in two buffers with
// one barrier a tile. Alone: wave w of n takes the tiles w, w + n, ... (of those that hold a token) in two buffers of its own,
// without barriers; the callers add up what the waves found. load(start, end) -> the lane's share of what belongs to a tile,
// bits(share) -> the rows that are there, publish(share, buffer) before and tile(buffer, bits) with the rows in LDS.
// rows() reads the own rows, once the first tiles are on their way.
template <bool MASK, int MODE, typename Rows, typename Load, typename Bits, typename Publish, typename Tile>
__device__ __forceinline__ void walk(const FaItem& it, const Stager& st, const uint8_t* mask,
                                     __bf16 (*lds)[2][kTokens<MODE> * kHeadDim], int wave, bool active, Rows rows,
                                     Load load, Bits bits, Publish publish, Tile tile) {
  constexpr int kN = kTokens<MODE>;
  if constexpr (MASK)
    if (!__syncthreads_or(active)) return;  // no row of its own: nothing to walk for
  Tiles<MASK, MODE> tiles(it, mask);
  const int nw = tiles.nw;
  auto fetch = [&](int i, int buf) {
    int start, end;
    walk_tile<kN>(it, tiles.na, i, &start, &end);
    end = min(end, start + kN);
    const auto share = load(start, end);
    stage<MODE>(st, start, end, lds[buf][0], lds[buf][1]);
    return share;
  };
  if constexpr (kAlone<MODE>) {
    if (!active) return;
    int i = tiles.after(-1, wave + 1);
    if (i >= nw) return;
    int buf = 2 * wave, behind = tiles.after(i, MODE);
    auto now = fetch(i, buf), next = now;
    if (behind < nw) next = fetch(behind, buf + 1);
    rows();
    while (true) {
      if (behind < nw)
        wait_vm<8>();  // all but the next tile's copies
      else
        wait_vm<0>();
      const uint64_t there = bits(now);
      if constexpr (MASK) clear_rows<MODE>(st, lds[buf][0], lds[buf][1], there);
      publish(now, buf);
      if (there) tile(buf, there);
      i = behind;
      if (i >= nw) return;
      behind = tiles.after(i, MODE);
      now = next;
      wait_lds();  // this tile's reads, before its buffer is filled again
      if (behind < nw) next = fetch(behind, buf);
      buf ^= 1;
    }
  } else if constexpr (!MASK) {  // (every tile: the same loop with less to decide, 150 us in place of 175 in dK and dV)
    if (nw == 0) return;
    constexpr int kGroups = MODE == kPairs ? 2 : 1;
    const int group = wave >> 2, buf0 = 2 * group;
    auto now = fetch(min(group, nw - 1), buf0);
    rows();
    for (int i = group, step = 0; step * kGroups < nw; i += kGroups, ++step) {
      const int buf = buf0 + (step & 1);
      const uint64_t there = bits(now);
      wait_vm<0>();
      if ((wave & 3) == 0) publish(now, buf);
      __syncthreads();
      if (i + kGroups < nw) now = fetch(i + kGroups, buf ^ 1);
      if (active && there && i < nw) tile(buf, there);
    }
  } else {
    // first: the tile of the first group, own: of the wave's group (all groups step alike, to the last barrier)
    int first = tiles.after(-1, 1), last = MODE == kPairs ? tiles.after(first, 1) : first;
    if (first >= nw) return;
    const int group = MODE == kPairs ? wave >> 2 : 0;
    int own = group ? last : first;
    const int buf0 = 2 * group;
    auto now = fetch(min(own, nw - 1), buf0);
    rows();
    for (int step = 0; first < nw; ++step) {
      const int buf = buf0 + (step & 1);
      const bool has = MODE != kPairs || own < nw;
      const uint64_t there = bits(now);
      wait_vm<0>();
      clear_rows<MODE>(st, lds[buf][0], lds[buf][1], there);
      if ((wave & 3) == 0) publish(now, buf);
      __syncthreads();
      first = tiles.after(last, 1);
      last = MODE == kPairs ? tiles.after(first, 1) : first;
      own = group ? last : first;
      if (own < nw) now = fetch(own, buf ^ 1);
      if (active && there && has) tile(buf, there);  // (a tile without a row changes nothing)
    }
  }
}

// kPairs: the second group leaves what it found for the first, which adds it up: N values a lane, at x + 64 n.
__device__ __forceinline__ float* pair_slot(void* lds, int wave, int lane, int n) {
  return reinterpret_cast<float*>(lds) + (wave & 3) * n * 64 + lane;
}
__device__ __forceinline__ void put_sums(float* at, const f32x16& x) {
#pragma unroll
  for (int j = 0; j < 16; ++j) at[64 * j] = x[j];
}
__device__ __forceinline__ void add_sums(const float* at, f32x16& x, float own = 1.f, float other = 1.f) {
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = x[j] * own + at[64 * j] * other;
}

// What the waves of a work-group that walked alone have to add up: a 64 x 32 result (rows 32 dh + 8 (j / 4) + 4 h + j % 4
// of lane % 32's column) a wave, in LDS rows of 33.
constexpr int kPart = 64 * 33;
static_assert(4 * 64 * 64 * 4 <= kBuffers<kPairs> * 2 * kTileElems * 2, "the second group's sums in the buffers");
static_assert((kPart + 64) * 4 <= 2 * 2 * kTokens<4> * kHeadDim * 2, "a wave's part in its buffers");
__device__ __forceinline__ void put_part(float* part, const f32x16 (&x)[2], int lane) {
#pragma unroll
  for (int dh = 0; dh < 2; ++dh)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      part[(32 * dh + 8 * (j / 4) + 4 * (lane >> 5) + j % 4) * 33 + (lane & 31)] = x[dh][j];
}

// Joining: a thread of a work-group takes column tid % 32 and this many consecutive rows.
template <int MODE>
constexpr int kJoin = 64 * 32 / kThreads<MODE>;

// The sum of a part's element over the waves, pairs first.
template <int MODE>
__device__ __forceinline__ float sum_waves(const float* x) {
  float y = (x[0] + x[kPart]) + (x[2 * kPart] + x[3 * kPart]);
  if constexpr (MODE == 8) y += (x[4 * kPart] + x[5 * kPart]) + (x[6 * kPart] + x[7 * kPart]);
  return y;
}

template <int N>
__device__ __forceinline__ void store_row(__bf16* at, const float (&x)[N]) {
  typedef __bf16 vec __attribute__((ext_vector_type(N)));
  vec v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (__bf16)x[e];
  *reinterpret_cast<vec*>(at) = v;
}

// A token of the mask (1 where there is none), or whether it lies in the range at all.
template <bool MASK>
__device__ __forceinline__ uint8_t mask_byte(const uint8_t* mask, int start, int end) {
  const int tok = start + (tid_x() & 63);
  if (!MASK) return tok < end;
  return tok < end ? mask[tok] : 0;
}

// Sets the scores of keys that are not there to -inf; half: keys 32 half .. + 31 of the tile.
__device__ __forceinline__ void mask_scores(f32x16& s, uint64_t bits, int half, int h) {
  const uint32_t w = (uint32_t)(bits >> (32 * half)) >> (4 * h);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!((w >> (8 * (i / 4) + i % 4)) & 1)) s[i] = -__builtin_inff();
}

// ---------------------------------------------------------------------------------------
// Forward: a wave owns 32 query rows as columns of S^T = K Q^T; O^T += V^T P^T.
// The running reference m of a row is the maximum of its first tile; it moves only when a tile's sum of
// exp2(S c - m) leaves [0, 2^40], so that tiles after the first take no maximum (fp32 holds the sums, and
// bf16 the probabilities, at the same relative precision for any m at or below the row's maximum).
//
// A wave owns 32 rows and three waves share a SIMD. (64 rows a wave, two waves: the same rate over long walks, 1.4
// times the time over 522 tokens.) The modes that share a walk join their sums at the end.
//
// Bound by the issue of vector instructions: fma, exponential, add and half a conversion an element against 16 matrix
// products a tile (vector pipe busy 58% of the time, matrix pipe 41%, seldom both). 12 frames of 1374 tokens, 10 of 16 heads dense: 870 us, 849 TFLOP/s of the pairs (1357 is what a
// large matrix product reaches here); 8 x 1374 frames 101 us; 522 tokens 11 us.
// ---------------------------------------------------------------------------------------
template <bool MASK, int MODE>
__global__ void __launch_bounds__(kThreads<MODE>, MODE == kTogether ? 3 : 2) frame_attn_fwd_kernel(const FaParams p) {
  __shared__ __align__(16) __bf16 lds[kBuffers<MODE>][2][kTokens<MODE> * kHeadDim];
  constexpr int kH = kTokens<MODE> / 32;
  const FaItem it = fa_item(p, kRows<MODE>);
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6), h = lane >> 5;
  const FragAddr fa = frag_addr(lane);
  const uint8_t* mask = MASK ? p.mask + (int64_t)it.clip * p.N : nullptr;
  const int first = it.row0 + (kAlone<MODE> ? 0 : (wave & 3) * 32), r = first + (lane & 31);
  const bool valid = r < it.row_end && (!MASK || mask[r]), active = __any(valid);

  bf16x8 qf[4];
  const __bf16* qp = p.q.ptr + it.clip * p.q.clip + it.head * p.q.head + r * p.q.token + 8 * h;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) qf[ks] = valid ? *reinterpret_cast<const bf16x8*>(qp + 16 * ks) : bf16x8{};
  f32x16 o[2] = {};
  float m = -__builtin_inff(), l = 0.f;

  const Stager st = stager<MODE>(p.k.ptr + it.clip * p.k.clip + it.head * p.k.head, p.k.token,
                                  p.v.ptr + it.clip * p.v.clip + it.head * p.v.head, p.v.token, p.wide, wave, lane);
  walk<MASK, MODE>(
      it, st, mask, lds, wave, active, [] {},
      [&](int start, int end) { return mask_byte<MASK>(mask, start, end); },
      [](uint8_t b) { return __ballot(b != 0); }, [](uint8_t, int) {},
      [&](int buf, uint64_t bits) {
        const __bf16 *kt = lds[buf][0], *vt = lds[buf][1];
        f32x16 s[kH], e[kH];
#pragma unroll
        for (int kh = 0; kh < kH; ++kh)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) s[kh] = mma(row_frag(kt, fa, kh, ks), qf[ks], ks ? s[kh] : f32x16{});
        if (bits != kAllRows<MODE>) {
#pragma unroll
          for (int kh = 0; kh < kH; ++kh) mask_scores(s[kh], bits, kh, h);
        }
        float sum = 0.f;
        bool moved = m == -__builtin_inff();
        if (!__any(moved)) {
#pragma unroll
          for (int kh = 0; kh < kH; ++kh)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              e[kh][j] = __builtin_amdgcn_exp2f(s[kh][j] * p.c - m);
              sum += e[kh][j];
            }
          moved = !(sum <= 0x1p40f);
        }
        if (__any(moved)) {
          float mx = -__builtin_inff();
#pragma unroll
          for (int kh = 0; kh < kH; ++kh)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[kh][j]);
          const float next = fmaxf(m, pair_max(mx) * p.c);
          const float base = next == -__builtin_inff() ? 0.f : next;  // no key yet
          const float f = __builtin_amdgcn_exp2f(m - base);
          l *= f;
#pragma unroll
          for (int dh = 0; dh < 2; ++dh)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[dh][j] *= f;
          m = next;
          sum = 0.f;
#pragma unroll
          for (int kh = 0; kh < kH; ++kh)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              e[kh][j] = __builtin_amdgcn_exp2f(s[kh][j] * p.c - base);
              sum += e[kh][j];
            }
        }
        l += sum;
#pragma unroll
        for (int step = 0; step < 2 * kH; ++step) {
          const bf16x8 pf = pack8(e[step / 2], step % 2);
#pragma unroll
          for (int dh = 0; dh < 2; ++dh) o[dh] = mma(tr_frag(vt, fa, step, dh), pf, o[dh]);
        }
      });

  if constexpr (MODE == kPairs) {
    float* at = pair_slot(lds, wave, lane, 34);
    __syncthreads();
    if (wave >= 4) {
      put_sums(at, o[0]);
      put_sums(at + 64 * 16, o[1]);
      at[64 * 32] = m;
      at[64 * 33] = l;
    }
    __syncthreads();
    if (wave >= 4) return;
    const float other = at[64 * 32], top = fmaxf(m, other), base = top == -__builtin_inff() ? 0.f : top;
    const float fm = __builtin_amdgcn_exp2f(m - base), fo = __builtin_amdgcn_exp2f(other - base);
    add_sums(at, o[0], fm, fo);
    add_sums(at + 64 * 16, o[1], fm, fo);
    l = l * fm + at[64 * 33] * fo;
    m = top;
  }
  const float sum = pair_sum(l);
  const int64_t stat = ((int64_t)it.clip * p.H + it.head) * p.N;
  __bf16* op = p.o.ptr + it.clip * p.o.clip + it.head * p.o.head;
  __bf16* rp = p.rest.ptr + it.clip * p.rest.clip + it.head * p.rest.head;
  if constexpr (kAlone<MODE>) {
    // joined: the largest reference, every wave's sums on its scale
    float* part = reinterpret_cast<float*>(lds);
    __syncthreads();
    put_part(part + wave * (kPart + 64), o, lane);
    if (h == 0) {
      part[wave * (kPart + 64) + kPart + lane] = m;
      part[wave * (kPart + 64) + kPart + 32 + lane] = sum;
    }
    __syncthreads();
    constexpr int kN = kJoin<MODE>;
    const int col = tid_x() & 31, d0 = (tid_x() >> 5) * kN, row = it.row0 + col;
    if (row >= it.row_end) return;
    float mw[MODE], top = -__builtin_inff(), total = 0.f;
#pragma unroll
    for (int w = 0; w < MODE; ++w) {
      mw[w] = part[w * (kPart + 64) + kPart + col];
      top = fmaxf(top, mw[w]);
    }
    const bool some = (!MASK || mask[row]) && top != -__builtin_inff();
    float y[kN] = {}, x[kN];
#pragma unroll
    for (int w = 0; w < MODE; ++w) {
      const float f = some ? __builtin_amdgcn_exp2f(mw[w] - top) : 0.f;
      total += f * part[w * (kPart + 64) + kPart + 32 + col];
#pragma unroll
      for (int e = 0; e < kN; ++e) y[e] += f * part[w * (kPart + 64) + (d0 + e) * 33 + col];
    }
    const float inv = some ? 1.f / total : 0.f;
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      y[e] = some ? y[e] * inv : 0.f;
      x[e] = y[e] - (float)(__bf16)y[e];
    }
    store_row(op + row * p.o.token + d0, y);
    if (p.rest.ptr) store_row(rp + row * p.rest.token + d0, x);
    if (d0 == 0) p.lse[stat + row] = some ? (top + __builtin_amdgcn_logf(total)) * kLn2 : -__builtin_inff();
  } else {
    if (r >= it.row_end) return;
    const bool some = valid && m != -__builtin_inff();
    const float inv = some ? 1.f / sum : 0.f;
    op += r * p.o.token + 4 * h;
    rp += r * p.rest.token + 4 * h;
#pragma unroll
    for (int dh = 0; dh < 2; ++dh)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __bf16 w[4], x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = some ? o[dh][4 * j + e] * inv : 0.f;
          w[e] = (__bf16)y;
          x[e] = (__bf16)(y - (float)w[e]);
        }
        *reinterpret_cast<u32x2*>(op + 32 * dh + 8 * j) = *reinterpret_cast<u32x2*>(w);
        if (p.rest.ptr) *reinterpret_cast<u32x2*>(rp + 32 * dh + 8 * j) = *reinterpret_cast<u32x2*>(x);
      }
    if (h == 0) p.lse[stat + r] = some ? (m + __builtin_amdgcn_logf(sum)) * kLn2 : -__builtin_inff();
  }
}

// ---------------------------------------------------------------------------------------
// Backward over queries: D and dQ. A wave owns 32 query rows as columns of S^T and dP^T = V dO^T;
// dQ^T += K^T dS^T.
// The sums of dP start at -D. Three waves a SIMD (64 rows a wave and two waves: the same rate).
//
// Matrix and vector pipes are about equally busy, 51% each and seldom both (24 products a tile against fma, exponential,
// product and half a conversion an element): 12 frames of 1374, 10 of 16 heads dense 1120 us, 990 TFLOP/s; 8 x 1374 frames 120 us.
//
// The dS of a row add up to zero, so that what its keys have in common cancels in dQ, and the roundings of dS do not: over
// a few keys that are alike dQ loses another bit. Short walks add what the rounding took away (a third more products: 5% of
// the time over 60 x 120 tokens, 30% over 8 x 1374; waves that walk alone wait for memory anyway, 3% over 256 tokens). What
// is short goes by the mode, and the mode by the whole launch: dQ of a clip of 129 to 512 tokens is finer in a launch of few
// rows than in one of many.
// ---------------------------------------------------------------------------------------
template <int MODE>
constexpr int kFineUpTo = kAlone<MODE> ? 512 : 128;

template <bool MASK, int MODE>
__global__ void __launch_bounds__(kThreads<MODE>, MODE == kTogether ? 3 : 2) frame_attn_dq_kernel(const FaParams p) {
  __shared__ __align__(16) __bf16 lds[kBuffers<MODE>][2][kTokens<MODE> * kHeadDim];
  const FaItem it = fa_item(p, kRows<MODE>);
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6), h = lane >> 5;
  const FragAddr fa = frag_addr(lane);
  const uint8_t* mask = MASK ? p.mask + (int64_t)it.clip * p.N : nullptr;
  const int64_t stat = ((int64_t)it.clip * p.H + it.head) * p.N;
  const int first = it.row0 + (kAlone<MODE> ? 0 : (wave & 3) * 32), r = first + (lane & 31);
  const bool active = __any(r < it.row_end && (!MASK || mask[r]));

  bf16x8 qf[4], dof[4];
  float lse2 = __builtin_inff();  // rows without a key, or not there: probabilities of zero
  f32x16 dq[2] = {}, from;        // from: where the sums of dP start
  auto rows = [&] {
    float ls = -__builtin_inff(), d = 0.f;
    bf16x8 of[4] = {}, rf[4] = {};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qf[ks] = dof[ks] = bf16x8{};
    if (r < it.row_end) {
      const __bf16* qp = p.q.ptr + it.clip * p.q.clip + it.head * p.q.head + r * p.q.token + 8 * h;
      const __bf16* dp = p.doo.ptr + it.clip * p.doo.clip + it.head * p.doo.head + r * p.doo.token + 8 * h;
      const __bf16* op = p.o.ptr + it.clip * p.o.clip + it.head * p.o.head + r * p.o.token + 8 * h;
      ls = p.lse[stat + r];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
        dof[ks] = *reinterpret_cast<const bf16x8*>(dp + 16 * ks);
        of[ks] = *reinterpret_cast<const bf16x8*>(op + 16 * ks);
      }
      if (p.rest.ptr) {
        const __bf16* rp = p.rest.ptr + it.clip * p.rest.clip + it.head * p.rest.head + r * p.rest.token + 8 * h;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) rf[ks] = *reinterpret_cast<const bf16x8*>(rp + 16 * ks);
      }
    }
    const bool valid = ls != -__builtin_inff();
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      qf[ks] = valid ? qf[ks] : bf16x8{};
      dof[ks] = valid ? dof[ks] : bf16x8{};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        d += (float)dof[ks][j] * (float)of[ks][j];
        d += (float)dof[ks][j] * (float)rf[ks][j];
      }
    }
    d = valid ? pair_sum(d) : 0.f;
    if (h == 0 && r < it.row_end && wave < kRows<MODE> / 32) p.delta[stat + r] = d;
    if (valid) lse2 = ls * kLog2e;
#pragma unroll
    for (int j = 0; j < 16; ++j) from[j] = -d;
  };

  const bool fine = it.a1 - it.a0 + it.b1 - it.b0 <= kFineUpTo<MODE>;
  const Stager st = stager<MODE>(p.k.ptr + it.clip * p.k.clip + it.head * p.k.head, p.k.token,
                                  p.v.ptr + it.clip * p.v.clip + it.head * p.v.head, p.v.token, p.wide, wave, lane);
  walk<MASK, MODE>(
      it, st, mask, lds, wave, active, rows,
      [&](int start, int end) { return mask_byte<MASK>(mask, start, end); },
      [](uint8_t b) { return __ballot(b != 0); }, [](uint8_t, int) {},
      [&](int buf, uint64_t bits) {
        const __bf16 *kt = lds[buf][0], *vt = lds[buf][1];
#pragma unroll
        for (int kh = 0; kh < kTokens<MODE> / 32; ++kh) {
          if (!(uint32_t)(bits >> (32 * kh))) continue;
          f32x16 s, dp;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            s = mma(row_frag(kt, fa, kh, ks), qf[ks], ks ? s : f32x16{});
            dp = mma(row_frag(vt, fa, kh, ks), dof[ks], ks ? dp : from);
          }
          if (bits != kAllRows<MODE>) mask_scores(s, bits, kh, h);
#pragma unroll
          for (int j = 0; j < 16; ++j) s[j] = __builtin_amdgcn_exp2f(s[j] * p.c - lse2) * dp[j];
#pragma unroll
          for (int step = 0; step < 2; ++step) {
            const bf16x8 ds = pack8(s, step);
#pragma unroll
            for (int dh = 0; dh < 2; ++dh) dq[dh] = mma(tr_frag(kt, fa, 2 * kh + step, dh), ds, dq[dh]);
          }
          if (fine) {  // what the rounding of dS took away
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] -= (float)(__bf16)s[j];
#pragma unroll
            for (int step = 0; step < 2; ++step) {
              const bf16x8 low = pack8(s, step);
#pragma unroll
              for (int dh = 0; dh < 2; ++dh) dq[dh] = mma(tr_frag(kt, fa, 2 * kh + step, dh), low, dq[dh]);
            }
          }
        }
      });

  if constexpr (MODE == kPairs) {
    float* at = pair_slot(lds, wave, lane, 32);
    __syncthreads();
    if (wave >= 4) {
      put_sums(at, dq[0]);
      put_sums(at + 64 * 16, dq[1]);
    }
    __syncthreads();
    if (wave >= 4) return;
    add_sums(at, dq[0]);
    add_sums(at + 64 * 16, dq[1]);
  }
  __bf16* base = p.dq.ptr + it.clip * p.dq.clip + it.head * p.dq.head;
  if constexpr (kAlone<MODE>) {
    float* part = reinterpret_cast<float*>(lds);
    __syncthreads();
    put_part(part + wave * kPart, dq, lane);
    __syncthreads();
    constexpr int kN = kJoin<MODE>;
    const int col = tid_x() & 31, d0 = (tid_x() >> 5) * kN, row = it.row0 + col;
    if (row >= it.row_end) return;
    float y[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) y[e] = sum_waves<MODE>(part + (d0 + e) * 33 + col) * p.scale;
    store_row(base + row * p.dq.token + d0, y);
  } else {
    if (r >= it.row_end) return;
    base += r * p.dq.token + 4 * h;
#pragma unroll
    for (int dh = 0; dh < 2; ++dh)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __bf16 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (__bf16)(dq[dh][4 * j + e] * p.scale);
        *reinterpret_cast<u32x2*>(base + 32 * dh + 8 * j) = *reinterpret_cast<u32x2*>(w);
      }
  }
}

// ---------------------------------------------------------------------------------------
// Backward over keys, short launches: dK and dV. A wave owns 32 key rows as columns of S = Q K^T and dP = dO V^T;
// dV^T += dO^T P, dK^T += Q^T dS. The sums of S start at -lse / scale and those of dP at -D of their rows (from LDS); a
// query that is not there starts at -inf, so that its probabilities are zero. Three waves a SIMD without a mask (four
// registers spilled to hold them: 8 x 1374 frames 161 us against 174); with one, three spill too much (254 us against
// 200 on the masked mix). 32 products a tile: 8 x 1374 frames 150 us, 825 TFLOP/s of the pairs.
// ---------------------------------------------------------------------------------------
struct RowStats {
  float ls, dl;
};

template <bool MASK, int MODE>
__global__ void __launch_bounds__(kThreads<MODE>, MODE == kTogether && !MASK ? 3 : 2) frame_attn_dkv_short_kernel(const FaParams p) {
  __shared__ __align__(16) __bf16 lds[kBuffers<MODE>][2][kTokens<MODE> * kHeadDim];
  __shared__ __align__(16) float stats[kBuffers<MODE>][2 * kTile];
  const FaItem it = fa_item(p, kRows<MODE>);
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6), h = lane >> 5;
  const FragAddr fa = frag_addr(lane);
  const uint8_t* mask = MASK ? p.mask + (int64_t)it.clip * p.N : nullptr;
  const int64_t stat = ((int64_t)it.clip * p.H + it.head) * p.N;
  const int first = it.row0 + (kAlone<MODE> ? 0 : (wave & 3) * 32), r = first + (lane & 31);
  const bool valid = r < it.row_end && (!MASK || mask[r]), active = __any(valid);

  bf16x8 kf[4], vf[4];
  const __bf16* kp = p.k.ptr + it.clip * p.k.clip + it.head * p.k.head + r * p.k.token + 8 * h;
  const __bf16* vp = p.v.ptr + it.clip * p.v.clip + it.head * p.v.head + r * p.v.token + 8 * h;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    kf[ks] = valid ? *reinterpret_cast<const bf16x8*>(kp + 16 * ks) : bf16x8{};
    vf[ks] = valid ? *reinterpret_cast<const bf16x8*>(vp + 16 * ks) : bf16x8{};
  }
  f32x16 dk[2] = {}, dv[2] = {};

  const float inv_scale = 1.f / p.scale;
  const Stager st = stager<MODE>(p.q.ptr + it.clip * p.q.clip + it.head * p.q.head, p.q.token,
                                  p.doo.ptr + it.clip * p.doo.clip + it.head * p.doo.head, p.doo.token, p.wide, wave,
                                  lane);
  walk<MASK, MODE>(
      it, st, mask, lds, wave, active, [] {},
      [&](int start, int end) {
        const int tok = start + lane;  // (end: at most the tile's)
        RowStats x;
        x.ls = tok < end ? p.lse[stat + tok] : -__builtin_inff();
        x.dl = tok < end ? p.delta[stat + tok] : 0.f;
        return x;
      },
      [](const RowStats& x) { return __ballot(x.ls != -__builtin_inff()); },
      [&](const RowStats& x, int buf) {
        const bool there = x.ls != -__builtin_inff();
        stats[buf][lane] = there ? -x.ls * inv_scale : -__builtin_inff();
        stats[buf][kTile + lane] = there ? -x.dl : 0.f;
      },
      [&](int buf, uint64_t bits) {
        const __bf16 *qt = lds[buf][0], *dt = lds[buf][1];
#pragma unroll
        for (int qh = 0; qh < kTokens<MODE> / 32; ++qh) {
          if (!(uint32_t)(bits >> (32 * qh))) continue;
          f32x16 s, dp;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(&stats[buf][32 * qh + 8 * j + 4 * h]);
            const f32x4 b = *reinterpret_cast<const f32x4*>(&stats[buf][kTile + 32 * qh + 8 * j + 4 * h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[4 * j + e] = a[e];
              dp[4 * j + e] = b[e];
            }
          }
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            s = mma(row_frag(qt, fa, qh, ks), kf[ks], s);
            dp = mma(row_frag(dt, fa, qh, ks), vf[ks], dp);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            s[j] = __builtin_amdgcn_exp2f(s[j] * p.c);
            dp[j] *= s[j];
          }
#pragma unroll
          for (int step = 0; step < 2; ++step) {
            const bf16x8 pf = pack8(s, step), ds = pack8(dp, step);
#pragma unroll
            for (int dh = 0; dh < 2; ++dh) {
              dv[dh] = mma(tr_frag(dt, fa, 2 * qh + step, dh), pf, dv[dh]);
              dk[dh] = mma(tr_frag(qt, fa, 2 * qh + step, dh), ds, dk[dh]);
            }
          }
        }
      });

  if constexpr (MODE == kPairs) {
    float* at = pair_slot(lds, wave, lane, 64);
    __syncthreads();
    if (wave >= 4) {
#pragma unroll
      for (int dh = 0; dh < 2; ++dh) {
        put_sums(at + 64 * 16 * dh, dk[dh]);
        put_sums(at + 64 * 16 * (2 + dh), dv[dh]);
      }
    }
    __syncthreads();
    if (wave >= 4) return;
#pragma unroll
    for (int dh = 0; dh < 2; ++dh) {
      add_sums(at + 64 * 16 * dh, dk[dh]);
      add_sums(at + 64 * 16 * (2 + dh), dv[dh]);
    }
  }
  __bf16* dkp = p.dk.ptr + it.clip * p.dk.clip + it.head * p.dk.head;
  __bf16* dvp = p.dv.ptr + it.clip * p.dv.clip + it.head * p.dv.head;
  if constexpr (kAlone<MODE>) {
    float* part = reinterpret_cast<float*>(lds);
    __syncthreads();
    constexpr int kN = kJoin<MODE>;
    const int col = tid_x() & 31, d0 = (tid_x() >> 5) * kN, row = it.row0 + col;
    auto total = [&](const f32x16(&x)[2], float (&y)[kN]) {  // (one result at a time: half the buffers hold it)
      put_part(part + wave * kPart, x, lane);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kN; ++e) y[e] = sum_waves<MODE>(part + (d0 + e) * 33 + col);
      __syncthreads();
    };
    float a[kN], b[kN];
    total(dk, a);
    total(dv, b);
    if (row >= it.row_end) return;
    const bool there = !MASK || mask[row];
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      a[e] = there ? a[e] * p.scale : 0.f;
      b[e] = there ? b[e] : 0.f;
    }
    store_row(dkp + row * p.dk.token + d0, a);
    store_row(dvp + row * p.dv.token + d0, b);
  } else {
    if (r >= it.row_end) return;
    dkp += r * p.dk.token + 4 * h;
    dvp += r * p.dv.token + 4 * h;
#pragma unroll
    for (int dh = 0; dh < 2; ++dh)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __bf16 a[4], b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = (__bf16)(valid ? dk[dh][4 * j + e] * p.scale : 0.f);
          b[e] = (__bf16)(valid ? dv[dh][4 * j + e] : 0.f);
        }
        *reinterpret_cast<u32x2*>(dkp + 32 * dh + 8 * j) = *reinterpret_cast<u32x2*>(a);
        *reinterpret_cast<u32x2*>(dvp + 32 * dh + 8 * j) = *reinterpret_cast<u32x2*>(b);
      }
  }
}

// ---------------------------------------------------------------------------------------
// Backward over keys, long launches without a mask: the same with 64 key rows a wave (two groups of 32).
//
// Two groups share every operand read from LDS (16 KB a wave for 32 queries: with one group LDS would be as busy as
// the matrix cores). Their sums, keys and values fill 192 registers, so one wave runs on a SIMD and has to overlap
// its own matrix products and vector work: a half tile (32 queries) is 32 products in a fixed order, with the
// exponentials and roundings of one group placed behind the products of the other (32 cycles each, room for seven
// vector instructions) and the LDS reads a phase ahead. (Compiler's order, two-phase loop: 686 TFLOP/s over 12 frames
// of 1374 tokens, 16 heads.) 12 frames of 1374, 10 of 16 heads dense: 1310 us, 1130 TFLOP/s of the pairs; matrix pipe busy
// 53%, vector pipe 44%.
//
// The products are inline assembly, for which the compiler keeps no distance to the instructions that read their results:
// nothing but this order may touch them, so the kernel must not spill (tests/test_frame_attn_build.py, _order.py).
// ---------------------------------------------------------------------------------------
struct DkvRows {
  bf16x8 q[4], d[4];  // row operands of Q and dO
  f32x16 ls, dl;      // where the sums of S and dP start: -lse / scale and -D of the rows
};

// One of the 16 reads of a half tile's row operands and statistics.
template <int I>
__device__ __forceinline__ void dkv_read(DkvRows& r, const __bf16* qt, const __bf16* dt, const float* stats,
                                         const FragAddr& fa, int qh, int h) {
  if constexpr (I < 4) {
    r.q[I] = row_frag(qt, fa, qh, I);
  } else if constexpr (I < 8) {
    r.d[I - 4] = row_frag(dt, fa, qh, I - 4);
  } else {
    constexpr int j = I % 4;
    const f32x4 x = *reinterpret_cast<const f32x4*>(stats + (I < 12 ? 0 : kTile) + 32 * qh + 8 * j + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) (I < 12 ? r.ls : r.dl)[4 * j + e] = x[e];
  }
}

struct DkvAcc {
  bf16x8 k[2][4], v[2][4];
  f32x16 dk[2][2], dv[2][2];
};

// Products with a fixed register class: results that vector instructions read stay in VGPRs, the running sums and the
// stationary operands in AGPRs. (With the builtin and more than 256 registers the compiler takes every result in
// AGPRs and copies: 728 copies beside 64 products in this kernel's loop.) The hazard rules are the caller's: a result is
// read by vector instructions three products later at the earliest, an operand is written by them a product ahead, and
// a separate third operand stays live for two more products.
__device__ __forceinline__ void mma_sum(f32x16& d, const bf16x8& a, const bf16x8& b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(d) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mma_from(f32x16& d, const bf16x8& a, const bf16x8& b, const f32x16& c) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %3" : "=&v"(d) : "v"(a), "a"(b), "v"(c));
}
__device__ __forceinline__ void mma_more(f32x16& d, const bf16x8& a, const bf16x8& b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "a"(b));
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}
__device__ __forceinline__ bf16x8 frag4(const uint32_t (&w)[8], int st) {
  return __builtin_bit_cast(bf16x8, u32x4{w[4 * st], w[4 * st + 1], w[4 * st + 2], w[4 * st + 3]});
}

// Keeps values where they are computed: the compiler may not move their computation behind this point.
__device__ __forceinline__ void pin(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
}
template <int FIRST, int N>
__device__ __forceinline__ void pin_elems(f32x16& x) {
#pragma unroll
  for (int i = FIRST; i < FIRST + N; ++i) {
    float e = x[i];
    asm volatile("" : "+v"(e));
    x[i] = e;
  }
}

// One half tile. `mid` runs when every read of this half is issued (its barrier waits for them); `ahead(Int<i>)` issues
// read i of the next half's 16.
template <typename Mid, typename Ahead>
__device__ __forceinline__ void dkv_half(DkvAcc& A, const DkvRows& r, const __bf16* qt, const __bf16* dt,
                                         const FragAddr& fa, int qh, float c, Mid mid, Ahead ahead) {
  f32x16 s[2], dp[2];
  uint32_t pw[2][8], dw[2][8];
  bf16x8 td[2][2], tq[2][2];  // transposed operands [step][dh]
  // vector work of one pair of elements, in steps that are a product apart (a lone wave waits for each result)
  auto fm = [&](int g, int t) {
    s[g][2 * t] *= c;
    s[g][2 * t + 1] *= c;
  };
  auto ex = [&](int g, int t) {
    s[g][2 * t] = __builtin_amdgcn_exp2f(s[g][2 * t]);
    s[g][2 * t + 1] = __builtin_amdgcn_exp2f(s[g][2 * t + 1]);
  };
  auto cv = [&](int g, int t) { pw[g][t] = pack2(s[g][2 * t], s[g][2 * t + 1]); };
  auto ml = [&](int g, int t) {
    dp[g][2 * t] *= s[g][2 * t];
    dp[g][2 * t + 1] *= s[g][2 * t + 1];
  };
  auto cw = [&](int g, int t) { dw[g][t] = pack2(dp[g][2 * t], dp[g][2 * t + 1]); };
#define FENCE __builtin_amdgcn_sched_barrier(0)
#define S0(g) mma_from(s[g], r.q[0], A.k[g][0], r.ls)
#define S_(g, ks) mma_more(s[g], r.q[ks], A.k[g][ks])
#define P0(g) mma_from(dp[g], r.d[0], A.v[g][0], r.dl)
#define P_(g, ks) mma_more(dp[g], r.d[ks], A.v[g][ks])
#define V_(g, st, dh) mma_sum(A.dv[g][dh], td[st][dh], frag4(pw[g], st))
#define K_(g, st, dh) mma_sum(A.dk[g][dh], tq[st][dh], frag4(dw[g], st))
#define TD(st, dh) td[st][dh] = tr_frag(dt, fa, 2 * qh + st, dh)
#define TQ(st, dh) tq[st][dh] = tr_frag(qt, fa, 2 * qh + st, dh)
#define NEXT(i) ahead(Int<i>())
  FENCE;
  S0(0); TD(0, 0); FENCE;
  S_(0, 1); TD(0, 1); FENCE;
  S_(0, 2); TD(1, 0); FENCE;
  S_(0, 3); TD(1, 1); FENCE;
  S0(1); TQ(0, 0); FENCE;
  S_(1, 1); TQ(0, 1); FENCE;
  S_(1, 2); TQ(1, 0); fm(0, 0); FENCE;
  asm volatile("" ::"v"(r.ls));  // (third operand of S0: live until here)
  S_(1, 3); TQ(1, 1); fm(0, 1); ex(0, 0); FENCE;
  P0(0); fm(0, 2); ex(0, 1); cv(0, 0); FENCE;
  P_(0, 1); fm(0, 3); ex(0, 2); cv(0, 1); FENCE;
  pin_elems<0, 8>(s[0]);
  pin(pw[0][0], pw[0][1], pw[0][0], pw[0][1]);
  mid();
  FENCE;
  P_(0, 2); NEXT(0); fm(0, 4); ex(0, 3); cv(0, 2); FENCE;
  P_(0, 3); NEXT(1); fm(0, 5); ex(0, 4); cv(0, 3); fm(1, 0); FENCE;
  P0(1); NEXT(2); fm(0, 6); ex(0, 5); cv(0, 4); ex(1, 0); FENCE;
  P_(1, 1); NEXT(3); fm(0, 7); ex(0, 6); cv(0, 5); fm(1, 1); FENCE;
  P_(1, 2); NEXT(8); ex(0, 7); cv(0, 6); ml(0, 0); ex(1, 1); FENCE;
  asm volatile("" ::"v"(r.dl));  // (third operand of P0: live until here)
  P_(1, 3); NEXT(9); cv(0, 7); ml(0, 1); ml(0, 2); cv(1, 0); cw(0, 0); FENCE;
  V_(0, 0, 0); NEXT(10); ml(0, 3); cw(0, 1); cw(0, 2); fm(1, 2); cv(1, 1); FENCE;
  V_(0, 0, 1); NEXT(11); ml(0, 4); cw(0, 3); fm(1, 3); ex(1, 2); FENCE;
  V_(0, 1, 0); NEXT(4); ml(0, 5); cw(0, 4); ex(1, 3); cv(1, 2); FENCE;
  V_(0, 1, 1); NEXT(5); ml(0, 6); cw(0, 5); fm(1, 4); cv(1, 3); FENCE;
  K_(0, 0, 0); NEXT(6); ml(0, 7); cw(0, 6); fm(1, 5); ex(1, 4); FENCE;
  K_(0, 0, 1); NEXT(7); cw(0, 7); fm(1, 6); ex(1, 5); cv(1, 4); FENCE;
  V_(1, 0, 0); NEXT(12); fm(1, 7); ex(1, 6); cv(1, 5); FENCE;
  V_(1, 0, 1); NEXT(13); ex(1, 7); cv(1, 6); ml(1, 0); FENCE;
  K_(0, 1, 0); NEXT(14); cv(1, 7); ml(1, 1); ml(1, 2); cw(1, 0); FENCE;
  K_(0, 1, 1); NEXT(15); ml(1, 3); ml(1, 4); cw(1, 1); cw(1, 2); FENCE;
  V_(1, 1, 0); ml(1, 5); cw(1, 3); cw(1, 4); FENCE;
  V_(1, 1, 1); ml(1, 6); ml(1, 7); cw(1, 5); FENCE;
  K_(1, 0, 0); cw(1, 6); cw(1, 7); FENCE;
  K_(1, 0, 1); FENCE;
  K_(1, 1, 0); FENCE;
  K_(1, 1, 1); FENCE;
#undef FENCE
#undef S0
#undef S_
#undef P0
#undef P_
#undef V_
#undef K_
#undef TD
#undef TQ
#undef NEXT
}

__global__ void __launch_bounds__(256, 1) frame_attn_dkv_long_kernel(const FaParams p) {
  __shared__ __align__(16) __bf16 lds[2][2][kTileElems];
  __shared__ __align__(16) float stats[2][2 * kTile];
  const FaItem it = fa_item(p, 256);
  const int lane = tid_x() & 63, wave = __builtin_amdgcn_readfirstlane(tid_x() >> 6), h = lane >> 5;
  const FragAddr fa = frag_addr(lane);
  const __bf16* qb = p.q.ptr + it.clip * p.q.clip + it.head * p.q.head;
  const __bf16* db = p.doo.ptr + it.clip * p.doo.clip + it.head * p.doo.head;
  const int64_t stat = ((int64_t)it.clip * p.H + it.head) * p.N;
  const int first = it.row0 + wave * 64;
  const bool active = first < it.row_end;

  const int na = tiles_of<kTile>(it.a1 - it.a0), nw = na + tiles_of<kTile>(it.b1 - it.b0);
  const float inv_scale = 1.f / p.scale;
  const Stager st = stager<0>(qb, p.q.token, db, p.doo.token, p.wide, wave, lane);
  float ls = 0.f, dl = 0.f;
  auto load = [&](int i) {
    int start, end;
    walk_tile<kTile>(it, na, i, &start, &end);
    const int tok = start + lane;
    ls = tok < end ? p.lse[stat + tok] : -__builtin_inff();
    dl = tok < end ? p.delta[stat + tok] : 0.f;
    stage<0>(st, start, end, lds[i & 1][0], lds[i & 1][1]);
  };
  // tile i, loaded before, becomes readable; the other buffer is free from here on
  auto ready = [&](int i) {
    const bool there = ls != -__builtin_inff();
    wait_vm<0>();
    if (wave == 0) {
      stats[i & 1][lane] = there ? -ls * inv_scale : -__builtin_inff();
      stats[i & 1][kTile + lane] = there ? -dl : 0.f;
    }
    __syncthreads();
    if (i + 1 < nw) load(i + 1);
  };

  if (nw > 0) load(0);
  DkvAcc A;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int r = first + 32 * g + (lane & 31);
    const bool valid = r < it.row_end;
    const __bf16* kp = p.k.ptr + it.clip * p.k.clip + it.head * p.k.head + r * p.k.token + 8 * h;
    const __bf16* vp = p.v.ptr + it.clip * p.v.clip + it.head * p.v.head + r * p.v.token + 8 * h;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      A.k[g][ks] = valid ? *reinterpret_cast<const bf16x8*>(kp + 16 * ks) : bf16x8{};
      A.v[g][ks] = valid ? *reinterpret_cast<const bf16x8*>(vp + 16 * ks) : bf16x8{};
    }
    A.dk[g][0] = A.dk[g][1] = A.dv[g][0] = A.dv[g][1] = f32x16{};
  }

  if (nw > 0) ready(0);
  if (!active) {
    for (int i = 1; i < nw; ++i) ready(i);
    return;
  }
  DkvRows r0, r1;  // first and second half tiles
  // the reads of a half tile of tile i
  auto first_half = [&](int i) {
    return [&, i](auto n) {
      dkv_read<decltype(n)::value>(r0, lds[i & 1][0], lds[i & 1][1], stats[i & 1], fa, 0, h);
    };
  };
  auto second_half = [&](int i) {
    return [&, i](auto n) {
      dkv_read<decltype(n)::value>(r1, lds[i & 1][0], lds[i & 1][1], stats[i & 1], fa, 1, h);
    };
  };
  if (nw > 0) {
    const auto read = first_half(0);
    read(Int<0>()), read(Int<1>()), read(Int<2>()), read(Int<3>()), read(Int<4>()), read(Int<5>()), read(Int<6>());
    read(Int<7>()), read(Int<8>()), read(Int<9>()), read(Int<10>()), read(Int<11>()), read(Int<12>());
    read(Int<13>()), read(Int<14>()), read(Int<15>());
  }
  for (int i = 0; i < nw; ++i) {
    const __bf16* qt = lds[i & 1][0];
    const __bf16* dt = lds[i & 1][1];
    dkv_half(A, r0, qt, dt, fa, 0, p.c, [] {}, second_half(i));
    // every read of this tile is done at `mid` of its second half
    dkv_half(A, r1, qt, dt, fa, 1, p.c,
             [&] {
               if (i + 1 < nw) ready(i + 1);
             },
             first_half(i + 1));
  }
  // The last products are done before the sums are read: the wait stands right behind the loop, where no copy of a sum can
  // come ahead of it, and the statement that takes the sums keeps their first use behind it.
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile(""
               : "+a"(A.dk[0][0]), "+a"(A.dk[0][1]), "+a"(A.dk[1][0]), "+a"(A.dk[1][1]), "+a"(A.dv[0][0]),
                 "+a"(A.dv[0][1]), "+a"(A.dv[1][0]), "+a"(A.dv[1][1]));
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int r = first + 32 * g + (lane & 31);
    if (r < it.row_end) {
      __bf16* kp = p.dk.ptr + it.clip * p.dk.clip + it.head * p.dk.head + r * p.dk.token + 4 * h;
      __bf16* vp = p.dv.ptr + it.clip * p.dv.clip + it.head * p.dv.head + r * p.dv.token + 4 * h;
#pragma unroll
      for (int dh = 0; dh < 2; ++dh)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          __bf16 a[4], b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] = (__bf16)(A.dk[g][dh][4 * j + e] * p.scale);
            b[e] = (__bf16)A.dv[g][dh][4 * j + e];
          }
          *reinterpret_cast<u32x2*>(kp + 32 * dh + 8 * j) = *reinterpret_cast<u32x2*>(a);
          *reinterpret_cast<u32x2*>(vp + 32 * dh + 8 * j) = *reinterpret_cast<u32x2*>(b);
        }
    }
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Row tiles of every head, the longest walks first, at most one class of each kind. keys: the tiles are key rows and
// walk queries. Returns the number of work-groups.
static int64_t make_classes(FaParams* p, const int32_t* patterns, int frames, int rows, bool keys) {
  const int T = p->T, N = p->N;
  uint64_t of[SAF3R_SKIP + 1] = {};
  for (int h = 0; h < p->H; ++h) of[patterns[h]] |= 1ull << h;
  int64_t total = 0;
  int n = 0;
  auto add = [&](uint64_t heads, int tok0, int tok1, bool per_frame, int walk) {
    if (!heads || tok1 <= tok0) return;
    FaClass& c = p->cls[n++];
    c.start = (int)std::min<int64_t>(total, 0x7fffffff);
    c.nt = per_frame ? (int)ceil_div(T, rows) : 0;
    const int64_t per_clip = per_frame ? (int64_t)c.nt * ((tok1 - tok0) / T) : ceil_div(tok1 - tok0, rows);
    c.per_clip = (int)per_clip;
    c.tok0 = tok0;
    c.tok1 = tok1;
    c.walk = walk;
    c.heads = heads;
    total += per_clip * __builtin_popcountll(heads) * p->clips;
  };
  const uint64_t anchor = of[SAF3R_ANCHOR], both = of[SAF3R_ANCHOR_LOCAL], local = of[SAF3R_FRAME_LOCAL];
  add(of[SAF3R_DENSE], 0, N, false, kAll);
  if (keys) {  // the first frame's keys serve every query, those of the others their own frame or none
    add(anchor | both, 0, T, false, kAll);
    add(local, 0, N, true, kOwn);
    add(both, T, N, true, kOwn);
    add(anchor, T, N, false, kNone);
  } else {
    add(both, 0, N, true, kFirstOwn);
    add(local, 0, N, true, kOwn);
    add(anchor, 0, N, false, kFirst);
  }
  add(of[SAF3R_SKIP], 0, N, false, kNone);
  for (; n < kFaClasses; ++n) {
    p->cls[n] = FaClass{};
    p->cls[n].start = 0x7fffffff;
    p->cls[n].per_clip = 1;
    p->cls[n].heads = 1;
  }
  return total;
}

static bool fa_tensor(FaTensor* t, const saf3r_heads* h) {
  if (!h || !h->ptr) return false;
  t->ptr = (__bf16*)const_cast<void*>(h->ptr);
  t->clip = h->clip_stride;
  t->token = h->token_stride;
  t->head = h->head_stride;
  return true;
}

static bool fa_aligned(const FaTensor& t) {
  return (uintptr_t)t.ptr % 16 == 0 && t.clip % 8 == 0 && t.token % 8 == 0 && t.head % 8 == 0;
}

// Whether rows that are written would lie on each other (a stride of zero).
static bool fa_overlaps(const FaTensor& t, const FaParams& p) {
  return t.ptr && ((t.clip == 0 && p.clips > 1) || (t.token == 0 && p.N > 1) || (t.head == 0 && p.H > 1));
}

// Whether the rows of a walk tile are so far apart (or in descending order) that their byte offsets need 64 bits.
static bool fa_wide(const FaTensor& t) { return t.token < 0 || t.token >= ((int64_t)1 << 31) / 2 / kTile; }

static int fa_check(const char* who, FaParams* p, int clips, int frames, int tokens_per_frame, int num_heads,
                    const int32_t* patterns, const uint8_t* mask, float scale) {
  if (clips < 0 || frames <= 0 || tokens_per_frame <= 0)
    return fail(SAF3R_ERR_INVALID, "%s: invalid sizes: %d clips, %d frames x %d tokens", who, clips, frames,
                tokens_per_frame);
  if (num_heads <= 0) return fail(SAF3R_ERR_INVALID, "%s: bad num_heads %d", who, num_heads);
  if (num_heads > kMaxHeads)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: %d heads (at most %d)", who, num_heads, kMaxHeads);
  if ((int64_t)frames * tokens_per_frame > 0x7fffff00 - 512)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: %d frames x %d tokens pass 31 bits", who, frames, tokens_per_frame);
  if (!patterns) return fail(SAF3R_ERR_INVALID, "%s: null patterns", who);
  for (int h = 0; h < num_heads; ++h) {
    const int x = patterns[h];
    if (x != SAF3R_DENSE && x != SAF3R_FRAME_LOCAL && x != SAF3R_ANCHOR_LOCAL && x != SAF3R_ANCHOR && x != SAF3R_SKIP)
      return fail(x < 0 || x > SAF3R_TOKEN_DYNAMIC_KEYSET ? SAF3R_ERR_INVALID : SAF3R_ERR_UNSUPPORTED,
                  "%s: head %d: pattern %d is not one of dense, frame-local, anchor-local, anchor, skip", who, h, x);
  }
  // (the backward pass starts its sums at lse / scale, in fp32)
  if (!(scale >= 1e-30f && scale <= 1e30f)) return fail(SAF3R_ERR_INVALID, "%s: scale %g (1e-30 to 1e30)", who, scale);
  p->N = frames * tokens_per_frame;
  p->T = tokens_per_frame;
  p->H = num_heads;
  p->clips = clips;
  p->mask = mask;
  p->scale = scale;
  p->c = scale * kLog2e;
  return SAF3R_OK;
}

// The mode of a launch, by its work-groups of 128 rows and its longest walk; the figures are forward / dQ / dK and dV in
// us, dense heads.
// Below half a work-group a compute unit the waves walk alone (16 heads of 522 tokens, 80 work-groups: 10.6 / 13.9 / 12.9,
// together 13.9 / 17.6 / 16.4; 16 of 800, 112: 13 / 17 / 17, in pairs 15 / 20 / 21; one of 16000, 125: 130 / 140 / 189, in
// pairs 153 / 181 / 238; 16 of 1041, 144: 23 / 27 / 30, in pairs 18 / 24 / 26),
constexpr int64_t kAloneBelow = 128;
// eight of them where the work-groups of 32 rows all run at once like that, on long walks (8 heads of 1000 tokens: 10.8 /
// 14.4 / 13.0, four waves 11.7 / 13.9 / 15.0; one of 4096: 19 / 24 / 28 and 26 / 29 / 38; 8 of 512: 7.9 / 11.7 / 9.4 and
// 7.6 / 10.6 / 9.6).
constexpr int64_t kEightUpTo = 256;
constexpr int kEightFrom = 768;
// Up to one work-group a compute unit, pairs of groups, on long walks (3 heads of 8192 tokens, 192 work-groups: 82 / 99 /
// 127, together 109 / 133 / 200; 16 of 2048, 256: 29 / 36 / 42 and 34 / 42 / 58; 4 clips of 16 of 512: 13.9 / 18.3 / 19.1
// and 14.7 / 18.1 / 21.0; 10 of 8 of 256: 10.0 / 13.2 / 11.7 and 9.8 / 12.4 / 12.7). Shorter walks count by their share of the
// longest: few long ones bound a launch, whatever runs beside them (2 clips of 32 x 77 tokens, 2 heads dense, 5 local, 9
// on the first frame: 32 / 39 / 44 and 41 / 50 / 68; 2 of 22 x 269, 1, 6 and 9: 91 / 116 / 133 and 93 / 114 / 165).
constexpr int64_t kPairsUpTo = 256;
constexpr int kPairsFrom = 512;

// Tokens that a work-group of a class walks (of a lone frame once), and the most of a launch.
static int fa_walked(const FaParams& p, const FaClass& c) {
  if (c.walk == kFirstOwn) return p.N > p.T ? 2 * p.T : p.T;  // (two frames are at most N)
  return c.walk == kAll ? p.N : c.walk == kNone ? 0 : p.T;
}
static int fa_longest(const FaParams& p) {
  int longest = 0;
  for (const FaClass& c : p.cls) longest = std::max(longest, fa_walked(p, c));
  return longest;
}

// The n work-groups of a launch as so many of its longest walk (in tiles, one more for the rest of a work-group).
static int64_t fa_load(const FaParams& p, int64_t n) {
  const int64_t longest = tiles_of<kTile>(fa_longest(p)) + 1;
  int64_t tiles = 0;
  for (int i = 0; i < kFaClasses; ++i) {
    const int64_t end = i + 1 < kFaClasses ? std::min<int64_t>(p.cls[i + 1].start, n) : n;
    const int64_t walk = tiles_of<kTile>(fa_walked(p, p.cls[i])) + 1;
    tiles += std::max<int64_t>(0, end - p.cls[i].start) * walk;
  }
  return ceil_div(tiles, longest);
}

// Whether the backward pass over keys takes 64 rows a wave (without a mask, where groups walk together): `load` and
// `load256` of its launches of 128 and 256 rows a work-group. The wide ones run one a compute unit, in rounds of 256 that
// take 7 units of time a walked tile where 256 work-groups of 128 rows take 4, and start and end without another to fill the
// time, about five tiles. (16 dense heads, long and short in us: 2050 tokens, 1 round against 2, 64 and 75; 4096, 1 and 2,
// 133 and 155; 6144, 2 and 3, 330 and 307; 7168, 2 and 4, 386 and 473; 10240, 3 and 5, 810 and 816; 12288, 3 and 6, 1021
// and 1145; 20 frames of 1374, 8 and 14, 411 and 365; 8 of them, 3 and 6, 151 and 147; 60 of 250, 4 and 8, 72 and 61.)
static bool fa_takes_long(int64_t load, int64_t load256, int longest) {
  const int64_t tiles = tiles_of<kTile>(longest);
  return 7 * ceil_div(load256, 256) * (tiles + 5) <= 4 * ceil_div(load, 256) * (tiles + 1);
}

// The mode of a launch and its classes; n: its work-groups.
static int fa_mode(FaParams* p, const int32_t* patterns, int frames, bool keys, int64_t* n) {
  *n = make_classes(p, patterns, frames, kRows<kTogether>, keys);
  if (*n >= kAloneBelow) return fa_load(*p, *n) <= kPairsUpTo && fa_longest(*p) >= kPairsFrom ? kPairs : kTogether;
  *n = make_classes(p, patterns, frames, kRows<4>, keys);
  return *n <= kEightUpTo && fa_longest(*p) >= kEightFrom ? 8 : 4;
}

// f(whether there is a mask, mode)
template <typename F>
static void fa_launch(bool mask, int mode, F f) {
  auto with = [&](auto m) {
    switch (mode) {
      case 8: return f(m, Int<8>());
      case 4: return f(m, Int<4>());
      case kPairs: return f(m, Int<kPairs>());
      default: return f(m, Int<kTogether>());
    }
  };
  if (mask)
    with(std::true_type());
  else
    with(std::false_type());
}

static int fa_grid(const char* who, int64_t total) {
  // (a launch counts its threads in 32 bits)
  if (total > 0xffffffffll / 512) return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many row tiles for one launch", who);
  return SAF3R_OK;
}

}  // namespace saf3r

using namespace saf3r;

extern "C" int saf3r_frame_attn_fwd(const saf3r_heads* q, const saf3r_heads* k, const saf3r_heads* v, int clips,
                                    int frames, int tokens_per_frame, int num_heads, const int32_t* patterns,
                                    const uint8_t* token_mask, float scale, const saf3r_heads* out,
                                    const saf3r_heads* out_rest, float* lse, void* stream) {
  const char* who = "saf3r_frame_attn_fwd";
  if (int e = injected(who)) return e;
  FaParams p{};
  if (int e = fa_check(who, &p, clips, frames, tokens_per_frame, num_heads, patterns, token_mask, scale)) return e;
  if (clips == 0) return SAF3R_OK;
  if (!fa_tensor(&p.q, q) || !fa_tensor(&p.k, k) || !fa_tensor(&p.v, v) || !fa_tensor(&p.o, out) || !lse)
    return fail(SAF3R_ERR_INVALID, "%s: null tensor pointer", who);
  if (out_rest && !fa_tensor(&p.rest, out_rest)) return fail(SAF3R_ERR_INVALID, "%s: null out_rest", who);
  if (!fa_aligned(p.q) || !fa_aligned(p.k) || !fa_aligned(p.v) || !fa_aligned(p.o) || !fa_aligned(p.rest) ||
      (uintptr_t)lse % 4)
    return fail(SAF3R_ERR_INVALID, "%s: rows must be 16-byte aligned with strides a multiple of 8", who);
  if (fa_overlaps(p.o, p) || fa_overlaps(p.rest, p))
    return fail(SAF3R_ERR_INVALID, "%s: written rows overlap (a stride of zero)", who);
  p.lse = lse;
  p.wide = fa_wide(p.k) || fa_wide(p.v);
  int64_t n;
  const int mode = fa_mode(&p, patterns, frames, false, &n);
  if (int e = fa_grid(who, n)) return e;
  fa_launch(token_mask != nullptr, mode, [&](auto m, auto d) {
    constexpr int kMode = decltype(d)::value;
    hipLaunchKernelGGL((frame_attn_fwd_kernel<decltype(m)::value, kMode>), dim3((uint32_t)n), dim3(kThreads<kMode>), 0,
                       (hipStream_t)stream, p);
  });
  return check_launch(who);
}

extern "C" int64_t saf3r_frame_attn_bwd_workspace_bytes(int clips, int frames, int tokens_per_frame, int num_heads) {
  const char* who = "saf3r_frame_attn_bwd_workspace_bytes";
  if (clips < 0 || frames <= 0 || tokens_per_frame <= 0 || num_heads <= 0 || num_heads > kMaxHeads ||
      (int64_t)frames * tokens_per_frame > 0x7fffff00 - 512) {
    fail(SAF3R_ERR_INVALID, "%s: invalid sizes", who);
    return -1;
  }
  return (int64_t)clips * num_heads * frames * tokens_per_frame * 4;
}

extern "C" int saf3r_frame_attn_bwd(const saf3r_heads* dout, const saf3r_heads* q, const saf3r_heads* k,
                                    const saf3r_heads* v, const saf3r_heads* out, const saf3r_heads* out_rest,
                                    const float* lse, int clips, int frames, int tokens_per_frame, int num_heads,
                                    const int32_t* patterns, const uint8_t* token_mask, float scale,
                                    const saf3r_heads* dq, const saf3r_heads* dk, const saf3r_heads* dv,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "saf3r_frame_attn_bwd";
  if (int e = injected(who)) return e;
  FaParams p{};
  if (int e = fa_check(who, &p, clips, frames, tokens_per_frame, num_heads, patterns, token_mask, scale)) return e;
  if (clips == 0) return SAF3R_OK;
  if (!fa_tensor(&p.doo, dout) || !fa_tensor(&p.q, q) || !fa_tensor(&p.k, k) || !fa_tensor(&p.v, v) ||
      !fa_tensor(&p.o, out) || !fa_tensor(&p.dq, dq) || !fa_tensor(&p.dk, dk) || !fa_tensor(&p.dv, dv) || !lse)
    return fail(SAF3R_ERR_INVALID, "%s: null tensor pointer", who);
  if (out_rest && !fa_tensor(&p.rest, out_rest)) return fail(SAF3R_ERR_INVALID, "%s: null out_rest", who);
  for (const FaTensor* t : {&p.doo, &p.q, &p.k, &p.v, &p.o, &p.rest, &p.dq, &p.dk, &p.dv})
    if (!fa_aligned(*t))
      return fail(SAF3R_ERR_INVALID, "%s: rows must be 16-byte aligned with strides a multiple of 8", who);
  if (fa_overlaps(p.dq, p) || fa_overlaps(p.dk, p) || fa_overlaps(p.dv, p))
    return fail(SAF3R_ERR_INVALID, "%s: written rows overlap (a stride of zero)", who);
  const int64_t need = saf3r_frame_attn_bwd_workspace_bytes(clips, frames, tokens_per_frame, num_heads);
  if (workspace_bytes < need || !workspace || (uintptr_t)workspace % 16 || (uintptr_t)lse % 4)
    return fail(SAF3R_ERR_INVALID, "%s: workspace of %lld bytes: %lld, 16-byte aligned, are needed", who,
                (long long)workspace_bytes, (long long)need);
  p.lse = const_cast<float*>(lse);
  p.delta = (float*)workspace;
  p.wide = fa_wide(p.q) || fa_wide(p.k) || fa_wide(p.v) || fa_wide(p.doo);
  FaParams pk = p;
  const bool masked = token_mask != nullptr;
  int64_t n, nk;
  const int mode = fa_mode(&p, patterns, frames, false, &n), mode_k = fa_mode(&pk, patterns, frames, true, &nk);
  bool long_k = false;
  if (!masked && mode_k == kTogether) {
    FaParams wide = pk;
    const int64_t n256 = make_classes(&wide, patterns, frames, 256, true);
    long_k = fa_takes_long(fa_load(pk, nk), fa_load(wide, n256), fa_longest(wide));
    if (long_k) {
      pk = wide;
      nk = n256;
    }
  }
  if (int e = fa_grid(who, std::max(n, nk))) return e;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 gk((uint32_t)nk);
  fa_launch(masked, mode, [&](auto m, auto d) {
    constexpr int kMode = decltype(d)::value;
    hipLaunchKernelGGL((frame_attn_dq_kernel<decltype(m)::value, kMode>), dim3((uint32_t)n), dim3(kThreads<kMode>), 0, s, p);
  });
  if (long_k)
    hipLaunchKernelGGL(frame_attn_dkv_long_kernel, gk, dim3(256), 0, s, pk);
  else
    fa_launch(masked, mode_k, [&](auto m, auto d) {
      constexpr int kMode = decltype(d)::value;
      hipLaunchKernelGGL((frame_attn_dkv_short_kernel<decltype(m)::value, kMode>), gk, dim3(kThreads<kMode>), 0, s, pk);
    });
  return check_launch(who);
}
