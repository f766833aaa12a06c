// Keep masks from a counter: sixteen random bits for every element of a matrix as a function of (seed, stream, row, column),
// so that the backward pass, a captured graph or another kernel computes the mask again instead of reading one.
//
// Generator: Philox4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", 2011). A block of 128 bits serves eight columns of a row: counter (column / 8, row's low half, row's high half,
// stream's low half), key = seed; column 8 g + j takes the low half of word j / 2 for even j, its high half for odd j.
// Sixteen bits an element: one block per 16-byte vector of a 16-bit row in place of two. An element is dropped when its bits
// are below `limit`, a probability of limit / 65536 exactly; the scale of the others is 65536 / (65536 - limit), so the
// mean is kept exactly whatever p was rounded to (by at most 2^-17).
#pragma once

#include "common.h"

namespace saf3r {

struct DropParams {
  const int64_t* state;  // device: seed, stream
  int limit;             // 0: no dropout; 65536: everything is dropped
  float scale;
};

struct DropKey {
  uint32_t k0, k1, stream;
};

__device__ __forceinline__ DropKey drop_key(const DropParams& p) {
  const uint64_t seed = (uint64_t)p.state[0];
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)(uint64_t)p.state[1]};
}

__device__ __forceinline__ void philox(const DropKey& key, uint32_t group, uint64_t row, uint32_t (&w)[4]) {
  uint32_t c0 = group, c1 = (uint32_t)row, c2 = (uint32_t)(row >> 32), c3 = key.stream, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// x *= keep / (1 - p) for the eight columns from 8 * group of a row. A dropped element is zero whatever x holds; so is z's, which
// a gradient multiplies by x (an infinity there would be a NaN).
__device__ __forceinline__ void drop8(const DropKey& key, int limit, float scale, uint32_t group, uint64_t row,
                                      float (&x)[8], float (&z)[8]) {
  uint32_t w[4];
  philox(key, group, row, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t bits = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
    const bool keep = (int)bits >= limit;
    x[j] = keep ? x[j] * scale : 0.f;
    z[j] = keep ? z[j] : 0.f;
  }
}

__device__ __forceinline__ void drop8(const DropKey& key, int limit, float scale, uint32_t group, uint64_t row,
                                      float (&x)[8]) {
  float none[8] = {};
  drop8(key, limit, scale, group, row, x, none);
}

inline int drop_check(const char* who, int limit, const int64_t* state, DropParams* p) {
  if (limit < 0 || limit > 65536)
    return fail(SAF3R_ERR_INVALID, "%s: drop %d: 65536 times the probability, 0 to 65536", who, limit);
  if (limit && (!state || (uintptr_t)state % 8))
    return fail(SAF3R_ERR_INVALID, "%s: dropout needs its state (two int64)", who);
  *p = {limit ? state : nullptr, limit, limit < 65536 ? 65536.f / (float)(65536 - limit) : 0.f};
  return SAF3R_OK;
}

}  // namespace saf3r
