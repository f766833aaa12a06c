// Prologue of q and k on their way into attention, with its backward pass: LayerNorm over the head dimension
// (optional) and rotary positions (optional), straight from the qkv buffer.
//
// The first `rot` elements of a row are `axes` equal sections; section a is rotated by the angles of the token's
// a-th position: pairs (j, j + S/2) of a section of S elements (half layout) or (2 j, 2 j + 1) (interleaved),
//   (u, v) -> (u cos - v sin, v cos + u sin),  cos / sin = table[position][j];
// the elements behind `rot` are only normed. Backward: the inverse rotation of dy, then LayerNorm's backward pass with
// the row's statistics recomputed from x.
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx; next to that by vector
// instructions (about 25 an element in the backward pass), so that nothing but the rows themselves is computed in the
// loop. A lane holds both sides of its pairs (two vectors of VE elements), so that the rotation needs no exchange;
// D / (2 VE) lanes own a row. A work-group serves one group (q or k), so that its lanes keep the norm's parameters, and
// the sums of their gradients, in registers, and takes whole tokens: a lane keeps its head, the lanes of a token share
// the table lines, and the next tokens' rows are on their way while the current ones are used. The partial sums of
// the work-groups are added by a second kernel in a fixed order. Without the norm the backward pass is the inverse
// rotation, the forward kernel's.
// Measured, bf16, q and k of 21984 tokens of 16 heads of 64: forward 31 us for 180 MB (5.8 TB/s), backward 54 us for
// 270 MB (5.0 TB/s) and 5 us for the sums; with one row at a time and no read ahead the backward took 113 us. 1041
// tokens: 6 us.
#include "row_ops.h"

namespace saf3r {

struct RotTensor {
  char* ptr;
  int64_t clip, token, group, head;  // strides in elements
};

struct RotParams {
  RotTensor x, dy, y;  // y: forward's result, or dx
  const int32_t* pos;  // [clip][token][axes], words between positions pos_step
  const float* cosine;
  const float* sine;
  const void* w;
  const void* b;
  float* part;       // [parts][2][groups * dim]
  int n;             // clips * tokens
  int units;         // steps of a group: `per` tokens, or one of `blocks` parts of a token's heads
  int per, blocks;
  int parts;         // work-groups of a group (the grid's size comes from host memory in a kernel: slow)
  int tokens, heads, groups, dim;
  float sign;        // forward kernel: 1, or -1 for the inverse rotation
  int flat;          // every tensor's clips follow each other as its tokens do
  int rot, axes, positions, pos_step, interleaved, norm;
  float eps;
};

// A lane's place in its row: two vectors of VE elements, and how they are rotated.
struct RotLane {
  int a, b;      // element offsets
  int axis;      // -1: passed through
  int table;     // first table column
  bool on;
};

template <int VE>
__device__ inline RotLane rot_lane(const RotParams& p, int t) {
  RotLane r;
  const int turned = p.rot / (2 * VE);
  r.on = t * 2 * VE < p.dim;
  r.axis = -1;
  r.table = 0;
  if (t >= turned || !p.cosine) {
    r.a = t * 2 * VE;
    r.b = r.a + VE;
    return r;
  }
  const int S = p.rot / p.axes;
  if (p.interleaved) {
    r.a = t * 2 * VE;
    r.b = r.a + VE;
    r.axis = r.a / S;
    r.table = (r.a - r.axis * S) / 2;
  } else {
    const int per = S / (2 * VE);
    r.axis = t / per;
    r.table = (t - r.axis * per) * VE;
    r.a = r.axis * S + r.table;
    r.b = r.a + S / 2;
  }
  return r;
}

// Rotates the lane's pairs by the cosines c and sines s of their angles.
template <int VE>
__device__ __forceinline__ void rotate(const RotParams& p, const float (&c)[VE], const float (&s)[VE], float (&u)[VE],
                                       float (&v)[VE]) {
  if (p.interleaved) {
    if constexpr (VE > 1) {
      // pairs lie side by side: VE / 2 of them in each vector, their angles consecutive over both
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) {
        const float a0 = u[2 * e], a1 = u[2 * e + 1], b0 = v[2 * e], b1 = v[2 * e + 1];
        u[2 * e] = a0 * c[e] - a1 * s[e];
        u[2 * e + 1] = a1 * c[e] + a0 * s[e];
        v[2 * e] = b0 * c[VE / 2 + e] - b1 * s[VE / 2 + e];
        v[2 * e + 1] = b1 * c[VE / 2 + e] + b0 * s[VE / 2 + e];
      }
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const float a = u[e], b = v[e];
    u[e] = a * c[e] - b * s[e];
    v[e] = b * c[e] + a * s[e];
  }
}

template <typename T>
__device__ inline T* rot_ptr(const RotParams& p, const RotTensor& t, int clip, int token, int head) {
  return (T*)t.ptr + ((int64_t)clip * t.clip + (int64_t)token * t.token + (int64_t)head * t.head);
}

// Table row of a section's position; positions outside the table are taken to its ends.
__device__ inline int64_t rot_table(const RotParams& p, const RotLane& l, int low, int high) {
  int64_t pos = p.pos_step == 2 ? (int64_t)(((uint64_t)(uint32_t)high << 32) | (uint32_t)low) : (int64_t)low;
  pos = pos < 0 ? 0 : pos >= p.positions ? p.positions - 1 : pos;
  return pos * (p.rot / p.axes / 2) + l.table;
}

// What a lane has read ahead of a row.
template <typename T, int VE>
struct RotRow {
  typedef T vec __attribute__((ext_vector_type(VE)));
  vec u, v, du, dv;
  int low, high;  // position
  T* out;         // null: no row
};

template <typename T, typename TP, int VE, int TPR, bool BWD>
__global__ void __launch_bounds__(256) head_rotary_kernel(const RotParams p) {
  constexpr int kRows = 256 / TPR;
  typedef T vec __attribute__((ext_vector_type(VE)));
  __shared__ float sums[BWD ? 256 * VE : 1];
  const int part = bid_x() / p.groups, group = bid_x() - part * p.groups;
  const int lane = tid_x() % TPR, slot = tid_x() / TPR;
  const RotLane l = rot_lane<VE>(p, lane);
  // the lane's place in a step: token `ahead` of its first one, head (blocks > 1: of each block)
  const int ahead = p.blocks > 1 ? 0 : slot / p.heads, head0 = slot - ahead * p.heads;
  const bool on = l.on && ahead < p.per;
  RotTensor x = p.x, dy = p.dy, y = p.y;
  x.ptr += group * x.group * (int64_t)sizeof(T);
  dy.ptr += group * dy.group * (int64_t)sizeof(T);
  y.ptr += group * y.group * (int64_t)sizeof(T);
  float wa[VE], wb[VE], ba[VE], bb[VE];
  float dwa[VE], dwb[VE], dba[VE], dbb[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    wa[e] = wb[e] = 1.f;
    ba[e] = bb[e] = dwa[e] = dwb[e] = dba[e] = dbb[e] = 0.f;
  }
  if ((BWD || p.norm) && l.on) {
    const int64_t c = (int64_t)group * p.dim;
    load_param<VE, TP>(p.w, c + l.a, 1.f, wa);
    load_param<VE, TP>(p.w, c + l.b, 1.f, wb);
    if constexpr (!BWD) {
      load_param<VE, TP>(p.b, c + l.a, 0.f, ba);
      load_param<VE, TP>(p.b, c + l.b, 0.f, bb);
    }
  }
  auto fetch = [&](int unit) {
    RotRow<T, VE> r;
    r.u = r.v = r.du = r.dv = vec{};
    r.low = r.high = 0;
    r.out = nullptr;
    const int first = p.blocks > 1 ? unit / p.blocks : unit * p.per;
    const int head = head0 + (p.blocks > 1 ? (unit - first * p.blocks) * kRows : 0);
    int token = first + ahead, clip = 0;
    if (!on || unit >= p.units || token >= p.n || head >= p.heads) return r;
    if (l.axis >= 0) {
      const int32_t* w = p.pos + ((int64_t)token * p.axes + l.axis) * p.pos_step;
      r.low = w[0];
      r.high = w[p.pos_step - 1];  // (int32: the same word)
    }
    if (!p.flat) {
      clip = token / p.tokens;
      token -= clip * p.tokens;
    }
    const T* xp = rot_ptr<T>(p, x, clip, token, head);
    r.u = *reinterpret_cast<const vec*>(xp + l.a);
    r.v = *reinterpret_cast<const vec*>(xp + l.b);
    if constexpr (BWD) {
      const T* gp = rot_ptr<T>(p, dy, clip, token, head);
      r.du = *reinterpret_cast<const vec*>(gp + l.a);
      r.dv = *reinterpret_cast<const vec*>(gp + l.b);
    }
    r.out = rot_ptr<T>(p, y, clip, token, head);
    return r;
  };
  const float inv_n = 1.f / (float)p.dim;
  RotRow<T, VE> next = fetch(part);
  for (int unit = part; unit < p.units; unit += p.parts) {
    const RotRow<T, VE> r = next;
    if (unit + p.parts < p.units) next = fetch(unit + p.parts);
    const bool there = r.out != nullptr, turn = there && l.axis >= 0;
    float c[VE], sn[VE];  // read before they are needed: the row's statistics come first
    if (turn) {
      const int64_t at = rot_table(p, l, r.low, r.high);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        c[e] = p.cosine[at + e];
        sn[e] = (BWD ? -1.f : p.sign) * p.sine[at + e];
      }
    }
    float u[VE], v[VE], du[VE], dv[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      u[e] = (float)r.u[e];
      v[e] = (float)r.v[e];
      du[e] = (float)r.du[e];
      dv[e] = (float)r.dv[e];
    }
    float rstd = 0.f;
    if (BWD || p.norm) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e) s += u[e] + v[e];
      const float mean = lanes_sum<TPR>(s) * inv_n;
      s = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        u[e] -= mean;
        v[e] -= mean;
        s += u[e] * u[e] + v[e] * v[e];
      }
      s = lanes_sum<TPR>(l.on ? s : 0.f);
      if (there) rstd = inv_sqrt(s * inv_n + p.eps);  // (eps may be zero: no row, no infinity)
    }
    if constexpr (!BWD) {
      if (p.norm) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          u[e] = u[e] * rstd * wa[e] + ba[e];
          v[e] = v[e] * rstd * wb[e] + bb[e];
        }
      }
      if (turn) rotate<VE>(p, c, sn, u, v);
      if (there) {
        store_vec<VE>(r.out + l.a, u);
        store_vec<VE>(r.out + l.b, v);
      }
    } else {
      if (turn) rotate<VE>(p, c, sn, du, dv);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e) {  // (lanes without a row hold zeros in du, dv)
        u[e] *= rstd;
        v[e] *= rstd;
        dwa[e] += du[e] * u[e];
        dwb[e] += dv[e] * v[e];
        dba[e] += du[e];
        dbb[e] += dv[e];
        du[e] *= wa[e];
        dv[e] *= wb[e];
        s1 += du[e] + dv[e];
        s2 += du[e] * u[e] + dv[e] * v[e];
      }
      const float m1 = lanes_sum<TPR>(s1) * inv_n, m2 = lanes_sum<TPR>(s2) * inv_n;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        du[e] = rstd * (du[e] - m1 - u[e] * m2);
        dv[e] = rstd * (dv[e] - m1 - v[e] * m2);
      }
      if (there) {
        store_vec<VE>(r.out + l.a, du);
        store_vec<VE>(r.out + l.b, dv);
      }
    }
  }
  if constexpr (BWD) {
    if (!p.part) return;
    const int n = p.groups * p.dim;
    float* out = p.part + (int64_t)part * 2 * n + group * p.dim;
    const bool store = slot == 0 && l.on;
    add_slots<VE, TPR>(dwa, sums);
    if (store) store_vec<VE>(out + l.a, dwa);
    add_slots<VE, TPR>(dwb, sums);
    if (store) store_vec<VE>(out + l.b, dwb);
    add_slots<VE, TPR>(dba, sums);
    if (store) store_vec<VE>(out + n + l.a, dba);
    add_slots<VE, TPR>(dbb, sums);
    if (store) store_vec<VE>(out + n + l.b, dbb);
  }
}

constexpr int kRotMaxDim = 128;

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Vector width: 8 or 4 elements where every vector is whole and aligned, else single elements.
static int rot_vec(const RotParams& p, int type, std::initializer_list<const RotTensor*> tensors) {
  const int size = type == SAF3R_FP32 ? 4 : 2;
  for (int ve : {8, 4}) {
    // a lane's vector is one load of up to 16 bytes: eight 16-bit elements or four fp32
    if (ve * size > 16) continue;
    bool ok = (p.dim - p.rot) % (2 * ve) == 0;
    if (p.rot) {
      const int S = p.rot / p.axes;
      ok = ok && S % (2 * ve) == 0;
    }
    for (const RotTensor* t : tensors)
      ok = ok && (!t->ptr || ((uintptr_t)t->ptr % (ve * size) == 0 && t->clip % ve == 0 && t->token % ve == 0 &&
                              t->group % ve == 0 && t->head % ve == 0));
    ok = ok && (uintptr_t)p.w % 16 == 0 && (uintptr_t)p.b % 16 == 0 && (uintptr_t)p.part % 16 == 0;
    if (ok) return ve;
  }
  return 1;
}

template <typename F>
static int rot_dispatch(int type, int param_type, int ve, int dim, F f) {
  auto lanes = [&](auto t, auto tp, auto v) {
    const int n = dim / (2 * decltype(v)::value);
    if (n <= 2) return f(t, tp, v, Int<2>());
    if (n <= 4) return f(t, tp, v, Int<4>());
    if (n <= 8) return f(t, tp, v, Int<8>());
    if (n <= 16) return f(t, tp, v, Int<16>());
    if (n <= 32) return f(t, tp, v, Int<32>());
    return f(t, tp, v, Int<64>());
  };
  auto vecs = [&](auto t, auto tp) {
    if constexpr (sizeof(t) == 2)
      if (ve == 8) return lanes(t, tp, Int<8>());
    if (ve == 4) return lanes(t, tp, Int<4>());
    return lanes(t, tp, Int<1>());
  };
  auto rows = [&](auto t) { return param_type == SAF3R_FP32 ? vecs(t, float()) : vecs(t, t); };
  if (type == SAF3R_FP32) return vecs(float(), float());
  if (type == SAF3R_BF16) return rows(__bf16());
  return rows(_Float16());
}

static int rot_check(const char* who, RotParams* p, int type, int64_t clips, int tokens, int groups, int heads, int dim,
                     const void* pos, int pos_int64, int axes, const float* rope_cos, const float* rope_sin,
                     int positions, int rotary_dim, int interleaved, int norm, int param_type, float eps) {
  if (clips < 0 || tokens < 0 || groups <= 0 || heads <= 0 || dim <= 0)
    return fail(SAF3R_ERR_INVALID, "%s: invalid sizes: %lld clips, %d tokens, %d groups, %d heads, rows of %d", who,
                (long long)clips, tokens, groups, heads, dim);
  if (dim > kRotMaxDim || dim % 2)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: rows of %d (even, at most %d)", who, dim, kRotMaxDim);
  if (groups > 64) return fail(SAF3R_ERR_UNSUPPORTED, "%s: %d groups (at most 64)", who, groups);
  const int64_t most = 0x7fffffff - 65536;  // rows of a group are counted in 32 bits, a step beyond the last included
  if (clips > most || clips * tokens > most || clips * tokens * heads > most)
    return fail(SAF3R_ERR_UNSUPPORTED, "%s: too many rows for one launch", who);
  for (int t : {type, param_type})
    if (t < SAF3R_FP32 || t > SAF3R_FP16) return fail(SAF3R_ERR_INVALID, "%s: unknown element type %d", who, t);
  if (rope_cos) {
    if (!rope_sin || (!pos && clips * tokens > 0) || positions <= 0)
      return fail(SAF3R_ERR_INVALID, "%s: rotary positions need positions and both tables", who);
    if (axes < 1 || axes > 8 || rotary_dim <= 0 || rotary_dim > dim || rotary_dim % (2 * axes))
      return fail(SAF3R_ERR_INVALID, "%s: rotary_dim %d of %d over %d axes", who, rotary_dim, dim, axes);
    if ((uintptr_t)pos % (pos_int64 ? 8 : 4) || ((uintptr_t)rope_cos | (uintptr_t)rope_sin) % 4)
      return fail(SAF3R_ERR_INVALID, "%s: positions and tables must be aligned to their elements", who);
  }
  if (norm && !(eps >= 0.f && eps < 3.0e38f))
    return fail(SAF3R_ERR_INVALID, "%s: eps must be finite and not negative", who);
  if (int e = param_check(who, param_type, type)) return e;
  p->pos = (const int32_t*)pos;
  p->cosine = rope_cos;
  p->sine = rope_sin;
  p->n = (int)(clips * tokens);
  p->tokens = tokens;
  p->heads = heads;
  p->groups = groups;
  p->dim = dim;
  p->rot = rope_cos ? rotary_dim : 0;
  p->axes = rope_cos ? axes : 1;
  p->positions = positions;
  p->pos_step = pos_int64 ? 2 : 1;
  p->interleaved = interleaved != 0;
  p->norm = norm != 0;
  p->eps = eps;
  p->sign = 1.f;
  return SAF3R_OK;
}

static RotTensor rot_tensor(const saf3r_heads* h) {
  if (!h) return RotTensor{};
  return {(char*)const_cast<void*>(h->ptr), h->clip_stride, h->token_stride, h->group_stride, h->head_stride};
}

// Whether rows that are written would lie on each other (a stride of zero).
static bool rot_overlaps(const RotTensor& t, const RotParams& p, int64_t clips) {
  return (t.clip == 0 && clips > 1) || (t.token == 0 && p.tokens > 1) || (t.group == 0 && p.groups > 1) ||
         (t.head == 0 && p.heads > 1);
}

// Whether a tensor's clips follow each other as its tokens do.
static bool rot_flat(const RotTensor& t, int clips, int tokens) {
  return !t.ptr || clips <= 1 || t.clip == t.token * tokens;
}

// Steps of `rows` rows: whole tokens, or parts of a token's heads where those are more.
static int rot_units(const RotParams& p, int rows, int* per, int* blocks) {
  *blocks = (int)ceil_div(p.heads, rows);
  *per = *blocks > 1 ? 1 : rows / p.heads;
  return (int)(*blocks > 1 ? (int64_t)p.n * *blocks : ceil_div(p.n, *per));
}

// Work-groups of a group: as many as run at once, four a compute unit, or three in the backward pass with its sums, and
// there at least four steps each (the sums are small then next to the rows). 21984 tokens, bf16, forward / backward: 31
// and 54 us; with two to three a unit 32 and 57, with six 33 and 58, with sixteen and eight 36 and 62.
static int64_t rot_parts(int64_t units, int groups, bool sums) {
  const int64_t most = std::max<int64_t>(1, (sums ? 768 : 1024) / groups);
  return std::max<int64_t>(1, std::min<int64_t>(most, sums ? (units + 3) / 4 : units));
}

static void rot_steps(RotParams* p, int64_t clips, int rows) {
  p->units = rot_units(*p, rows, &p->per, &p->blocks);
  p->parts = (int)rot_parts(p->units, p->groups, p->part != nullptr);
  p->flat = rot_flat(p->x, (int)clips, p->tokens) && rot_flat(p->dy, (int)clips, p->tokens) &&
            rot_flat(p->y, (int)clips, p->tokens);
}

// The forward kernel from p->x to p->y.
static int rot_forward(const char* who, RotParams* p, int type, int param_type, int64_t clips, hipStream_t stream) {
  return rot_dispatch(type, param_type, rot_vec(*p, type, {&p->x, &p->y}), p->dim,
                      [&](auto t, auto tp, auto ve, auto tpr) {
    constexpr int kTpr = decltype(tpr)::value;
    rot_steps(p, clips, 256 / kTpr);
    hipLaunchKernelGGL((head_rotary_kernel<decltype(t), decltype(tp), decltype(ve)::value, kTpr, false>),
                       dim3((uint32_t)(p->parts * p->groups)), dim3(256), 0, stream, *p);
    return check_launch(who);
  });
}

}  // namespace saf3r

using namespace saf3r;

extern "C" int saf3r_head_rotary_fwd(const saf3r_heads* x, int type, int64_t clips, int tokens, int groups, int heads,
                                     int dim, const void* pos, int pos_int64, int axes, const float* rope_cos,
                                     const float* rope_sin, int positions, int rotary_dim, int interleaved, int norm,
                                     const void* weight, const void* bias, int param_type, float eps,
                                     const saf3r_heads* y, void* stream) {
  const char* who = "saf3r_head_rotary_fwd";
  if (int e = injected(who)) return e;
  RotParams p{};
  if (int e = rot_check(who, &p, type, clips, tokens, groups, heads, dim, pos, pos_int64, axes, rope_cos, rope_sin,
                        positions, rotary_dim, interleaved, norm, param_type, eps))
    return e;
  if (p.n == 0) return SAF3R_OK;
  p.x = rot_tensor(x);
  p.y = rot_tensor(y);
  if (!p.x.ptr || !p.y.ptr) return fail(SAF3R_ERR_INVALID, "%s: null tensor pointer", who);
  const int size = type == SAF3R_FP32 ? 4 : 2;
  if (((uintptr_t)p.x.ptr | (uintptr_t)p.y.ptr) % size)
    return fail(SAF3R_ERR_INVALID, "%s: rows must be aligned to their elements", who);
  if (rot_overlaps(p.y, p, clips)) return fail(SAF3R_ERR_INVALID, "%s: written rows overlap (a stride of zero)", who);
  if (norm) {
    p.w = weight;
    p.b = bias;
  }
  return rot_forward(who, &p, type, param_type, clips, (hipStream_t)stream);
}

extern "C" int64_t saf3r_head_rotary_bwd_workspace_bytes(int64_t clips, int tokens, int groups, int heads, int dim) {
  const char* who = "saf3r_head_rotary_bwd_workspace_bytes";
  RotParams p{};
  if (rot_check(who, &p, SAF3R_FP32, clips, tokens, groups, heads, dim, nullptr, 0, 1, nullptr, nullptr, 0, 0, 0, 0,
                SAF3R_FP32, 0.f))
    return -1;
  int per, blocks;
  // the fewest rows of a step are four
  return rot_parts(rot_units(p, 4, &per, &blocks), groups, true) * 2 * groups * dim * 4;
}

extern "C" int saf3r_head_rotary_bwd(const saf3r_heads* dy, const saf3r_heads* x, int type, int64_t clips, int tokens,
                                     int groups, int heads, int dim, const void* pos, int pos_int64, int axes,
                                     const float* rope_cos, const float* rope_sin, int positions, int rotary_dim,
                                     int interleaved, int norm, const void* weight, int param_type, float eps,
                                     const saf3r_heads* dx, void* dweight, void* dbias, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  const char* who = "saf3r_head_rotary_bwd";
  if (int e = injected(who)) return e;
  RotParams p{};
  if (int e = rot_check(who, &p, type, clips, tokens, groups, heads, dim, pos, pos_int64, axes, rope_cos, rope_sin,
                        positions, rotary_dim, interleaved, norm, param_type, eps))
    return e;
  const bool params = norm && (dweight || dbias);
  const int64_t need = params ? saf3r_head_rotary_bwd_workspace_bytes(clips, tokens, groups, heads, dim) : 0;
  if (workspace_bytes < need || (need > 0 && (!workspace || (uintptr_t)workspace % 16)))
    return fail(SAF3R_ERR_INVALID, "%s: workspace of %lld bytes: %lld, 16-byte aligned, are needed", who,
                (long long)workspace_bytes, (long long)need);
  int64_t parts = 0;
  int rc = SAF3R_OK;
  if (p.n > 0) {
    p.dy = rot_tensor(dy);
    p.x = norm ? rot_tensor(x) : RotTensor{};
    p.y = rot_tensor(dx);
    if (!p.dy.ptr || !p.y.ptr || (norm && !p.x.ptr)) return fail(SAF3R_ERR_INVALID, "%s: null tensor pointer", who);
    const int size = type == SAF3R_FP32 ? 4 : 2;
    if (((uintptr_t)p.x.ptr | (uintptr_t)p.y.ptr | (uintptr_t)p.dy.ptr) % size)
      return fail(SAF3R_ERR_INVALID, "%s: rows must be aligned to their elements", who);
    if (rot_overlaps(p.y, p, clips)) return fail(SAF3R_ERR_INVALID, "%s: written rows overlap (a stride of zero)", who);
    if (!norm) {  // the inverse rotation is all there is
      p.x = p.dy;
      p.dy = RotTensor{};
      p.sign = -1.f;
      return rot_forward(who, &p, type, param_type, clips, (hipStream_t)stream);
    }
    p.w = weight;
    if (params) p.part = (float*)workspace;
    rc = rot_dispatch(type, param_type, rot_vec(p, type, {&p.x, &p.dy, &p.y}), dim,
                      [&](auto t, auto tp, auto ve, auto tpr) {
      constexpr int kTpr = decltype(tpr)::value;
      rot_steps(&p, clips, 256 / kTpr);
      parts = p.parts;
      hipLaunchKernelGGL((head_rotary_kernel<decltype(t), decltype(tp), decltype(ve)::value, kTpr, true>),
                         dim3((uint32_t)(parts * groups)), dim3(256), 0, (hipStream_t)stream, p);
      return check_launch(who);
    });
  }
  if (rc != SAF3R_OK || !params) return rc;
  return sum_parts(who, (const float*)workspace, parts, groups * dim, dweight, dbias, param_type, (hipStream_t)stream);
}
