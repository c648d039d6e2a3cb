// state_attend.hip -- attention of single query tokens over the 4-bit state cache.
//
// Row i has a query of q_heads heads and attends to the first len_i slots of its table row;
// query head a reads the K and V rows of head a / G, G = q_heads / heads:
//   x_j = scale * q . k_j,  p_j = exp(x_j - max x) / sum exp(x - max x),  out = sum_j p_j v_j.
// One pass over the slots with the running maximum m and sum l of the softmax, in 32 bits and
// base 2 (scale * log2 e goes into q).  Long rows are split into chunks of slots whose (m, l,
// sum p v) go through the workspace; the finishing kernel joins them.  When the caller keeps
// attention weights, the logits of every slot go through the workspace too and the finishing
// kernel adds the G heads' probabilities in head order: no atomics, so results do not vary.
//
// A slot past the length, or on a page outside the cache (reported), has logit -inf, and its scale
// and base are replaced by zeros before use: what lies there (NaN, infinities) is never multiplied.
#include "dgs_lane.cuh"
#include "dgs_state.cuh"

namespace dgs {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
  StateView c;
  const void *q;
  int64_t q_row, q_head;
  int64_t rows;
  int q_heads, g;  // g = query heads per head
  IdArray table, lens;
  int64_t width;
  float scale2;  // scale * log2 e
  int64_t chunk;  // slots per split
  int splits;
  float *part_o;   // [rows, q_heads, splits, dim], unnormalised (splits > 1)
  float2 *part_ml;  // [rows, q_heads, splits] (splits > 1 or weights)
  float *logits;   // [rows, q_heads, cap] (weights)
  int64_t cap;     // width << pshift
  float *weights;
  int64_t weights_cols;
  float decay;
  void *out;
  GatherGuard gd;
};

__device__ __forceinline__ int64_t row_length(const AttendArgs &a, int64_t row, bool report) {
  const int64_t len = a.lens[row];
  if ((uint64_t)len > (uint64_t)a.cap) {
    if (report) report_bad_id(a.gd.err, kAsyncErrLength, len, a.cap + 1, a.gd.tag);
    return len < 0 ? 0 : a.cap;
  }
  return len;
}

__device__ __forceinline__ void store_out(int type, void *out, int64_t elem, const float (&x)[8]) {
  if (type == kStateF32)
    store8<kStateF32>(out, elem, x);
  else if (type == kStateBF16)
    store8<kStateBF16>(out, elem, x);
  else
    store8<kStateF16>(out, elem, x);
}
__device__ __forceinline__ void load_q(int type, const void *q, int64_t elem, float (&x)[8]) {
  if (type == kStateF32)
    load8<kStateF32>(q, elem, x);
  else if (type == kStateBF16)
    load8<kStateBF16>(q, elem, x);
  else
    load8<kStateF16>(q, elem, x);
}

template <int LPR>
__device__ __forceinline__ float sum_lanes(float x) {
  if constexpr (LPR >= 2) x += lane_xor32<1>(x);
  if constexpr (LPR >= 4) x += lane_xor32<2>(x);
  if constexpr (LPR >= 8) x += lane_xor32<4>(x);
  if constexpr (LPR >= 16) x += lane_xor32<8>(x);
  if constexpr (LPR >= 32) x += lane_xor32<16>(x);
  return x;
}

// Vector form, for every type and size.  A work item is (row, head, GC query heads, split).  LPR
// lanes hold a row (eight channels each); SL groups of them take every SL-th slot with a softmax
// state of their own, joined at the end by exchanges between lanes.  kU slots a group are loaded
// while the kU before them are computed, ids another step ahead.  As in the matrix form, the
// running maximum is only followed when a logit passes it by 8.
// SL = 1 is for rows of at most 16 slots: no join, and with all query heads of a head in the item
// the probabilities stay in registers and the item writes its weights itself.
template <int LPR, int SL, int GC>
__global__ __launch_bounds__(kThreads) void k_attend_vec(AttendArgs a, int type, int gchunks,
                                                         int64_t items) {
  constexpr int kItem = LPR * SL, kU = 4, kStep = SL * kU;
  constexpr int kKeep = SL > 1 ? 1 : (LPR >= 16 ? 1 : 16 / LPR);
  const int lane = threadIdx.x & (kItem - 1);
  int64_t item64 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / kItem;
  if (item64 >= items) return;  // whole items leave together: no exchange crosses an item
  uint32_t item = (uint32_t)item64;
  const int sub = lane % LPR, sl = lane / LPR;
  const int split = (int)(item % (uint32_t)a.splits);
  item /= (uint32_t)a.splits;
  const int gc = (int)(item % (uint32_t)gchunks);
  item /= (uint32_t)gchunks;
  const int h = (int)(item % (uint32_t)a.c.heads);
  const int64_t row = item / (uint32_t)a.c.heads;
  const int words = a.c.dim >> 3;
  const bool live = sub < words;
  const int w = live ? sub : 0, ng = a.c.dim / a.c.group, grp = 8 * w / a.c.group;
  const int len = (int)row_length(a, row, split == 0 && h == 0 && gc == 0 && lane == 0);
  const int first = split * (int)a.chunk;
  if (split > 0 && first >= len) return;
  const int last = a.splits == 1 ? len : (int)(first + a.chunk < len ? first + a.chunk : len);
  const int a0 = h * a.g + gc * GC, gn = a.g - gc * GC < GC ? a.g - gc * GC : GC;

  float q[GC][8], o[GC][8], m[GC], l[GC], xs[kKeep][GC];
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    if (live && g < gn) {
      load_q(type, a.q, row * a.q_row + (a0 + g) * a.q_head + 8 * w, q[g]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[g][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[g][i] *= a.scale2;
      o[g][i] = 0.f;
    }
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) xs[i][g] = -INFINITY;
  }
  const int ps = a.c.pshift, mask = (1 << ps) - 1;
  const bool wide = a.table.bytes == 8;
  const char *tab = (const char *)a.table.p + ((row * a.width) << (wide ? 3 : 2));
  const uint32_t pages = (uint32_t)a.c.pages;
  uint32_t id[kU], id_hi[kU];
  struct Rows {
    uint32_t kq[kU], vq[kU], km[kU], vm[kU], ok;
  };
  Rows t;
  auto slot_of = [&](int j0, int u) {
    const int j = j0 + u * SL + sl;
    return j < last ? j : last - 1;
  };
  auto load_ids = [&](int j0) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const char *at = tab + ((int64_t)(slot_of(j0, u) >> ps) << (wide ? 3 : 2));
      id[u] = *(const uint32_t *)at;
      id_hi[u] = *(const uint32_t *)(at + (wide ? 4 : 0));
    }
  };
  auto load_rows = [&](int j0) {
    t.ok = 0;
    uint32_t page[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool in = j0 + u * SL + sl < last;
      const bool out = id[u] >= pages || (wide && id_hi[u] != 0);
      if (out && in && sub == 0)
        report_bad_id(a.gd.err, kAsyncErrSlot,
                      wide ? (int64_t)((uint64_t)id_hi[u] << 32 | id[u]) : (int64_t)(int32_t)id[u],
                      pages, a.gd.tag);
      page[u] = out ? 0u : id[u];
      t.ok |= (in && !out ? 1u : 0u) << u;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t r = (((int64_t)page[u] * a.c.heads + h) << ps) + (slot_of(j0, u) & mask);
      t.kq[u] = *(const uint32_t *)(a.c.kc + r * (a.c.dim >> 1) + 4 * w);
      t.vq[u] = *(const uint32_t *)(a.c.vc + r * (a.c.dim >> 1) + 4 * w);
      t.km[u] = a.c.ks[r * ng + grp];
      t.vm[u] = a.c.vs[r * ng + grp];
    }
  };
  auto compute = [&](const Rows &t, int j0, int keep) {
    float x[GC][kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool ok = (t.ok >> u) & 1;
      const uint32_t km = live ? t.km[u] : 0u;
      const float ks = scale_of(km), kb = base_of(km);
      float kv[8];
      codes8(t.kq[u], kv);
#pragma unroll
      for (int i = 0; i < 8; ++i) kv[i] = __builtin_fmaf(kv[i], ks, kb);
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(q[g][i], kv[i], s);
        s = sum_lanes<LPR>(s);
        x[g][u] = ok ? s : -INFINITY;
      }
    }
    if (SL == 1) {
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
          if ((keep + u) / LPR == i && (keep + u) % LPR == sub)
#pragma unroll
            for (int g = 0; g < GC; ++g) xs[i][g] = x[g][u];
    }
    if (a.logits && sub == 0) {
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (j0 + u * SL + sl < last)
#pragma unroll
          for (int g = 0; g < GC; ++g)
            if (g < gn) a.logits[(row * a.q_heads + a0 + g) * a.cap + j0 + u * SL + sl] = x[g][u];
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      float top = fmaxf(fmaxf(x[g][0], x[g][1]), fmaxf(x[g][2], x[g][3]));
      if (top > m[g] + 8.f) {
        const float f = __builtin_amdgcn_exp2f(m[g] - top);
        m[g] = top;
        l[g] *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[g][i] *= f;
      }
      const float ms = m[g] == -INFINITY ? 0.f : m[g];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        x[g][u] = __builtin_amdgcn_exp2f(x[g][u] - ms);
        l[g] += x[g][u];
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint32_t vm = live && ((t.ok >> u) & 1) ? t.vm[u] : 0u;
      const float vs = scale_of(vm), vb = base_of(vm);
      float vv[8];
      codes8(t.vq[u], vv);
#pragma unroll
      for (int i = 0; i < 8; ++i) vv[i] = __builtin_fmaf(vv[i], vs, vb);
#pragma unroll
      for (int g = 0; g < GC; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[g][i] = __builtin_fmaf(x[g][u], vv[i], o[g][i]);
    }
  };
  if (first < last) {
    load_ids(first);
    load_rows(first);
    load_ids(first + kStep);
    if constexpr (SL == 1) {
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (4 * st >= last) break;
        const Rows now = t;
        if (4 * st + 4 < last) {
          load_rows(4 * st + 4);
          load_ids(4 * st + 8);
        }
        compute(now, 4 * st, 4 * st);
      }
    } else {
#pragma unroll 1
      for (int j0 = first; j0 < last; j0 += kStep) {
        const Rows now = t;
        load_rows(j0 + kStep);
        load_ids(j0 + 2 * kStep);
        compute(now, j0, 0);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GC; ++g) {
#pragma unroll
    for (int s = LPR; s < kItem; s <<= 1) {
      const float mo = __shfl_xor(m[g], s, 64);
      const float mn = fmaxf(m[g], mo), ms = mn == -INFINITY ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f(m[g] - ms), fo = __builtin_amdgcn_exp2f(mo - ms);
      m[g] = mn;
      l[g] = l[g] * f + __shfl_xor(l[g], s, 64) * fo;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[g][i] = o[g][i] * f + __shfl_xor(o[g][i], s, 64) * fo;
    }
    if (g >= gn || sl != 0) continue;
    const int64_t qh = row * a.q_heads + a0 + g;
    if (a.splits > 1) {
      if (live) store8<kStateF32>(a.part_o, (qh * a.splits + split) * a.c.dim + 8 * w, o[g]);
    } else if (live) {
      const float inv = len == 0 ? 0.f : 1.f / l[g];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[g][i] *= inv;
      store_out(type, a.out, qh * a.c.dim + 8 * w, o[g]);
    }
    if (a.part_ml && sub == 0) a.part_ml[qh * a.splits + split] = make_float2(m[g], l[g]);
  }
  if constexpr (SL == 1) {
    if (a.weights && !a.logits) {  // every query head of this head is here
      float *wr = a.weights + (row * a.c.heads + h) * a.weights_cols;
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        const int j = i * LPR + sub;
        if (j >= len) continue;
        float sum = 0.f;
#pragma unroll
        for (int g = 0; g < GC; ++g)
          if (g < gn) {
            const float ms = m[g] == -INFINITY ? 0.f : m[g];
            sum += __builtin_amdgcn_exp2f(xs[i][g] - ms) * (1.f / l[g]);
          }
        wr[j] = a.decay != 0.f ? sum + a.decay * wr[j] : sum;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// Matrix form, for 16-bit queries.  One wave takes 16 query heads of a head (the unused ones are
// zeros) through 32 slots at a time, in v_mfma_f32_16x16x32_bf16 (operands: lane l holds row or
// column l & 15 and the eight k of quarter l >> 4; result: column l & 15, rows 4 (l >> 4) + i).
//
//  - A code c becomes the bfloat16 0x4300 | c = 128 + c, exactly, with one mask-or a pair.
//  - x = K q: rows are slots, columns query heads, k channels; one product chain per channel group,
//    r_g = sum q (128 + c).  Then x = sum_g s_g r_g + sum_g (b_g - 128 s_g) Q_g with Q_g = sum q over
//    the group; the second sum is one more product whose slot operand is the stored (s, b) words
//    themselves and whose other operand holds -128 Q_g and Q_g in three bfloat16 terms (24 bits).
//  - The result leaves four slots of one query head in a lane, which is what the second product
//    wants of its operand: p needs no exchange.  Which slot counts as which k is free; V follows.
//  - out = V p: rows are channels (16 units of GROUP / 16 channels of one group), columns query
//    heads, k slots.  a_g = p s_g is rounded to two bfloat16 terms (17 bits: one term's 2^-9 would
//    show in the output), and the 128 sum a_g that the codes' offset adds is taken out with the same
//    rounded terms, through a product with a constant operand.  sum p b_g is summed in 32 bits.
//    The pairs of slots that a register of V holds are made with v_perm_b32.
//  - Rows come in 16 bytes a lane, two tiles ahead in registers, and pass through the wave's own
//    corner of LDS, from which every lane takes its words: 26 narrow loads a tile straight to their
//    lanes kept the wave waiting (60 % of its time) and the texture unit half busy.  A row's 16-byte
//    pieces are stored in an order that depends on the row, so that the rows a read touches lie in
//    different banks.
//  - m only follows the maximum when a logit passes it by 8 (in base 2): p stays below 2^8, and
//    the rescaling is a rare branch.
// The waves of a workgroup take their 32 slots in turn and join through LDS in wave order.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
union Op {
  uint32_t u[4];
  bf16x8 v;
};

__device__ __forceinline__ f32x4 mfma(const Op &a, const Op &b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
// Two floats rounded to nearest even (one instruction).
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(lo), "v"(hi));
  return r;
}
// The low nibbles of a word's halves as bfloat16 128 + c.  `magic` is 0x43004300 in a vector
// register: one instruction takes one constant from a scalar register, so with both there the
// mask-or would be two.
__device__ __forceinline__ uint32_t code_pair(uint32_t x, uint32_t magic) {
  return (x & 0x000f000fu) | magic;
}
__device__ __forceinline__ float xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float((threadIdx.x & 16) ? r[0] : r[1]);
}
__device__ __forceinline__ float xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

template <int NG, int GROUP, int QT>
__global__ __launch_bounds__(512, 2) void k_attend_mfma(AttendArgs a, int type, int tiles) {
  constexpr int kD = NG * GROUP, kC = kD / 32, kU = GROUP / 16, kGC = GROUP / 32;
  extern __shared__ float s_mem[];
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, q4 = lane >> 4;
  uint32_t b = blockIdx.x;
  const int split = (int)(b % (uint32_t)a.splits);
  b /= (uint32_t)a.splits;
  const int rt = (int)(b % (uint32_t)tiles);
  b /= (uint32_t)tiles;
  const int h = (int)(b % (uint32_t)a.c.heads);
  const int64_t row = b / (uint32_t)a.c.heads;
  // slots of a row fit 32 bits (checked on the host)
  const int len = __builtin_amdgcn_readfirstlane(
      (int)row_length(a, row, split == 0 && h == 0 && rt == 0 && threadIdx.x == 0));
  const int chunk = (int)a.chunk, first = split * chunk;
  if (split > 0 && first >= len) return;
  const int last = a.splits == 1 ? len : (first + chunk < len ? first + chunk : len);
  const int gn = a.g - rt * 16 < 16 ? a.g - rt * 16 : 16;
  const int64_t qh0 = row * a.q_heads + h * a.g + rt * 16;
  // logits grow with x: a negative scale is taken into q
  const float sign = a.scale2 < 0.f ? -1.f : 1.f, scale2 = fabsf(a.scale2);
  uint32_t magic = 0x43004300u;
  asm volatile("" : "+v"(magic));

  // q in bfloat16 terms, in the order in which code_pair() yields a word's channels: 0 4 1 5 2 6 3 7
  Op qv[QT][kC], qm;
  float qsum[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) qsum[g] = 0.f;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n < gn)
      load_q(type, a.q, row * a.q_row + (h * a.g + rt * 16 + n) * a.q_head + 32 * c + 8 * q4, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] *= sign;
      qsum[c / kGC] += x[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t hi = pack_bf16(x[i], x[4 + i]);
      qv[0][c].u[i] = hi;
      if constexpr (QT == 2)
        qv[1][c].u[i] = pack_bf16(x[i] - __uint_as_float(hi << 16),
                                  x[4 + i] - __uint_as_float(hi & 0xffff0000u));
    }
  }
  // quarter 0 holds the first bfloat16 terms of (-128 Q_g, Q_g), 1 the second, 2 the third
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    qm.u[g] = 0;
    if (g < NG) {
      float s = qsum[g < NG ? g : 0];
      s += xor16(s);
      s += xor32(s);
      const float t0 = (float)(__bf16)s, t1 = (float)(__bf16)(s - t0);
      const float t2 = (s - t0) - t1;
      const float t = q4 == 0 ? t0 : (q4 == 1 ? t1 : (q4 == 2 ? t2 : 0.f));
      qm.u[g] = pack_bf16(-128.f * t, t);
    }
  }

  f32x4 o[NG][kU], co[NG];
  float cb[NG], m = -INFINITY, ms = 0.f, l = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    co[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    cb[g] = 0.f;
#pragma unroll
    for (int j = 0; j < kU; ++j) o[g][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  Op ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) ones.u[i] = 0x43004300u;  // 128, the codes' offset

  const int ps = a.c.pshift, mask = (1 << ps) - 1;
  const int64_t trow = row * a.width;
  const int unit = n * (GROUP / 32);  // byte of this lane's unit of V in a group's codes
  const uint32_t sel = GROUP == 128 ? 0x05040100u
                       : GROUP == 64 ? ((unit & 2) ? 0x07060302u : 0x05040100u)
                                     : (0x0c000c00u | (uint32_t)(unit & 3) |
                                        ((uint32_t)(4 + (unit & 3)) << 16));
  const int step = waves * 32;
  const uint32_t pages = (uint32_t)a.c.pages;

  // A tile is kPR x 64 pieces of 16 bytes: those of K, then those of V, row by row.  kL loads of a
  // lane; load i of the first kL / 2 (kPR = 1: the lower half of the wave) belongs to K.  kRows rows
  // a load; a lane meets kIds different slots.
  constexpr int kPR = kD / 32, kL = kPR < 2 ? 1 : kPR, kRows = 64 / kPR > 32 ? 32 : 64 / kPR;
  constexpr int kIds = 32 / kRows;
  // the words of a row: NG of K, NG of V; kPR lanes of the row fetch them in kW loads
  constexpr int kW = (2 * NG + kPR - 1) / kPR;
  // Piece p of row r lies at p ^ key(r) (in its low two bits): rows that share banks differ.
  auto key = [](int r) { return kPR == 1 ? 0 : (kPR == 2 ? (r >> 3) & 1 : (r >> 2) & 3); };
  su32x4 *s_c = (su32x4 *)s_mem + wave * (kPR * 64 + NG * 16);  // codes of K, then of V
  uint32_t *s_w = (uint32_t *)(s_c + kPR * 64);                 // words of K, then of V
  const int lrow = (lane / kPR) % kRows, lpiece = lane % kPR;
  // where this lane finds its words of K (chunk c: kp[c & 3]) and of V (group g: vp[g % kVP]); the
  // keys of its rows 16 i + n and 16 i + 4 q4 + y do not depend on i and y
  constexpr int kKP = kPR < 4 ? kPR : 4, kVP = GROUP == 128 ? 1 : (GROUP == 64 ? 2 : 4);
  const char *kp[kKP], *vp[kVP];
#pragma unroll
  for (int c = 0; c < kKP; ++c) kp[c] = (const char *)(s_c + n * kPR + (c ^ key(n))) + 4 * q4;
#pragma unroll
  for (int g = 0; g < kVP; ++g) {
    const int p = g * (GROUP / 32) + (unit >> 4);
    vp[g] = (const char *)(s_c + 32 * kPR + 4 * q4 * kPR + (p ^ key(4 * q4))) + (unit & 12);
  }
  struct Rows {
    su32x4 c[kL];
    uint32_t w[kIds][kW];
    uint64_t bad[kIds];  // lanes whose page lies outside the cache
  };
  Rows t0, t1;
  // pages of the next tile's slots, as read (low and high words; looked at when its rows are
  // loaded, without a branch on the table's type, which would wait for every load before it)
  uint32_t id[kIds], id_hi[kIds];
  const bool wide = a.table.bytes == 8;
  const char *tab = (const char *)a.table.p + (trow << (wide ? 3 : 2));

  auto slot_of = [&](int j0, int i) {
    const int j = j0 + i * kRows + lrow;
    return j < last ? j : last - 1;
  };
  auto load_ids = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      const char *at = tab + ((int64_t)(slot_of(j0, i) >> ps) << (wide ? 3 : 2));
      id[i] = *(const uint32_t *)at;
      id_hi[i] = *(const uint32_t *)(at + (wide ? 4 : 0));
    }
  };
  // Loads tile j0's rows, and before them the ids of tile j0 + step: memory returns in order, so
  // whoever waits for an id would wait for rows issued before it.
  auto load_rows = [&](int j0, Rows &t) {
    uint32_t page[kIds];
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      const bool out = id[i] >= pages || (wide && id_hi[i] != 0);
      if (out)
        report_bad_id(a.gd.err, kAsyncErrSlot,
                      wide ? (int64_t)((uint64_t)id_hi[i] << 32 | id[i]) : (int64_t)(int32_t)id[i],
                      pages, a.gd.tag);
      page[i] = out ? 0u : id[i];
      t.bad[i] = __ballot(out);
    }
    load_ids(j0 + step);
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      const int64_t r = (((int64_t)page[i] * a.c.heads + h) << ps) + (slot_of(j0, i) & mask);
      if constexpr (kPR == 1) {
        t.c[0] = *(const su32x4 *)((lane < 32 ? a.c.kc : a.c.vc) + r * 16);
      } else {
        t.c[i] = *(const su32x4 *)(a.c.kc + r * (kD / 2) + 16 * lpiece);
        t.c[kIds + i] = *(const su32x4 *)(a.c.vc + r * (kD / 2) + 16 * lpiece);
      }
#pragma unroll
      for (int y = 0; y < kW; ++y) {
        // word e of the row's 2 NG (kPR = 1: the lower lanes fetch K's, the upper V's)
        const int e = kPR == 1 ? (lane < 32 ? y : NG + y) : lpiece + y * kPR;
        const uint32_t *wp = e < NG ? a.c.ks : a.c.vs;
        t.w[i][y] = e < 2 * NG ? wp[r * NG + (e < NG ? e : e - NG)] : 0u;
      }
    }
  };
  auto stage = [&](const Rows &t) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      const int r = i * kRows + lrow;
      if constexpr (kPR == 1) {
        s_c[(lane < 32 ? 0 : 32) + r] = t.c[0];
      } else {
        s_c[r * kPR + (lpiece ^ key(r))] = t.c[i];
        s_c[(32 + r) * kPR + (lpiece ^ key(r))] = t.c[kIds + i];
      }
#pragma unroll
      for (int y = 0; y < kW; ++y) {
        const int e = kPR == 1 ? (lane < 32 ? y : NG + y) : lpiece + y * kPR;
        if (e < 2 * NG) s_w[e < NG ? r * NG + e : (32 + r) * NG + e - NG] = t.w[i][y];
      }
    }
    __builtin_amdgcn_wave_barrier();
  };
  auto compute = [&](int j0, const uint64_t *bad) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      Op av;
#pragma unroll
      for (int g = 0; g < 4; ++g) av.u[g] = g < NG ? s_w[(16 * i + n) * NG + (g < NG ? g : 0)] : 0u;
      f32x4 s = mfma(av, qm, f32x4{0.f, 0.f, 0.f, 0.f});
      su32x4 kw[NG];
#pragma unroll
      for (int y = 0; y < NG; ++y)
        kw[y] = *(const su32x4 *)(s_w + (16 * i + 4 * q4) * NG + 4 * y);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 r = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = g * kGC; c < (g + 1) * kGC; ++c) {
          const uint32_t w = *(const uint32_t *)(kp[c % kKP] + 256 * kPR * i + 64 * (c / 4));
          Op k;
#pragma unroll
          for (int y = 0; y < 4; ++y) k.u[y] = code_pair(w >> (4 * y), magic);
          r = mfma(k, qv[0][c], r);
          if constexpr (QT == 2) r = mfma(k, qv[1][c], r);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
          s[y] = __builtin_fmaf(scale_of(kw[(y * NG + g) / 4][(y * NG + g) % 4]), r[y], s[y]);
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) x[4 * i + y] = s[y];
    }
    su32x4 vw[2 * NG];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int y = 0; y < NG; ++y)
        vw[NG * i + y] = *(const su32x4 *)(s_w + (32 + 16 * i + 4 * q4) * NG + 4 * y);
    bool some = false;
#pragma unroll
    for (int i = 0; i < kIds; ++i) some |= bad[i] != 0;
    if (j0 + 32 > last || some) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 16 * (i >> 2) + 4 * q4 + (i & 3);
        bool out = j0 + r >= last;
        if (some)
#pragma unroll
          for (int y = 0; y < kIds; ++y)
            out |= r / kRows == y && ((bad[y] >> ((r % kRows) * (kPR == 1 ? 1 : kPR))) & 1);
        if (out) {
          x[i] = -INFINITY;
#pragma unroll
          for (int g = 0; g < NG; ++g) vw[(i * NG + g) / 4][(i * NG + g) % 4] = 0;
        }
      }
    }
    if (a.logits && n < gn) {
      float *lp = a.logits + (qh0 + n) * a.cap + j0 + 4 * q4;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if ((a.cap & 3) == 0) {  // whole quads fit
          if (j0 + 16 * i + 4 * q4 < last)
            *(f32x4 *)(lp + 16 * i) =
                f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]} * scale2;
        } else {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (j0 + 16 * i + 4 * q4 + y < last) lp[16 * i + y] = x[4 * i + y] * scale2;
        }
      }
    }
    // m and ms in units of base 2
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    top *= scale2;
    if (__any(top > m + 8.f)) {
      top = fmaxf(top, xor16(top));
      top = fmaxf(top, xor32(top));
      const float mn = fmaxf(m, top);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      ms = mn == -INFINITY ? 0.f : mn;
      l *= f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        cb[g] *= f;
        co[g] *= f;
#pragma unroll
        for (int j = 0; j < kU; ++j) o[g][j] *= f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], scale2, -ms));
      l += x[i];
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t vq[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        vq[i] = *(const uint32_t *)(vp[g % kVP] + 16 * kPR * (16 * (i >> 2) + (i & 3)) +
                                    64 * (g / kVP));
      Op hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w0 = vw[(2 * i * NG + g) / 4][(2 * i * NG + g) % 4];
        const uint32_t w1 = vw[((2 * i + 1) * NG + g) / 4][((2 * i + 1) * NG + g) % 4];
        cb[g] = __builtin_fmaf(x[2 * i], base_of(w0), cb[g]);
        cb[g] = __builtin_fmaf(x[2 * i + 1], base_of(w1), cb[g]);
        const float a0 = x[2 * i] * scale_of(w0), a1 = x[2 * i + 1] * scale_of(w1);
        hi.u[i] = pack_bf16(a0, a1);
        lo.u[i] = pack_bf16(a0 - __uint_as_float(hi.u[i] << 16),
                            a1 - __uint_as_float(hi.u[i] & 0xffff0000u));
      }
      co[g] = mfma(ones, hi, co[g]);
      co[g] = mfma(ones, lo, co[g]);
      uint32_t pair[GROUP == 128 ? 2 : 1][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pair[0][i] = __builtin_amdgcn_perm(vq[2 * i + 1], vq[2 * i], sel);
        if constexpr (GROUP == 128)
          pair[1][i] = __builtin_amdgcn_perm(vq[2 * i + 1], vq[2 * i], 0x07060302u);
      }
#pragma unroll
      for (int j = 0; j < kU; ++j) {
        Op v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v.u[i] = code_pair(pair[j >> 2][i] >> (4 * (j & 3)), magic);
        o[g][j] = mfma(v, hi, o[g][j]);
        o[g][j] = mfma(v, lo, o[g][j]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  };

  // Two tiles a turn, each staged from its own registers, which then take the tile after the next.
  // Tiles past the end load the last slot again and are masked whole: without conditions in the
  // loop the accumulators keep one set of registers.
  auto turn = [&](int j0, Rows &t) {
    stage(t);
    uint64_t bad[kIds];
#pragma unroll
    for (int i = 0; i < kIds; ++i) bad[i] = t.bad[i];
    load_rows(j0 + 2 * step, t);
    compute(j0, bad);
  };
  const int j1 = first + wave * 32;
  if (j1 < last) {
    load_ids(j1);
    load_rows(j1, t0);
    load_rows(j1 + step, t1);
#pragma unroll 1
    for (int j0 = j1; j0 < last; j0 += 2 * step) {
      turn(j0, t0);
      turn(j0 + step, t1);
    }
  }

  __syncthreads();  // the corners become the joining area
  // join the waves: [waves][16] maxima, [waves][16] sums, [waves][gn][kD] outputs
  l += xor16(l);
  l += xor32(l);
  float *s_m = s_mem, *s_l = s_mem + waves * 16, *s_o = s_mem + waves * 32;
  if (q4 == 0) s_m[wave * 16 + n] = m;
  __syncthreads();
  float all = -INFINITY;
  for (int w = 0; w < waves; ++w) all = fmaxf(all, s_m[w * 16 + n]);
  const float f = __builtin_amdgcn_exp2f(m - (all == -INFINITY ? 0.f : all));
  if (q4 == 0) s_l[wave * 16 + n] = l * f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float c = cb[g];
    c += xor16(c);
    c += xor32(c);
    if (n < gn) {
      float *dst = s_o + (wave * gn + n) * kD + g * GROUP + 4 * q4 * kU;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kU; ++j) dst[i * kU + j] = (o[g][j][i] - co[g][i] + c) * f;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < gn * (kD / 8); i += blockDim.x) {
    const int hd = i / (kD / 8), ch = (i % (kD / 8)) * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, ls = 0.f;
    for (int w = 0; w < waves; ++w) {
      ls += s_l[w * 16 + hd];
      const float *src = s_o + (w * gn + hd) * kD + ch;
#pragma unroll
      for (int y = 0; y < 8; ++y) acc[y] += src[y];
    }
    if (a.splits > 1) {
      store8<kStateF32>(a.part_o, ((qh0 + hd) * a.splits + split) * kD + ch, acc);
    } else {
      const float inv = len == 0 ? 0.f : 1.f / ls;
#pragma unroll
      for (int y = 0; y < 8; ++y) acc[y] *= inv;
      store_out(type, a.out, (qh0 + hd) * kD + ch, acc);
    }
    if (a.part_ml && ch == 0) {
      float mm = -INFINITY;
      for (int w = 0; w < waves; ++w) mm = fmaxf(mm, s_m[w * 16 + hd]);
      a.part_ml[(qh0 + hd) * a.splits + split] = make_float2(mm, ls);
    }
  }
}

// The maximum and 1 / sum of a query head over its splits, on every lane of the wave.
__device__ __forceinline__ float2 join_ml(const AttendArgs &a, int64_t qh, int splits, bool empty) {
  const float2 *ml = a.part_ml + qh * a.splits;
  float m = -INFINITY, l = 0.f;
  const int lane = threadIdx.x & 63;
  if (splits == 1) {
    m = ml[0].x;
    l = ml[0].y;
  } else {
    for (int s = lane; s < splits; s += 64) m = fmaxf(m, ml[s].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float ms = m == -INFINITY ? 0.f : m;
    for (int s = lane; s < splits; s += 64) l += ml[s].y * __builtin_amdgcn_exp2f(ml[s].x - ms);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  }
  return make_float2(m == -INFINITY ? 0.f : m, empty ? 0.f : 1.f / l);
}

// Joins the splits of the rows' query heads and adds the weights; every wave works alone.  The
// first `outs` waves take a query head's output each (eight channels a lane, the lanes' groups
// taking every n-th split), the others 256 slots of a (row, head)'s weights.
constexpr int kSpan = 256;
template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_attend_finish(AttendArgs a, int64_t outs,
                                                            int spans, int64_t waves) {
  const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (id >= waves) return;
  const int lane = threadIdx.x & 63;
  if (id < outs) {
    const int64_t row = id / a.q_heads;
    const int64_t len = row_length(a, row, false);
    const int splits = (int)(len == 0 ? 1 : (len + a.chunk - 1) / a.chunk);  // that were written
    const float2 ml = join_ml(a, id, splits, len == 0);
    const int words = a.c.dim >> 3;
    int lpr = 1;
    while (lpr < words) lpr <<= 1;
    const int w = lane & (lpr - 1), part = lane / lpr, parts = 64 / lpr;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (w < words && len > 0)
      for (int s = part; s < splits; s += parts) {
        const float f = __builtin_amdgcn_exp2f(a.part_ml[id * a.splits + s].x - ml.x);
        float x[8];
        load8<kStateF32>(a.part_o, (id * a.splits + s) * a.c.dim + 8 * w, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(x[i], f, acc[i]);
      }
    for (int o = lpr; o < 64; o <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
    if (part == 0 && w < words) {
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= ml.y;
      store8<TYPE>(a.out, id * a.c.dim + 8 * w, acc);
    }
    return;
  }
  const int64_t pair = (id - outs) / spans;
  const int64_t row = pair / a.c.heads;
  const int64_t len = row_length(a, row, false);
  const int64_t j0 = (id - outs) % spans * kSpan;
  if (j0 >= len) return;
  const int splits = (int)((len + a.chunk - 1) / a.chunk);
  const int64_t q0 = pair * a.g;  // the head's first query head: row * q_heads + h * g
  float sum[kSpan / 64] = {0.f, 0.f, 0.f, 0.f};
  constexpr int kG = 4;
  for (int g0 = 0; g0 < a.g; g0 += kG) {
    float x[kG][kSpan / 64];
    float2 ml[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g)
#pragma unroll
      for (int i = 0; i < kSpan / 64; ++i) {
        const int64_t j = j0 + 64 * i + lane;
        x[g][i] = g0 + g < a.g && j < len ? a.logits[(q0 + g0 + g) * a.cap + j] : 0.f;
      }
#pragma unroll
    for (int g = 0; g < kG; ++g)
      ml[g] = g0 + g < a.g ? join_ml(a, q0 + g0 + g, splits, false) : make_float2(0.f, 0.f);
#pragma unroll
    for (int g = 0; g < kG; ++g)
#pragma unroll
      for (int i = 0; i < kSpan / 64; ++i)
        if (g0 + g < a.g) sum[i] += __builtin_amdgcn_exp2f(x[g][i] - ml[g].x) * ml[g].y;
  }
  float *wr = a.weights + pair * a.weights_cols;
#pragma unroll
  for (int i = 0; i < kSpan / 64; ++i) {
    const int64_t j = j0 + 64 * i + lane;
    if (j < len) wr[j] = a.decay != 0.f ? sum[i] + a.decay * wr[j] : sum[i];
  }
}

struct AttendPlan {
  bool matrix;
  int waves;  // of a workgroup of the matrix form
  int64_t chunk;
  int splits;
  int64_t cap;
  int64_t o_bytes, ml_bytes, logit_bytes;
};

int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

// Query heads of a work item of the vector form, and items a head needs.
int vec_gc(int g) { return g >= 4 ? 4 : (g >= 2 ? 2 : 1); }
int vec_gchunks(int g) { return (g + vec_gc(g) - 1) / vec_gc(g); }

AttendPlan plan_attend(const StateView &c, const AttendCall &a) {
  AttendPlan p{};
  p.cap = a.width << c.pshift;
  const int ng = c.dim / c.group, g = a.q_heads / c.heads;
  p.matrix = a.type != kStateF32 && (c.group == 32 || c.group == 64 || c.group == 128) &&
             (ng == 1 || ng == 2 || ng == 4) && p.cap > 16;
  int64_t chunk;
  if (p.matrix) {
    const int64_t work = a.rows * c.heads * ((g + 15) / 16);
    const int gn = g < 16 ? g : 16;
    // 8 waves where the rows alone cannot fill the card, as far as LDS holds their outputs
    p.waves = work * ceil_div(p.cap, 512) <= 256 ? 8 : 4;
    while (p.waves > 4 && p.waves * gn * c.dim * 4 > 96 * 1024) p.waves >>= 1;
    chunk = ceil_div(p.cap * work, 1024);
    const int64_t low = p.waves * 64 > 512 ? p.waves * 64 : 512;
    chunk = chunk < low ? low : (chunk + 127) & ~int64_t(127);
  } else {
    chunk = ceil_div(p.cap * a.rows * c.heads * vec_gchunks(g), 16384);
    chunk = chunk < 64 ? 64 : (chunk + 63) & ~int64_t(63);
  }
  p.splits = (int)(p.cap <= chunk ? 1 : ceil_div(p.cap, chunk));
  p.chunk = p.splits == 1 ? (p.cap > 0 ? p.cap : 1) : chunk;
  const int64_t qh = a.rows * a.q_heads;
  if (p.splits > 1) p.o_bytes = up256(qh * p.splits * c.dim * 4);
  // short rows of the vector form write their weights themselves
  const bool later = a.weights && !(!p.matrix && p.cap <= 16 && vec_gchunks(g) == 1);
  if (p.splits > 1 || later) p.ml_bytes = up256(qh * p.splits * 8);
  if (later) p.logit_bytes = up256(qh * p.cap * 4);
  return p;
}

int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p <<= 1;
  return p;
}

template <int LPR, int SL>
void launch_vec_g(const AttendArgs &a, int type, hipStream_t st) {
  const int gc = vec_gc(a.g), gchunks = vec_gchunks(a.g);
  const int64_t items = a.rows * a.c.heads * gchunks * a.splits;
  const int64_t blocks = ceil_div(items * LPR * SL, kThreads);
  DGS_CHECK(blocks < (int64_t(1) << 31) && items < (int64_t(1) << 31),
            "attend: too many rows in one call");
  if (gc == 4)
    k_attend_vec<LPR, SL, 4><<<(unsigned)blocks, kThreads, 0, st>>>(a, type, gchunks, items);
  else if (gc == 2)
    k_attend_vec<LPR, SL, 2><<<(unsigned)blocks, kThreads, 0, st>>>(a, type, gchunks, items);
  else
    k_attend_vec<LPR, SL, 1><<<(unsigned)blocks, kThreads, 0, st>>>(a, type, gchunks, items);
  DGS_LAUNCH_CHECK();
}
template <int LPR>
void launch_vec(const AttendArgs &a, int type, hipStream_t st) {
  if (a.cap <= 16)
    launch_vec_g<LPR, 1>(a, type, st);
  else
    launch_vec_g<LPR, 64 / LPR>(a, type, st);
}

template <int NG, int GROUP>
void launch_mfma(const AttendArgs &a, const AttendPlan &p, int type, hipStream_t st) {
  const int tiles = (a.g + 15) / 16, gn = a.g < 16 ? a.g : 16;
  const int64_t blocks = a.rows * a.c.heads * tiles * a.splits;
  DGS_CHECK(blocks < (int64_t(1) << 31), "attend: too many rows in one call");
  const int join = 32 + gn * NG * GROUP, corner = 8 * NG * GROUP + 64 * NG;  // words a wave needs of LDS
  const size_t lds = (size_t)p.waves * (join > corner ? join : corner) * 4;
  const unsigned grid = (unsigned)blocks, threads = p.waves * 64;
  if (type == kStateBF16)
    k_attend_mfma<NG, GROUP, 1><<<grid, threads, lds, st>>>(a, type, tiles);
  else
    k_attend_mfma<NG, GROUP, 2><<<grid, threads, lds, st>>>(a, type, tiles);
  DGS_LAUNCH_CHECK();
}
template <int GROUP>
void launch_mfma_g(const AttendArgs &a, const AttendPlan &p, int type, hipStream_t st) {
  switch (a.c.dim / GROUP) {
    case 1: launch_mfma<1, GROUP>(a, p, type, st); break;
    case 2: launch_mfma<2, GROUP>(a, p, type, st); break;
    case 4:
      if constexpr (GROUP < 128) launch_mfma<4, GROUP>(a, p, type, st);
  }
}

}  // namespace

int64_t state_attend_workspace(const StateView &c, const AttendCall &a) {
  const AttendPlan p = plan_attend(c, a);
  return p.o_bytes + p.ml_bytes + p.logit_bytes;
}

void state_attend(const StateView &c, const AttendCall &call, void *ws, int64_t ws_bytes,
                  hipStream_t st) {
  if (call.rows <= 0) return;
  const AttendPlan p = plan_attend(c, call);
  const int64_t need = p.o_bytes + p.ml_bytes + p.logit_bytes;
  DGS_CHECK(ws_bytes >= need && (need == 0 || ws), "attend: workspace too small");
  DGS_CHECK(p.cap < (int64_t(1) << 30) && c.pages < (int64_t(1) << 31),
            "attend: rows of 2^30 slots or caches of 2^31 pages");
  AttendArgs a{};
  a.c = c;
  a.q = call.q;
  a.q_row = call.q_row;
  a.q_head = call.q_head;
  a.rows = call.rows;
  a.q_heads = call.q_heads;
  a.g = call.q_heads / c.heads;
  a.table = call.table;
  a.lens = call.lens;
  a.width = call.width;
  a.scale2 = call.scale * kLog2e;
  a.chunk = p.chunk;
  a.splits = p.splits;
  char *w = static_cast<char *>(ws);
  if (p.o_bytes) a.part_o = (float *)w;
  if (p.ml_bytes) a.part_ml = (float2 *)(w + p.o_bytes);
  if (p.logit_bytes) a.logits = (float *)(w + p.o_bytes + p.ml_bytes);
  a.cap = p.cap;
  a.weights = call.weights;
  a.weights_cols = call.weights_cols;
  a.decay = call.decay;
  a.out = call.out;
  a.gd = state_guard(kAsyncErrSlot, c.pages);
  if (p.matrix) {
    if (c.group == 32)
      launch_mfma_g<32>(a, p, call.type, st);
    else if (c.group == 64)
      launch_mfma_g<64>(a, p, call.type, st);
    else
      launch_mfma_g<128>(a, p, call.type, st);
  } else switch (pow2_at_least(c.dim >> 3)) {
    case 1: launch_vec<1>(a, call.type, st); break;
    case 2: launch_vec<2>(a, call.type, st); break;
    case 4: launch_vec<4>(a, call.type, st); break;
    case 8: launch_vec<8>(a, call.type, st); break;
    case 16: launch_vec<16>(a, call.type, st); break;
    default: launch_vec<32>(a, call.type, st); break;
  }
  if (!a.part_ml) return;
  const int64_t outs = p.splits > 1 ? call.rows * call.q_heads : 0;
  const int spans = p.logit_bytes ? (int)ceil_div(p.cap, kSpan) : 0;
  const int64_t waves = outs + call.rows * c.heads * spans;
  const int64_t blocks = ceil_div(waves, kThreads / 64);
  if (blocks == 0) return;
  DGS_CHECK(blocks < (int64_t(1) << 31), "attend: too many rows in one call");
  const unsigned grid = (unsigned)blocks;
  if (call.type == kStateF32)
    k_attend_finish<kStateF32><<<grid, kThreads, 0, st>>>(a, outs, spans, waves);
  else if (call.type == kStateBF16)
    k_attend_finish<kStateBF16><<<grid, kThreads, 0, st>>>(a, outs, spans, waves);
  else
    k_attend_finish<kStateF16><<<grid, kThreads, 0, st>>>(a, outs, spans, waves);
  DGS_LAUNCH_CHECK();
}

}  // namespace dgs
