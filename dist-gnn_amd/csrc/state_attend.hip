// state_attend.hip -- attention of single query tokens over the 4-bit state cache.
//
// Row i has a query of q_heads heads and attends to the first len_i slots of its table row;
// query head a reads the K and V rows of head a / G, G = q_heads / heads:
//   x_j = scale * q . k_j,  p_j = exp(x_j - max x) / sum exp(x - max x),  out = sum_j p_j v_j.
// One pass over the slots with the running maximum m and sum l of the softmax, in 32 bits and
// base 2 (scale * log2 e follows q . k).  Long rows are split into chunks of slots whose (m, l,
// sum p v) go through the workspace; the finishing kernel joins them.  When the caller keeps
// attention weights, the logits of every slot go through the workspace too and the finishing
// kernel adds the G heads' probabilities in head order: no atomics, so results do not vary.
//
// A slot past the length, or on a page outside the cache (reported), has logit -inf, and its scale
// and base are replaced by zeros before use: what lies there (NaN, infinities) is never multiplied.
#include "dgs_attend.cuh"

namespace dgs {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// A word's codes as 16-bit floats: channel c is number c / 4 of pair c % 4.  A code in the low bits
// of such a float is code * 2^-24 below its normal range, four bits up it is code * 2^-20: no
// conversion, and exact.  The multiply-adds that take 16-bit factors widen them by themselves.
struct Codes {
  half2v p[4];
};
__device__ __forceinline__ Codes codes_of(uint32_t w) {
  const uint32_t y = w >> 8;
  return Codes{{__builtin_bit_cast(half2v, w & 0x000f000fu), __builtin_bit_cast(half2v, w & 0x00f000f0u),
                __builtin_bit_cast(half2v, y & 0x000f000fu), __builtin_bit_cast(half2v, y & 0x00f000f0u)}};
}
// Channel c's unit is 2^-24 on even channels, 2^-20 on odd ones; the caller's scales make it 2^-24 on
// all, in which values are summed (no scale leaves the range).
constexpr float kTiny = 0x1p-24f, kUnTiny = 0x1p24f;

template <int LPR>
__device__ __forceinline__ float sum_lanes(float x) {
  if constexpr (LPR >= 2) x += lane_xor32<1>(x);
  if constexpr (LPR >= 4) x += lane_xor32<2>(x);
  if constexpr (LPR >= 8) x += lane_xor32<4>(x);
  if constexpr (LPR >= 16) x += lane_xor32<8>(x);
  if constexpr (LPR >= 32) x += lane_xor32<16>(x);
  return x;
}

// x of the lane o (a power of two) away.
__device__ __forceinline__ float over(float x, int o) {
  switch (o) {
    case 1: return lane_xor32<1>(x);
    case 2: return lane_xor32<2>(x);
    case 4: return lane_xor32<4>(x);
    case 8: return lane_xor32<8>(x);
    case 16: return xor16(x);
    default: return xor32(x);
  }
}

// x of lane u of this lane's four.
__device__ __forceinline__ uint32_t of_quad(uint32_t x, int u) {
  switch (u) {
    case 0: return (uint32_t)dpp_keep<0x00>((int32_t)x, (int32_t)x);
    case 1: return (uint32_t)dpp_keep<0x55>((int32_t)x, (int32_t)x);
    case 2: return (uint32_t)dpp_keep<0xAA>((int32_t)x, (int32_t)x);
    default: return (uint32_t)dpp_keep<0xFF>((int32_t)x, (int32_t)x);
  }
}

// Vector form, for every type and size.  A work item is (row, head, GC query heads) and the slots it
// takes: a run of the stream form, or one of the equal chunks.  LPR lanes hold a row (W words of eight
// channels each); SL groups of them take four slots in a row at a time, with a softmax state of their own,
// joined at the end by exchanges between lanes.  Rows are loaded one step ahead of the arithmetic, ids
// another one.  What belongs to a slot and not to a channel - its page and address, and with QG (groups
// of a multiple of 32 channels) its scale and base - is fetched by one lane of every four and passed on
// by lane moves: 11 loads a step instead of 24.  K and V are taken as values (one multiply-add a code,
// then one a query head).  Summing V's codes with p * scale and the bases apart spares V's first one,
// but the two sums cancel: 32-bit outputs were 3 times as far off as the formula in 32 bits.  As in the
// matrix form, the running maximum is only followed when a logit passes it by 8.
// SL = 1 is for rows of at most 16 slots: no join, and with all query heads of a head in the item
// the probabilities stay in registers and the item writes its weights itself.
// Bound by the vector instructions (profiles/state_cache_counters.txt): 16 rows of 8 heads (128 channels,
// 32-bit, 1 to 8192 slots) 9.6 million of a wave, which keep the SIMDs busy for 15.6 of 23.6 us; the
// sampled neighbours' rows (40960 rows of 0 to 15 slots, 4 heads of 32 channels) 13.4 million, 21.7 of 32.4.
template <int LPR, int W, int SL, int GC, bool QG, bool STREAM>
__global__ __launch_bounds__(kThreads) void k_attend_vec(AttendArgs a, int type,
                                                         FastDivU32 splits, FastDivU32 gchunks,
                                                         FastDivU32 heads, uint32_t items) {
  constexpr int kItem = LPR * SL, kU = 4, kStep = SL * kU;
  constexpr int kKeep = SL > 1 ? 1 : (LPR >= 16 ? 1 : 16 / LPR);
  const int lane = threadIdx.x & (kItem - 1);
  const int sub = lane % LPR, sl = lane / LPR, mine = sub & 3;  // mine: the slot of four I look up
  uint32_t item = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) / kItem;
  if (kItem == 64) item = __builtin_amdgcn_readfirstlane(item);
  Run run;
  int64_t row;
  int h, gc, split = 0, len, first, last;
  if constexpr (STREAM) {
    if (!run.start(a, a.shift, a.cost, a.least, a.c.heads * (int)gchunks.d, (int)item, lane)) return;
    row = run.row;
    h = run.pair / (int)gchunks.d;
    gc = run.pair - h * (int)gchunks.d;
    len = run.len;
    first = run.tile << a.shift;
    last = run.last(a.shift, a.cost);
  } else {
    if (item >= items) return;  // whole items leave together: no exchange crosses an item
    const uint32_t is = splits.div(item), ig = gchunks.div(is);
    row = heads.div(ig);
    split = (int)(item - is * splits.d);
    gc = (int)(is - ig * gchunks.d);
    h = (int)(ig - (uint32_t)row * heads.d);
    len = (int)row_length(a, row, split == 0 && h == 0 && gc == 0 && lane == 0);
    first = split * (int)a.chunk;
    if (split > 0 && first >= len) return;
    last = a.splits == 1 ? len : (int)(first + a.chunk < len ? first + a.chunk : len);
  }
  const int words = a.c.dim >> 3;
  const int ng = a.c.dim / a.c.group;
  const float scale = a.scale2 * kUnTiny;  // of the sums, after them: only those can overflow
  bool live[W];
  int w[W], grp[W];  // my words of a row, and their groups
#pragma unroll
  for (int k = 0; k < W; ++k) {
    live[k] = sub + k * LPR < words;
    w[k] = live[k] ? sub + k * LPR : 0;
    grp[k] = 8 * w[k] / a.c.group;
  }
  int a0 = h * a.g + gc * GC, gn = a.g - gc * GC < GC ? a.g - gc * GC : GC;

  float q[GC][W][8], o[GC][W][8], m[GC], l[GC], xs[kKeep][GC];
  const int ps = a.c.pshift, mask = (1 << ps) - 1;
  const bool wide = a.table.bytes == 8;
  const char *tab;  // the row's
  const uint32_t pages = (uint32_t)a.c.pages, half = (uint32_t)a.c.dim >> 1;
  uint32_t id = 0, id_hi = 0;  // of my slot of the next step
  struct Rows {
    uint32_t kq[kU][W], vq[kU][W], km[QG ? 1 : kU][W], vm[QG ? 1 : kU][W];
    int n;         // slots of the step before the end
    uint32_t bad;  // bit u: slot u's page lies outside the cache
  };
  Rows t;
  auto slot_of = [&](int j0) {
    const int j = j0 + sl * kU + mine;
    return j < last ? j : last - 1;
  };
  auto load_ids = [&](int j0) {
    const char *at = tab + ((int64_t)(slot_of(j0) >> ps) << (wide ? 3 : 2));
    id = *(const uint32_t *)at;
    if (wide) id_hi = *(const uint32_t *)(at + 4);
  };
  // Loads a step's rows, and before them the next step's ids: memory returns in order, so whoever
  // waits for an id would wait for rows issued before it.
  auto load_rows = [&](int j0) {
    const bool out = id >= pages || id_hi != 0;
    t.n = last - j0 - sl * kU;
    t.bad = 0;
    if (__any(out)) {
      if (out && mine < t.n && sub < 4)
        report_bad_id(a.gd.err, kAsyncErrSlot,
                      wide ? (int64_t)((uint64_t)id_hi << 32 | id) : (int64_t)(int32_t)id, pages,
                      a.gd.tag);
#pragma unroll
      for (int u = 0; u < kU; ++u) t.bad |= of_quad(out ? 1u : 0u, u) << u;
    }
    const uint32_t page = out ? 0u : id;
    const int64_t r = (((int64_t)page * a.c.heads + h) << ps) + (slot_of(j0) & mask);
    const uint64_t at = (uint64_t)r * half;
    load_ids(j0 + kStep);
    if constexpr (QG) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        t.km[0][k] = a.c.ks[r * ng + grp[k]];
        t.vm[0][k] = a.c.vs[r * ng + grp[k]];
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint64_t to =
          (uint64_t)of_quad((uint32_t)(at >> 32), u) << 32 | of_quad((uint32_t)at, u);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        t.kq[u][k] = *(const uint32_t *)(a.c.kc + to + 4 * w[k]);
        t.vq[u][k] = *(const uint32_t *)(a.c.vc + to + 4 * w[k]);
      }
      if constexpr (!QG) {
        const uint64_t rw = ((uint64_t)of_quad((uint32_t)((uint64_t)r >> 32), u) << 32 |
                             of_quad((uint32_t)r, u)) * ng;
#pragma unroll
        for (int k = 0; k < W; ++k) {
          t.km[u][k] = a.c.ks[rw + grp[k]];
          t.vm[u][k] = a.c.vs[rw + grp[k]];
        }
      }
    }
  };
  auto compute = [&](const Rows &t, int j0, int keep) {
    float x[GC][kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool ok = u < t.n && !((t.bad >> u) & 1);
      float s[GC];
#pragma unroll
      for (int g = 0; g < GC; ++g) s[g] = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const uint32_t kw = QG ? of_quad(t.km[0][k], u) : t.km[QG ? 0 : u][k];
        const uint32_t km = live[k] ? kw : 0u;
        const float ks[2] = {scale_of(km), scale_of(km) * 0x1p-4f}, kb = base_of(km) * kTiny;
        const Codes kc = codes_of(t.kq[u][k]);
        float kv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) kv[i] = __builtin_fmaf((float)kc.p[i & 3][i >> 2], ks[i & 1], kb);
#pragma unroll
        for (int g = 0; g < GC; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) s[g] = __builtin_fmaf(q[g][k][i], kv[i], s[g]);
      }
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        const float x0 = sum_lanes<LPR>(s[g]) * scale;
        x[g][u] = ok ? x0 : -INFINITY;
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
        if (j0 + sl * kU + u < last)
#pragma unroll
          for (int g = 0; g < GC; ++g)
            if (g < gn) a.logits[((int64_t)row * a.q_heads + a0 + g) * a.cap + j0 + sl * kU + u] = x[g][u];
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      float top = fmaxf(fmaxf(x[g][0], x[g][1]), fmaxf(x[g][2], x[g][3]));
      if (top > m[g] + 8.f) {
        const float f = __builtin_amdgcn_exp2f(m[g] - top);
        m[g] = top;
        l[g] *= f;
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) o[g][k][i] *= f;
      }
      const float ms = m[g] == -INFINITY ? 0.f : m[g];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        x[g][u] = __builtin_amdgcn_exp2f(x[g][u] - ms);
        l[g] += x[g][u];
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const uint32_t vw = QG ? of_quad(t.vm[0][k], u) : t.vm[QG ? 0 : u][k];
        const uint32_t vm = live[k] && u < t.n && !((t.bad >> u) & 1) ? vw : 0u;
        const float vs[2] = {scale_of(vm), scale_of(vm) * 0x1p-4f}, vb = base_of(vm) * kTiny;
        const Codes vc = codes_of(t.vq[u][k]);
        float vv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) vv[i] = __builtin_fmaf((float)vc.p[i & 3][i >> 2], vs[i & 1], vb);
#pragma unroll
        for (int g = 0; g < GC; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) o[g][k][i] = __builtin_fmaf(x[g][u], vv[i], o[g][k][i]);
      }
  };
#pragma unroll 1
  while (true) {
    tab = (const char *)a.table.p + ((row * a.width) << (wide ? 3 : 2));
    if (first < last) {  // the rows are on their way while the query is read
      load_ids(first);
      load_rows(first);
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if (live[k] && g < gn) {
          load_q(type, a.q, row * a.q_row + (a0 + g) * a.q_head + 8 * w[k], q[g][k]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) q[g][k][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[g][k][i] = 0.f;
        }
      }
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int i = 0; i < kKeep; ++i) xs[i][g] = -INFINITY;
    }
    if (first < last) {
      if constexpr (SL == 1) {
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          if (4 * st >= last) break;
          const Rows now = t;
          if (4 * st + 4 < last) load_rows(4 * st + 4);
          compute(now, 4 * st, 4 * st);
        }
      } else {
#pragma unroll 1
        for (int j0 = first; j0 < last; j0 += kStep) {
          const Rows now = t;
          load_rows(j0 + kStep);
          compute(now, j0, 0);
        }
      }
    }
    // a pair that a wave of the stream form holds whole is finished here
    const bool whole = STREAM ? first == 0 && last == len : a.splits == 1;
    if (!STREAM || first < last) {
      bool zero = false;  // a query head's sum is 0
#pragma unroll
      for (int g = 0; g < GC; ++g)
        if (g < gn) zero |= SL == 1 ? l[g] == 0.f : __all(l[g] == 0.f);
      if (zero) zero = some_left<SL == 1 ? 1 : 64>(a, row, first, last);
#pragma unroll
      for (int g = 0; g < GC; ++g) {
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            o[g][k][i] *= kUnTiny;
#pragma unroll
        for (int s = LPR; s < kItem; s <<= 1) {
          const float mo = __shfl_xor(m[g], s, 64);
          const float mn = fmaxf(m[g], mo), ms = mn == -INFINITY ? 0.f : mn;
          const float f = __builtin_amdgcn_exp2f(m[g] - ms), fo = __builtin_amdgcn_exp2f(mo - ms);
          m[g] = mn;
          l[g] = l[g] * f + __shfl_xor(l[g], s, 64) * fo;
#pragma unroll
          for (int k = 0; k < W; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              o[g][k][i] = o[g][k][i] * f + __shfl_xor(o[g][k][i], s, 64) * fo;
        }
        if (zero && l[g] == 0.f) m[g] = kNoSoftmax;
        if (g >= gn || sl != 0) continue;
        const int64_t qh = row * a.q_heads + a0 + g;
        const int64_t part = STREAM ? (row * run.pairs + run.pair + item) * (a.g < GC ? a.g : GC) + g
                                    : qh * a.splits + split;
        const float inv = inverse_sum(m[g], l[g]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
          if (!live[k]) continue;
          if (!whole) {
            store8<kStateF32>(a.part_o, part * a.c.dim + 8 * w[k], o[g][k]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[g][k][i] *= inv;
            store_out(type, a.out, qh * a.c.dim + 8 * w[k], o[g][k]);
          }
        }
        if (a.part_ml && sub == 0) a.part_ml[part] = make_float2(m[g], l[g]);
        if (SL == 1) l[g] = inv;  // of the weights below
      }
    }
    if constexpr (!STREAM) {
      break;
    } else {
      if (!run.next(a, a.shift, a.cost)) return;
      row = run.row;
      h = run.pair / (int)gchunks.d;
      gc = run.pair - h * (int)gchunks.d;
      a0 = h * a.g + gc * GC;
      gn = a.g - gc * GC < GC ? a.g - gc * GC : GC;
      len = run.len;
      first = 0;
      last = run.last(a.shift, a.cost);
    }
  }
  if constexpr (SL == 1) {
    if (a.weights && !a.logits) {  // every query head of this head is here
      float *wr = a.weights + ((int64_t)row * a.c.heads + h) * a.weights_cols;
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        const int j = i * LPR + sub;
        if (j >= len) continue;
        float sum = 0.f;
#pragma unroll
        for (int g = 0; g < GC; ++g)
          if (g < gn) {
            const float ms = m[g] == -INFINITY ? 0.f : m[g];
            sum += __builtin_amdgcn_exp2f(xs[i][g] - ms) * l[g];
          }
        wr[j] = a.decay != 0.f ? sum + a.decay * wr[j] : sum;
      }
    }
  }
}

// The parts of a query head: n of them, the first at `part`, `stride` apart.
struct Parts {
  int64_t part;
  int stride, n;
};
__device__ __forceinline__ Parts parts_of(const AttendArgs &a, int64_t row, int head, int64_t len) {
  if (a.splits)
    return Parts{(row * a.q_heads + head) * a.splits, 1,
                 len == 0 ? 1 : (int)((len + a.chunk - 1) / a.chunk)};
  const int t = a.together, tiles = (a.g + t - 1) / t, pairs = a.c.heads * tiles;
  const int gs = a.g < t ? a.g : t, h = head / a.g, n = head - h * a.g, pair = h * tiles + n / t;
  int64_t part = row * pairs + pair;
  int parts = 1;
  if (a.stream) {
    const int lane = threadIdx.x & 63, per = (int)((a.rows + 63) >> 6);
    int before, own, total, len_of_last;
    stream_sums(a, a.shift, a.cost, lane, per, before, own, total, len_of_last);
    const int who = (int)(row / per);
    int64_t front = __shfl(before, who, 64);
    for (int64_t r = (int64_t)who * per; r < row; ++r) front += row_units(a, r, a.shift, a.cost);
    const int q = stream_share(a, a.cost, a.least, (int64_t)total * pairs);
    const int u = row_units(a, row, a.shift, a.cost);
    const int64_t start = front * pairs + (int64_t)pair * u;
    const int64_t w0 = (start + a.cost) / q;  // the wave of its first tile
    parts = u == 0 ? 1 : (int)((start + u - 1) / q - w0) + 1;
    part += w0;
  }
  return Parts{part * gs + n % t, gs, parts};
}
// The maximum and 1 / sum of kG query heads over their parts (head g's `step` g behind), on every
// lane of the wave; heads at or past g_end repeat the first.  64 / kG lanes take a head's parts.
template <int kG>
__device__ __forceinline__ void join_ml(const AttendArgs &a, const Parts &p, int64_t step,
                                        int g_end, float2 (&out)[kG]) {
  constexpr int kL = 64 / kG;
  const int lane = threadIdx.x & 63, g = lane / kL, s0 = lane % kL;
  const float2 *ml = a.part_ml + p.part + (g < g_end ? g * step : 0);
  const float2 own = s0 < p.n ? ml[(int64_t)s0 * p.stride] : make_float2(-INFINITY, 0.f);
  float m = own.x;
  for (int s = s0 + kL; s < p.n; s += kL) m = fmaxf(m, ml[(int64_t)s * p.stride].x);
#pragma unroll
  for (int o = 1; o < kL; o <<= 1) m = fmaxf(m, over(m, o));
  const bool none = m == -INFINITY;
  m = none ? 0.f : m;
  float l = own.y * __builtin_amdgcn_exp2f(own.x - m);
  for (int s = s0 + kL; s < p.n; s += kL) {
    const float2 x = ml[(int64_t)s * p.stride];
    l += x.y * __builtin_amdgcn_exp2f(x.x - m);
  }
#pragma unroll
  for (int o = 1; o < kL; o <<= 1) l += over(l, o);
  l = none ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < kG; ++k)
    out[k] = make_float2(
        __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), k * kL)),
        __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l), k * kL)));
}

// Joins the parts of the rows' query heads and adds the weights; every wave works alone.  The
// first `outs` waves take 8 `lpr` channels of a query head's output each (eight channels a lane, the
// lanes' groups taking every n-th part), the others 1024 slots of a (row, head)'s weights.  64 rows of
// 8 heads, 32 query heads, 1 to 8192 slots (50 MB of logits and weights): 15.6 us, before whose rows come
// the lengths, parts and maxima, loads that wait for each other; 8 rows without weights 6 us.
constexpr int kSpan = 1024;
template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_attend_finish(AttendArgs a, int64_t outs, int lpr,
                                                            int spans, int64_t waves) {
  const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (id >= waves) return;
  const int lane = threadIdx.x & 63;
  if (id < outs) {
    const int words = a.c.dim >> 3, slices = (words + lpr - 1) / lpr;
    const int64_t qh = id / slices, row = qh / a.q_heads;
    const int64_t len = row_length(a, row, a.stream && id % (a.q_heads * slices) == 0 && lane == 0);
    const Parts p = parts_of(a, row, (int)(qh % a.q_heads), len);
    if (a.stream && p.n == 1 && len > 0) return;  // written by the wave that had it whole
    const int w = (int)(id % slices) * lpr + (lane & (lpr - 1));
    const int part = lane / lpr, parts = 64 / lpr;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (len > 0) {
      float2 joined[1];
      join_ml<1>(a, p, 0, 1, joined);
      const float2 ml = joined[0];
      if (w < words)
        for (int s0 = part; s0 < p.n; s0 += 4 * parts) {  // four parts in flight
          float x[4][8], f[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int s = s0 + u * parts < p.n ? s0 + u * parts : s0;
            const int64_t at = p.part + (int64_t)s * p.stride;
            f[u] = __builtin_amdgcn_exp2f(a.part_ml[at].x - ml.x);
            load8<kStateF32>(a.part_o, at * a.c.dim + 8 * w, x[u]);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (s0 + u * parts < p.n)
#pragma unroll
              for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(x[u][i], f[u], acc[i]);
        }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1)
        if (o >= lpr)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += over(acc[i], o);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= ml.y;
    }
    if (part == 0 && w < words) store8<TYPE>(a.out, qh * a.c.dim + 8 * w, acc);
    return;
  }
  const int64_t pair = (id - outs) / spans;
  const int64_t row = pair / a.c.heads;
  const int64_t len = row_length(a, row, false);
  const int64_t j0 = (id - outs) % spans * kSpan;
  if (j0 >= len) return;
  const int head0 = (int)(pair % a.c.heads) * a.g;  // the head's first query head
  const int64_t q0 = row * a.q_heads + head0;
  constexpr int kG = 4, kI = 4, kRuns = kSpan / (64 * kI);  // heads and slots in flight together
  // lane t takes slots j0 + t, + 64, ...; a slot past the end reads the last one
  float sum[kRuns][kI];
#pragma unroll
  for (int r = 0; r < kRuns; ++r)
#pragma unroll
    for (int i = 0; i < kI; ++i) sum[r][i] = 0.f;
  Parts p = parts_of(a, row, head0, len);
  for (int g0 = 0; g0 < a.g; g0 += kG) {
    // the query heads of a pair share their parts' places (kG divides 16 and 4)
    if (a.splits || (g0 > 0 && g0 % a.together == 0)) p = parts_of(a, row, head0 + g0, len);
    const Parts pg{p.part + (a.splits ? 0 : g0 % a.together), p.stride, p.n};
    float2 ml[kG];
    join_ml<kG>(a, pg, a.splits ? a.splits : 1, a.g - g0, ml);
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      if (j0 + r * kI * 64 >= len) break;
      float x[kG][kI];
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const float *lg = a.logits + (q0 + (g0 + g < a.g ? g0 + g : g0)) * a.cap;
#pragma unroll
        for (int i = 0; i < kI; ++i) {
          const int64_t j = j0 + (r * kI + i) * 64 + lane;
          x[g][i] = lg[j < len ? j : len - 1];
        }
      }
#pragma unroll
      for (int g = 0; g < kG; ++g)
        if (g0 + g < a.g)
#pragma unroll
          for (int i = 0; i < kI; ++i)
            sum[r][i] += __builtin_amdgcn_exp2f(x[g][i] - ml[g].x) * ml[g].y;
    }
  }
  float *wr = a.weights + pair * a.weights_cols;
#pragma unroll
  for (int r = 0; r < kRuns; ++r)
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      const int64_t j = j0 + (r * kI + i) * 64 + lane;
      if (j < len) wr[j] = a.decay != 0.f ? sum[r][i] + a.decay * wr[j] : sum[r][i];
    }
}

// The vector form's line: tiles are its steps, and a pair costs two of them (16 rows of 8 heads of 128
// channels, 1 to 8192 slots, 32-bit: 30 us, 32 at 4 and 30 at 6; 64 rows of 1 to 700: 30, 30, 35; 700 rows of
// 1 to 1000: 100, 108, 114).  4096 waves are the four a SIMD that the registers of two query heads leave;
// 8192 are no faster (30, 30 and 102).
constexpr int kVecWaves = 4096, kVecCost = 2, kVecLeast = 1;
// Waves below which the joining takes narrower slices of channels.
constexpr int kJoinWaves = 1024;

struct AttendPlan {
  bool matrix;
  int waves;   // of a workgroup of the matrix form
  int stream;  // waves of the stream form, or 0
  int64_t chunk;
  int splits;  // vector form without
  int64_t cap;
  bool finish;  // the finishing kernel runs
  int64_t o_bytes, ml_bytes, logit_bytes;
};

int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

// Query heads of a work item of the vector form, and items a head needs.
int vec_gc(int g) { return g < 4 ? g : 4; }
int vec_gchunks(int g) { return (g + vec_gc(g) - 1) / vec_gc(g); }

AttendPlan plan_attend(const StateView &c, const AttendCall &a) {
  AttendPlan p{};
  p.cap = a.width << c.pshift;
  const int ng = c.dim / c.group, g = a.q_heads / c.heads;
  p.matrix = a.type != kStateF32 && (c.group == 32 || c.group == 64 || c.group == 128) &&
             (ng == 1 || ng == 2 || ng == 4) && p.cap > 16;
  const int64_t qh = a.rows * a.q_heads;
  if (p.matrix) {
    const int64_t pairs = a.rows * c.heads * ((g + 15) / 16);
    // Rows that can be longer than 1024 slots, and few enough to add up, are cut evenly over the
    // waves that fit the card at once (256 CUs x 4 SIMDs x 2).
    p.stream = p.cap > 1024 && a.rows <= kStreamRows &&
                       a.rows * ceil_div(p.cap, 32) < (int64_t(1) << 30)
                   ? 2048
                   : 0;
    // Else the waves of a pair: one where the pairs fill the card (it holds 2048 waves), up to 8 where
    // they cannot, as far as 64 KB of LDS go (256 channels take the registers of two waves).  3713
    // rows of 8 heads, 9 to 13 slots in pages of 128: 485 us with 4 waves, 234 with 2, 128 with one;
    // 1500 rows of 100 to 1000 slots: 286, 214, 187 us.
    p.waves = p.stream || (pairs > 256 && pairs <= 512) ? 4
              : pairs > 1024                            ? 1
              : pairs > 512                             ? 2
              : pairs * ceil_div(p.cap, 512) <= 256 && c.dim < 256 ? 8
                                                                   : 4;
    while (p.waves > 1 &&
           p.waves * attend_matrix_lds(c.dim, c.group, g, p.stream != 0) * 4 > 64 * 1024)
      p.waves >>= 1;
    const int64_t parts = (pairs + p.stream) * (g < 16 ? g : 16);
    // a workgroup that has a row and all its query heads adds its weights itself, from the logits
    // that it wrote (a long row would be a tail: 8192 slots 38 us, the finishing kernel 17)
    p.finish = p.stream || (a.weights && (g > 16 || p.cap > 1024));
    if (p.stream) p.o_bytes = up256(parts * c.dim * 4);
    if (p.finish) p.ml_bytes = up256(parts * 8);
    if (a.weights) p.logit_bytes = up256(qh * p.cap * 4);
    return p;
  }
  // Rows that can be longer than 512 slots are cut evenly, as in the matrix form: 16 rows of 8 heads,
  // 1 to 8192 slots, 32-bit: 30 us against 48 in equal chunks; 300 rows of 1 to 2000, two query heads a head:
  // 100, 130; 4 rows of 500 to 700: 19, 19; 700 rows of 5 to 300, 4 heads of 64: 41, 30.
  p.stream = p.cap > 512 && a.rows <= kStreamRows &&
                     a.rows * ceil_div(p.cap, 8) < (int64_t(1) << 30)
                 ? kVecWaves
                 : 0;
  if (p.stream) {
    const int64_t parts =
        (a.rows * c.heads * vec_gchunks(g) + p.stream) * (int64_t)vec_gc(g);
    p.finish = true;
    p.o_bytes = up256(parts * c.dim * 4);
    p.ml_bytes = up256(parts * 8);
    if (a.weights) p.logit_bytes = up256(qh * p.cap * 4);
    return p;
  }
  int64_t chunk = ceil_div(p.cap * a.rows * c.heads * vec_gchunks(g), 16384);
  chunk = chunk < 64 ? 64 : (chunk + 63) & ~int64_t(63);
  p.splits = (int)(p.cap <= chunk ? 1 : ceil_div(p.cap, chunk));
  p.chunk = p.splits == 1 ? (p.cap > 0 ? p.cap : 1) : chunk;
  // items of short rows with all query heads of a head add their weights from registers
  const bool own = p.cap <= 16 && vec_gchunks(g) == 1;
  p.finish = p.splits > 1 || (a.weights && !own);
  if (p.splits > 1) p.o_bytes = up256(qh * p.splits * c.dim * 4);
  if (p.finish) p.ml_bytes = up256(qh * p.splits * 8);
  if (a.weights && !own) p.logit_bytes = up256(qh * p.cap * 4);
  return p;
}

int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p <<= 1;
  return p;
}

// How a row's words lie in lanes.  Two or three words a lane make less work of a slot (its softmax and
// addresses are shared by more channels, and 10 or 12 words fill their lanes), but steps of more slots,
// so not where slots are few or rows short, and not with the registers of three query heads: 16 rows
// of 8 heads, 1 to 8192 slots, of 256 channels 48 to 42 us, of 96 with two query heads a head 37 to 32;
// 700 rows of 1 to 1000 slots, 128 channels, 109 to 100; but 37 rows of 12 heads of 80 channels, 0 to
// 1531 slots, 29 to 31, and 5000 rows of 20 to 40 slots, 96 channels, 96 to 200.
struct VecShape {
  int lanes, words;
};
VecShape vec_shape(const StateView &c, int g, int64_t rows, int64_t cap) {
  const int n = c.dim >> 3;
  if (vec_gc(g) <= 2 && cap > 256 && rows * c.heads * cap >= 1 << 20) {
    const int lanes = n <= 12 ? 4 : (n <= 24 ? 8 : 16);
    return VecShape{lanes, (n + lanes - 1) / lanes};
  }
  return VecShape{n <= 4 ? 4 : (n <= 8 ? 8 : (n <= 16 ? 16 : 32)), 1};
}

template <int LPR, int W, int SL, int GC, bool QG, bool STREAM>
void launch_vec_k(const AttendArgs &a, int type, hipStream_t st) {
  const int gchunks = vec_gchunks(a.g);
  const int64_t items = STREAM ? a.stream : a.rows * a.c.heads * gchunks * a.splits;
  const int64_t blocks = ceil_div(items * LPR * SL, kThreads);
  DGS_CHECK(items * LPR * SL < (int64_t(1) << 32) - kThreads,
            "attend: too many rows in one call");
  k_attend_vec<LPR, W, SL, GC, QG, STREAM><<<(unsigned)blocks, kThreads, 0, st>>>(
      a, type, FastDivU32::make(STREAM ? 1 : a.splits), FastDivU32::make(gchunks),
      FastDivU32::make(a.c.heads), (uint32_t)items);
  DGS_LAUNCH_CHECK();
}
template <int LPR, int W, int SL, int GC, bool STREAM>
void launch_vec_q(const AttendArgs &a, int type, hipStream_t st) {
  if (a.c.group % 32 == 0)
    launch_vec_k<LPR, W, SL, GC, true, STREAM>(a, type, st);
  else
    launch_vec_k<LPR, W, SL, GC, false, STREAM>(a, type, st);
}
template <int LPR, int W, int GC>
void launch_vec(const AttendArgs &a, int type, hipStream_t st) {
  if (a.stream)
    launch_vec_q<LPR, W, 64 / LPR, GC, true>(a, type, st);
  else
    launch_vec_q<LPR, W, 64 / LPR, GC, false>(a, type, st);
}
template <int LPR, int GC>
void launch_vec_one(const AttendArgs &a, int type, hipStream_t st) {
  if (a.cap <= 16)
    launch_vec_q<LPR, 1, 1, GC, false>(a, type, st);
  else
    launch_vec<LPR, 1, GC>(a, type, st);
}
template <int GC>
void launch_vec_gc(const AttendArgs &a, VecShape s, int type, hipStream_t st) {
  if constexpr (GC <= 2) {
    if (s.words == 2 && s.lanes == 4) return launch_vec<4, 2, GC>(a, type, st);
    if (s.words == 2 && s.lanes == 8) return launch_vec<8, 2, GC>(a, type, st);
    if (s.words == 2) return launch_vec<16, 2, GC>(a, type, st);
    if (s.words == 3 && s.lanes == 4) return launch_vec<4, 3, GC>(a, type, st);
    if (s.words == 3) return launch_vec<8, 3, GC>(a, type, st);
  }
  switch (s.lanes) {
    case 4: return launch_vec_one<4, GC>(a, type, st);
    case 8: return launch_vec_one<8, GC>(a, type, st);
    case 16: return launch_vec_one<16, GC>(a, type, st);
    default: return launch_vec_one<32, GC>(a, type, st);
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
  a.stream = p.stream;
  a.together = p.matrix ? 16 : 4;
  const VecShape shape = vec_shape(c, a.g, call.rows, p.cap);
  a.shift = p.matrix ? kMatrixShift : shape.lanes == 4 ? 6 : shape.lanes == 8 ? 5 : shape.lanes == 16 ? 4 : 3;
  a.cost = p.matrix ? kMatrixCost : kVecCost;
  a.least = p.matrix ? kMatrixLeast : kVecLeast;
  char *w = static_cast<char *>(ws);
  if (p.o_bytes) a.part_o = (float *)w;
  if (p.ml_bytes) a.part_ml = (float2 *)(w + p.o_bytes);
  if (p.logit_bytes) a.logits = (float *)(w + p.o_bytes + p.ml_bytes);
  a.cap = p.cap;
  a.weights = call.weights;
  a.weights_cols = call.weights_cols;
  a.decay = call.decay;
  a.out = call.out;
  a.gd = state_guard();
  if (p.matrix) {
    (c.group == 32 ? attend_matrix_32 : c.group == 64 ? attend_matrix_64 : attend_matrix_128)(
        a, p.waves, call.type, st);
  } else {
    switch (vec_gc(a.g)) {
      case 1: launch_vec_gc<1>(a, shape, call.type, st); break;
      case 2: launch_vec_gc<2>(a, shape, call.type, st); break;
      case 3: launch_vec_gc<3>(a, shape, call.type, st); break;
      default: launch_vec_gc<4>(a, shape, call.type, st); break;
    }
  }
  if (!p.finish) return;
  const int64_t qh = call.rows * call.q_heads;
  // lanes of a part in the joining: few query heads have many parts each, which narrow slices take
  // more at a time: 32 query heads of 256 parts 11 us, 20 with 128 channels a wave; where there are
  // many heads it only makes waves (64 rows of 32: 64 us in all, 70 at 16384)
  int lpr = pow2_at_least(c.dim >> 3);
  while (lpr > 4 && qh * ceil_div(c.dim >> 3, lpr) < kJoinWaves) lpr >>= 1;
  const int64_t outs = p.splits > 1 || p.stream ? qh * ceil_div(c.dim >> 3, lpr) : 0;
  const int spans = p.logit_bytes ? (int)ceil_div(p.cap, kSpan) : 0;
  const int64_t waves = outs + call.rows * c.heads * spans;
  const int64_t blocks = ceil_div(waves, kThreads / 64);
  if (blocks == 0) return;
  DGS_CHECK(blocks < (int64_t(1) << 31), "attend: too many rows in one call");
  const unsigned grid = (unsigned)blocks;
  if (call.type == kStateF32)
    k_attend_finish<kStateF32><<<grid, kThreads, 0, st>>>(a, outs, lpr, spans, waves);
  else if (call.type == kStateBF16)
    k_attend_finish<kStateBF16><<<grid, kThreads, 0, st>>>(a, outs, lpr, spans, waves);
  else
    k_attend_finish<kStateF16><<<grid, kThreads, 0, st>>>(a, outs, lpr, spans, waves);
  DGS_LAUNCH_CHECK();
}

}  // namespace dgs
