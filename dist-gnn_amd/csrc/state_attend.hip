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

template <int TYPE>
__device__ __forceinline__ void store_row(void *out, int64_t elem, const float (&x)[8]) {
  store8<TYPE>(out, elem, x);
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

// Vector form, for every type and size.  A work item is (row, head, GC query heads, split).  LPR
// lanes hold a row (eight channels each), SL groups of them take every SL-th slot with a softmax
// state of their own, joined at the end by exchanges between lanes.
template <int LPR, int SL, int GC>
__global__ __launch_bounds__(kThreads) void k_attend_vec(AttendArgs a, int type, int gchunks,
                                                         int64_t items) {
  constexpr int kItem = LPR * SL, kU = SL == 1 ? 4 : 2;
  const int lane = threadIdx.x & (kItem - 1);
  int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / kItem;
  const bool here = item < items;
  if (!here) return;  // whole items leave together: no exchange crosses an item
  const int sub = lane % LPR, sl = lane / LPR;
  const int split = (int)(item % a.splits);
  item /= a.splits;
  const int gc = (int)(item % gchunks);
  item /= gchunks;
  const int h = (int)(item % a.c.heads);
  const int64_t row = item / a.c.heads;
  const int words = a.c.dim >> 3;
  const bool live = sub < words;
  const int w = live ? sub : 0, ng = a.c.dim / a.c.group, grp = 8 * w / a.c.group;
  const int64_t len = row_length(a, row, split == 0 && h == 0 && gc == 0 && lane == 0);
  const int64_t first = (int64_t)split * a.chunk;
  if (split > 0 && first >= len) return;
  const int64_t last = a.splits == 1 ? len : (first + a.chunk < len ? first + a.chunk : len);
  const int a0 = h * a.g + gc * GC, gn = a.g - gc * GC < GC ? a.g - gc * GC : GC;

  float q[GC][8], o[GC][8], m[GC], l[GC];
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
  }
  const int64_t mask = (int64_t(1) << a.c.pshift) - 1;
  for (int64_t j0 = first; j0 < last; j0 += SL * kU) {
    uint32_t kq[kU], vq[kU], km[kU], vm[kU];
    bool ok[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t j = j0 + u * SL + sl;
      ok[u] = j < last;
      const int64_t jj = ok[u] ? j : last - 1;
      int64_t page = a.table[row * a.width + (jj >> a.c.pshift)];
      if ((uint64_t)page >= (uint64_t)a.c.pages) {
        if (ok[u] && sub == 0) report_bad_id(a.gd.err, kAsyncErrSlot, page, a.c.pages, a.gd.tag);
        ok[u] = false;
        page = 0;
      }
      const int64_t r = ((page * a.c.heads + h) << a.c.pshift) + (jj & mask);
      kq[u] = *(const uint32_t *)(a.c.kc + r * (a.c.dim >> 1) + 4 * w);
      vq[u] = *(const uint32_t *)(a.c.vc + r * (a.c.dim >> 1) + 4 * w);
      km[u] = a.c.ks[r * ng + grp];
      vm[u] = a.c.vs[r * ng + grp];
      if (!ok[u] || !live) km[u] = vm[u] = 0;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float kv[8], vv[8];
      codes8(kq[u], kv);
      codes8(vq[u], vv);
      const float ks = scale_of(km[u]), kb = base_of(km[u]);
      const float vs = scale_of(vm[u]), vb = base_of(vm[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        kv[i] = __builtin_fmaf(kv[i], ks, kb);
        vv[i] = __builtin_fmaf(vv[i], vs, vb);
      }
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x = __builtin_fmaf(q[g][i], kv[i], x);
#pragma unroll
        for (int s = LPR >> 1; s > 0; s >>= 1) x += __shfl_xor(x, s, 64);
        if (!ok[u]) x = -INFINITY;
        if (a.logits && sub == 0 && g < gn && j0 + u * SL + sl < last)
          a.logits[(row * a.q_heads + a0 + g) * a.cap + j0 + u * SL + sl] = x;
        const float mn = fmaxf(m[g], x);
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m[g] - ms);
        const float p = __builtin_amdgcn_exp2f(x - ms);
        m[g] = mn;
        l[g] = __builtin_fmaf(l[g], f, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[g][i] = __builtin_fmaf(p, vv[i], o[g][i] * f);
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
}

// Joins the splits of a row's head into the output and adds the weights.  Block (x, y): x =
// (row, head), y = a range of slots of the weights; y = 0 also writes the output.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_attend_finish(AttendArgs a, int64_t span) {
  __shared__ float2 s_ml[64];
  const int64_t row = blockIdx.x / a.c.heads;
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t len = row_length(a, row, false);
  const int64_t j0 = (int64_t)blockIdx.y * span;
  if (blockIdx.y > 0 && j0 >= len) return;
  const int splits = (int)(len == 0 ? 1 : (len + a.chunk - 1) / a.chunk);  // that were written
  const int tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  for (int gb = 0; gb < a.g; gb += 64) {
    const int gn = a.g - gb < 64 ? a.g - gb : 64;
    const int64_t q0 = row * a.q_heads + h * a.g + gb;
    for (int g = wave; g < gn; g += kThreads / 64) {
      const float2 *ml = a.part_ml + (q0 + g) * a.splits;
      float m = -INFINITY;
      bool nan = false;
      for (int s = lane; s < splits; s += 64) m = fmaxf(m, ml[s].x);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
      const float ms = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      for (int s = lane; s < splits; s += 64)
        l += ml[s].y * __builtin_amdgcn_exp2f(ml[s].x - ms);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
      (void)nan;
      const float inv = len == 0 ? 0.f : 1.f / l;
      if (lane == 0) s_ml[g] = make_float2(ms, inv);
      if (a.splits > 1 && blockIdx.y == 0) {
        for (int w = lane; w < (a.c.dim >> 3); w += 64) {
          float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, x[8];
          for (int s = 0; s < splits && len > 0; ++s) {
            const float f = __builtin_amdgcn_exp2f(ml[s].x - ms);
            load8<kStateF32>(a.part_o, ((q0 + g) * a.splits + s) * a.c.dim + 8 * w, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(x[i], f, acc[i]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] *= inv;
          store8<TYPE>(a.out, (q0 + g) * a.c.dim + 8 * w, acc);
        }
      }
    }
    __syncthreads();
    if (a.weights) {
      float *wr = a.weights + (row * a.c.heads + h) * a.weights_cols;
      const int64_t jn = j0 + span < len ? j0 + span : len;
      for (int64_t j = j0 + tid; j < jn; j += kThreads) {
        float sum = 0.f;
        for (int g = 0; g < gn; ++g)
          sum += __builtin_amdgcn_exp2f(a.logits[(q0 + g) * a.cap + j] - s_ml[g].x) * s_ml[g].y;
        if (gb > 0)
          sum += wr[j];
        else if (a.decay != 0.f)
          sum += a.decay * wr[j];
        wr[j] = sum;
      }
    }
    __syncthreads();
  }
}

struct AttendPlan {
  int64_t chunk;
  int splits;
  int64_t cap;
  int64_t o_bytes, ml_bytes, logit_bytes;
};

int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

AttendPlan plan_attend(const StateView &c, const AttendCall &a) {
  AttendPlan p{};
  p.cap = a.width << c.pshift;
  const int64_t work = a.rows * c.heads;  // (row, head) pairs
  // Splits: enough waves to fill the card (256 CUs x 16), of at least 64 slots each.
  int64_t chunk = ceil_div(p.cap * work, 4096);
  chunk = chunk < 64 ? 64 : (chunk + 63) & ~int64_t(63);
  p.splits = (int)(p.cap <= chunk ? 1 : ceil_div(p.cap, chunk));
  p.chunk = p.splits == 1 ? (p.cap > 0 ? p.cap : 1) : chunk;
  const int64_t qh = a.rows * a.q_heads;
  if (p.splits > 1) p.o_bytes = up256(qh * p.splits * c.dim * 4);
  if (p.splits > 1 || a.weights) p.ml_bytes = up256(qh * p.splits * 8);
  if (a.weights) p.logit_bytes = up256(qh * p.cap * 4);
  return p;
}

int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p <<= 1;
  return p;
}

template <int LPR, int SL>
void launch_vec_g(const AttendArgs &a, int type, hipStream_t st) {
  const int gc = a.g >= 4 ? 4 : (a.g >= 2 ? 2 : 1);
  const int gchunks = (a.g + gc - 1) / gc;
  const int64_t items = a.rows * a.c.heads * gchunks * a.splits;
  const int64_t blocks = ceil_div(items * LPR * SL, kThreads);
  DGS_CHECK(blocks < (int64_t(1) << 31), "attend: too many rows in one call");
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
  switch (pow2_at_least(c.dim >> 3)) {
    case 1: launch_vec<1>(a, call.type, st); break;
    case 2: launch_vec<2>(a, call.type, st); break;
    case 4: launch_vec<4>(a, call.type, st); break;
    case 8: launch_vec<8>(a, call.type, st); break;
    case 16: launch_vec<16>(a, call.type, st); break;
    default: launch_vec<32>(a, call.type, st); break;
  }
  if (!a.part_ml) return;
  const int64_t pairs = call.rows * c.heads;
  DGS_CHECK(pairs < (int64_t(1) << 31), "attend: too many rows in one call");
  // slots of one finishing block: all of a short row, else 1024
  const int64_t span = 1024;
  int64_t ny = call.weights ? ceil_div(p.cap, span) : 1;
  if (ny < 1) ny = 1;
  DGS_CHECK(ny < 65536, "attend: rows longer than 67 million slots");
  const dim3 grid((unsigned)pairs, (unsigned)ny);
  if (call.type == kStateF32)
    k_attend_finish<kStateF32><<<grid, kThreads, 0, st>>>(a, span);
  else if (call.type == kStateBF16)
    k_attend_finish<kStateBF16><<<grid, kThreads, 0, st>>>(a, span);
  else
    k_attend_finish<kStateF16><<<grid, kThreads, 0, st>>>(a, span);
  DGS_LAUNCH_CHECK();
}

}  // namespace dgs
