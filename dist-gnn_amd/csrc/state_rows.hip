// state_rows.hip -- rows of the 4-bit state cache: writing (quantise and store) and reading.
//
// A group of `group` channels x of a row is held as codes c in 0..15, a scale s and a base b:
//   r = max x - min x,  s = bf16(r * fl(1/15)),  b = bf16(min x),  c = clamp(rint((x - b) / s), 0, 15)
// (r and the product in 32 bits) with the quotient taken exactly (ties to even), so that a code never
// depends on the order or width of the arithmetic; s = 0 gives c = 0.  Scale and base are rounded to 16
// bits because they are read with every row: 32-bit ones would add 8 bytes to the 72 of a row of 128
// channels in groups of 64.  b is exact for bfloat16 inputs, and the codes are taken against the rounded
// s and b, so their rounding costs at most 15 s / 512 + |b| / 512 at the ends of the range.  A group that
// holds a NaN or an infinity, or whose s or b is not finite, reads back as NaN (s = b = NaN).
#include <algorithm>

#include "dgs_lane.cuh"
#include "dgs_state.cuh"

namespace dgs {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t bf16_rne(float x) {
  union {
    __bf16 h;
    uint16_t u;
  } v;
  v.h = (__bf16)x;
  return v.u;
}

// The eight codes of a word.  The quotient in 32 bits is off by at most 4 of its units in the last place
// (a half in x - b and in the product, one in the reciprocal), 4e-6 below 16.  Within 1e-5 of a rounding
// border h (a multiple of a half) the sign of (x - b) - h s decides, which 32 bits give exactly: h s has
// 13 bits, the difference to the rounded x - b is exact because the two nearly cancel, and what x - b lost
// in rounding is added (an error-free difference).  Of bfloat16 inputs one in some hundreds lies on a
// border, so that most waves have one or two: a branch a channel, which the wave takes for those only.
// Scales too small or too large for a normal reciprocal take the quotient in 64 bits, where it is exact
// enough by far.  Adding 1.5 * 2^23 rounds to an integer and leaves it in the low bits.
constexpr float kNear = 0.5f - 1e-5f, kMagic = 12582912.f;
constexpr uint32_t kMagicBits = 0x4b400000u + (0x4b400000u << 4) + (0x4b400000u << 8);  // a word's
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float b, float s) {
  if (!(s >= 1e-30f && s <= 1e30f)) {
    uint32_t w = 0;
    for (int i = 0; i < 8; ++i) {
      const double t = s == 0.f ? 0. : ((double)x[i] - (double)b) / (double)s;
      w |= (uint32_t)fmin(fmax(rint(t), 0.), 15.) << (4 * i);
    }
    return w;
  }
  const float inv = __builtin_amdgcn_rcpf(s);
  uint32_t w = 0u - kMagicBits;
  bool near[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = __builtin_amdgcn_fmed3f((x[i] - b) * inv, 0.f, 15.f), r = t + kMagic;
    near[i] = fabsf(t - (r - kMagic)) > kNear;
    w += __float_as_uint(r) << (4 * i);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!__any(near[i])) continue;
    const float d = x[i] - b, back = x[i] - d, t = __builtin_amdgcn_fmed3f(d * inv, 0.f, 15.f);
    const float lost = (back - b) + (x[i] - (d + back));
    const float low = floorf(t), h = low + 0.5f;
    const float e = __builtin_fmaf(-h, s, d) + lost;
    const uint32_t c = (uint32_t)low, up = e > 0.f || (e == 0.f && (c & 1)) ? 1u : 0u;
    w = near[i] ? (w & ~(15u << (4 * i))) | (c + up) << (4 * i) : w;
  }
  return w;
}

struct WriteArgs {
  StateView c;
  StateRows x;
  int64_t n, t0;  // tokens, the launch's first
  const int64_t *slots;  // flat slots, or null: append
  IdArray table, lens;
  int64_t width;
  int64_t *slots_out;
  StateGuard gd;
};

// The flat slot of token t (-1: skipped; an id outside the cache is reported and skipped).
__device__ __forceinline__ int64_t write_slot(const WriteArgs &a, int64_t t, bool report) {
  if (a.slots) {
    const int64_t s = a.slots[t];
    const uint64_t total = (uint64_t)a.c.pages << a.c.pshift;
    if (s >= 0 && (uint64_t)s >= total) {
      if (report) report_bad_id(a.gd.err, kAsyncErrSlot, s, total, a.gd.tag);
      return -1;
    }
    return s < 0 ? -1 : s;
  }
  const int64_t len = a.lens[t], room = a.width << a.c.pshift;
  if ((uint64_t)len >= (uint64_t)room) {
    if (report) report_bad_id(a.gd.err, kAsyncErrLength, len, room, a.gd.tag);
    return -1;
  }
  const int64_t page = a.table[t * a.width + (len >> a.c.pshift)];
  if ((uint64_t)page >= (uint64_t)a.c.pages) {
    if (report) report_bad_id(a.gd.err, kAsyncErrSlot, page, a.c.pages, a.gd.tag);
    return -1;
  }
  return (page << a.c.pshift) | (len & ((int64_t(1) << a.c.pshift) - 1));
}

// LPG lanes (a power of two, at least group / 8) share a group; a lane holds eight channels.  Block
// row y: 0 = K, 1 = V.  A group of lanes takes kWU units (group `g` of head h of token t: unit (t heads
// + h) ng + g) that follow each other, for their loads to overlap; SAME: they belong to one token, whose
// slot is looked up once, while the rows are on their way: with a look-up a unit the kernel took 109 us
// for 65536 tokens of 8 heads x 128 bfloat16 channels (343 MB) to scattered slots, now 93, 3.7 TB/s;
// dense rows to consecutive slots 70, as fast as a copy.  2 and 8 units: 1 to 8 us more.
constexpr int kWU = 4;
template <int TYPE, int LPG, bool SAME>
__global__ __launch_bounds__(kThreads) void k_state_write(WriteArgs a, uint32_t units,
                                                          FastDivU32 per_token, FastDivU32 per_head) {
  const int words = a.c.group >> 3, ng = (int)per_head.d;
  const int sub = threadIdx.x % LPG;
  const bool live = sub < words;
  const int kv = blockIdx.y;
  const uint32_t u0 = (blockIdx.x * (kThreads / LPG) + threadIdx.x / LPG) * kWU;
  if (u0 >= units) return;  // whole groups of lanes
  const void *src = kv ? a.x.v : a.x.k;
  const int64_t st = kv ? a.x.vt : a.x.kt, sh = kv ? a.x.vh : a.x.kh;
  float x[kWU][8];
  int64_t slot[kWU];
  int h[kWU], g[kWU];
  uint32_t t[kWU];
#pragma unroll
  for (int i = 0; i < kWU; ++i) {
    const uint32_t u = u0 + i < units ? u0 + i : u0;
    t[i] = SAME && i > 0 ? t[0] : per_token.div(u);
    const uint32_t r = u - t[i] * per_token.d;
    h[i] = (int)per_head.div(r);
    g[i] = (int)(r - h[i] * per_head.d);
    load8<TYPE>(src, (a.t0 + t[i]) * st + h[i] * sh + g[i] * a.c.group + (live ? sub : 0) * 8, x[i]);
  }
#pragma unroll
  for (int i = 0; i < kWU; ++i) {
    if (SAME && i > 0) {
      slot[i] = slot[0];
      continue;
    }
    const bool in = u0 + i < units;
    slot[i] = in ? write_slot(a, a.t0 + t[i], sub == 0) : -1;
    if (in && a.slots_out && sub == 0 && h[i] == 0 && g[i] == 0 && kv == 0)
      a.slots_out[a.t0 + t[i]] = slot[i];
  }
#pragma unroll
  for (int i = 0; i < kWU; ++i) {
    // NaN passes through minimum and maximum, an infinity shows in the range
    float lo = x[i][0], hi = x[i][0];
#pragma unroll
    for (int y = 1; y < 8; ++y) {
      lo = __builtin_elementwise_minimum(lo, x[i][y]);
      hi = __builtin_elementwise_maximum(hi, x[i][y]);
    }
#pragma unroll
    for (int o = 1; o < LPG; o <<= 1) {
      lo = __builtin_elementwise_minimum(lo, lane_xor32v(lo, o));
      hi = __builtin_elementwise_maximum(hi, lane_xor32v(hi, o));
    }
    if (slot[i] < 0) continue;
    const float range = hi - lo;
    uint32_t sb = bf16_rne(range * (1.f / 15.f)), bb = bf16_rne(lo);
    const float s = bf16_bits(sb << 16), b = bf16_bits(bb << 16);
    uint32_t w = 0;
    if (range - range == 0.f && b - b == 0.f)
      w = codes_of(x[i], b, s);
    else
      sb = bb = 0x7fc0u;
    const int64_t row = (((slot[i] >> a.c.pshift) * a.c.heads + h[i]) << a.c.pshift) +
                        (slot[i] & ((int64_t(1) << a.c.pshift) - 1));
    if (live)
      *(uint32_t *)((kv ? a.c.vc : a.c.kc) + row * (a.c.dim >> 1) + ((g[i] * a.c.group) >> 1) +
                    4 * sub) = w;
    if (sub == 0) (kv ? a.c.vs : a.c.ks)[row * ng + g[i]] = sb | (bb << 16);
  }
}

// A lane writes 16 bytes of output (four or eight channels): piece i of K (block row 0) or V (1) is
// the i-th 16 bytes of the output.  kRU pieces a lane are in flight.  Bound by HBM: 65536 rows of 8
// heads x 128 channels as 32-bit floats (612 MB) in 112 us, 5.5 TB/s; 400000 scattered rows of 128
// (467 MB) in 88 us, 115 with stores that pass through the caches.
constexpr int kRU = 4;
template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_state_read(StateView c, const int64_t *slots,
                                                         uint32_t pieces, FastDivU32 per_row,
                                                         FastDivU32 heads, void *out_k, void *out_v,
                                                         StateGuard gd) {
  constexpr int kCh = TYPE == kStateF32 ? 4 : 8;
  const int kv = blockIdx.y, ng = c.dim / c.group;
  const uint8_t *codes = kv ? c.vc : c.kc;
  const uint32_t *words = kv ? c.vs : c.ks;
  const uint64_t total = (uint64_t)c.pages << c.pshift;
  const uint32_t i0 = blockIdx.x * (kThreads * kRU) + threadIdx.x;
  uint32_t q[kRU], m[kRU];
  int64_t slot[kRU];
  uint32_t h[kRU], ch[kRU];
#pragma unroll
  for (int u = 0; u < kRU; ++u) {
    uint32_t i = i0 + u * kThreads;
    i = i < pieces ? i : pieces - 1;
    const uint32_t r = per_row.div(i), t = heads.div(r);
    ch[u] = (i - r * per_row.d) * kCh;
    h[u] = r - t * heads.d;
    slot[u] = slots[t];
  }
#pragma unroll
  for (int u = 0; u < kRU; ++u) {
    const bool in = slot[u] >= 0 && (uint64_t)slot[u] < total;
    if (!in && slot[u] >= 0 && ch[u] == 0 && h[u] == 0 && kv == 0)
      report_bad_id(gd.err, kAsyncErrSlot, slot[u], total, gd.tag);
    const int64_t s = in ? slot[u] : 0;
    const int64_t row = (((s >> c.pshift) * c.heads + h[u]) << c.pshift) +
                        (s & ((int64_t(1) << c.pshift) - 1));
    const uint8_t *at = codes + row * (c.dim >> 1) + (ch[u] >> 1);
    if constexpr (TYPE == kStateF32)
      q[u] = *(const uint16_t *)at;
    else
      q[u] = *(const uint32_t *)at;
    m[u] = words[row * ng + ch[u] / (uint32_t)c.group];
    if (!in) q[u] = m[u] = 0;
  }
#pragma unroll
  for (int u = 0; u < kRU; ++u) {
    const uint32_t i = i0 + u * kThreads;
    if (i >= pieces) break;
    float x[8];
    codes8(q[u], x);
    const float s = scale_of(m[u]), b = base_of(m[u]);
#pragma unroll
    for (int y = 0; y < kCh; ++y) x[y] = x[y] * s + b;
    su32x4 *dst = (su32x4 *)(kv ? out_v : out_k) + i;
    su32x4 v;
    if constexpr (TYPE == kStateF32) {
#pragma unroll
      for (int y = 0; y < 4; ++y) v[y] = __float_as_uint(x[y]);
    } else {
      store8<TYPE>(&v, 0, x);
    }
    __builtin_nontemporal_store(v, dst);
  }
}

int shift_of(int words) {
  int s = 0;
  while ((1 << s) < words) ++s;
  return s;
}

template <int TYPE, int LPG>
void launch_write_l(const WriteArgs &a, int64_t n, hipStream_t st) {
  const uint32_t ng = a.c.dim / a.c.group, per_token = a.c.heads * ng;
  const uint32_t units = (uint32_t)(n * per_token);
  const FastDivU32 ft = FastDivU32::make(per_token), fh = FastDivU32::make(ng);
  const dim3 grid((unsigned)ceil_div((int64_t)units * LPG, kThreads * kWU), 2);
  if (per_token % kWU == 0)
    k_state_write<TYPE, LPG, true><<<grid, kThreads, 0, st>>>(a, units, ft, fh);
  else
    k_state_write<TYPE, LPG, false><<<grid, kThreads, 0, st>>>(a, units, ft, fh);
  DGS_LAUNCH_CHECK();
}
template <int TYPE>
void launch_write_t(const WriteArgs &a, int64_t n, hipStream_t st) {
  switch (shift_of(a.c.group >> 3)) {
    case 0: launch_write_l<TYPE, 1>(a, n, st); break;
    case 1: launch_write_l<TYPE, 2>(a, n, st); break;
    case 2: launch_write_l<TYPE, 4>(a, n, st); break;
    case 3: launch_write_l<TYPE, 8>(a, n, st); break;
    case 4: launch_write_l<TYPE, 16>(a, n, st); break;
    default: launch_write_l<TYPE, 32>(a, n, st); break;
  }
}
// Units and pieces of a launch are counted in 32 bits: more tokens take several launches.
int64_t tokens_a_launch(const StateView &c) {
  return std::max<int64_t>(1, (int64_t(1) << 30) / ((int64_t)c.heads * c.dim));
}
void launch_write(WriteArgs a, StateType type, hipStream_t st) {
  const int64_t step = tokens_a_launch(a.c);
  for (a.t0 = 0; a.t0 < a.n; a.t0 += step) {
    const int64_t n = std::min(step, a.n - a.t0);
    if (type == kStateF32)
      launch_write_t<kStateF32>(a, n, st);
    else if (type == kStateBF16)
      launch_write_t<kStateBF16>(a, n, st);
    else
      launch_write_t<kStateF16>(a, n, st);
  }
}
template <int TYPE>
void launch_read(const StateView &c, const int64_t *slots, int64_t n, void *k_out, void *v_out,
                 const StateGuard &gd, hipStream_t st) {
  constexpr int kCh = TYPE == kStateF32 ? 4 : 8;
  const uint32_t pieces = (uint32_t)(n * c.heads * (c.dim / kCh));
  const dim3 grid((unsigned)ceil_div(pieces, kThreads * kRU), 2);
  const FastDivU32 fr = FastDivU32::make(c.dim / kCh), fh = FastDivU32::make(c.heads);
  k_state_read<TYPE><<<grid, kThreads, 0, st>>>(c, slots, pieces, fr, fh, k_out, v_out, gd);
  DGS_LAUNCH_CHECK();
}

}  // namespace

void state_write(const StateView &c, const StateRows &x, StateType type, int64_t n,
                 const int64_t *slots, hipStream_t st) {
  WriteArgs a{};
  a.c = c;
  a.x = x;
  a.n = n;
  a.slots = slots;
  a.gd = state_guard();
  launch_write(a, type, st);
}

void state_append(const StateView &c, const StateRows &x, StateType type, int64_t n,
                  const IdArray &table, int64_t width, const IdArray &lens, int64_t *slots_out,
                  hipStream_t st) {
  WriteArgs a{};
  a.c = c;
  a.x = x;
  a.n = n;
  a.table = table;
  a.lens = lens;
  a.width = width;
  a.slots_out = slots_out;
  a.gd = state_guard();
  launch_write(a, type, st);
}

void state_read(const StateView &c, const int64_t *slots, int64_t n, StateType type, void *k_out,
                void *v_out, hipStream_t st) {
  if (n <= 0) return;
  const StateGuard gd = state_guard();
  const int64_t step = tokens_a_launch(c);
  const int64_t row = (int64_t)c.heads * c.dim * (type == kStateF32 ? 4 : 2);
  for (int64_t t = 0; t < n; t += step) {
    const int64_t m = std::min(step, n - t);
    void *k = (char *)k_out + t * row, *v = (char *)v_out + t * row;
    if (type == kStateF32)
      launch_read<kStateF32>(c, slots + t, m, k, v, gd, st);
    else if (type == kStateBF16)
      launch_read<kStateBF16>(c, slots + t, m, k, v, gd, st);
    else
      launch_read<kStateF16>(c, slots + t, m, k, v, gd, st);
  }
}

}  // namespace dgs
