// state_rows.hip -- rows of the 4-bit state cache: writing (quantise and store) and reading.
//
// A group of `group` channels x of a row is held as codes c in 0..15, a scale s and a base b:
//   r = max x - min x,  s = bf16(r * fl(1/15)),  b = bf16(min x),  c = clamp(rint((x - b) / s), 0, 15)
// (r and the product in 32 bits) with the quotient taken exactly (ties to even), so that a code never depends on the order or
// width of the arithmetic; s = 0 gives c = 0.  Scale and base are rounded to 16 bits because they
// are read with every row: 32-bit ones would add 8 bytes to the 72 of a row of 128 channels in
// groups of 64.  b is exact for bfloat16 inputs, and the codes are taken against the rounded s
// and b, so their rounding costs at most 15 s / 512 + |b| / 512 at the ends of the range.  A group
// that holds a NaN or an infinity, or whose s or b is not finite, reads back as NaN (s = b = NaN).
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

// One code.  The quotient in 32 bits is off by at most 2.5 of its units in the last place (one
// rounding in x - b, one in the reciprocal, one in the product), 2.5e-6 below 16; within 1e-5 of
// a rounding border, and for scales too small for a normal reciprocal, it is taken in 64 bits,
// where x - b and s are exact and the quotient's distance from a border survives its rounding.
__device__ __forceinline__ uint32_t code_of(float x, float b, float s, float inv, bool tiny) {
  const float t = (x - b) * inv;
  float r = rintf(t);
  if (tiny || fabsf(fabsf(t - r) - 0.5f) < 1e-5f)
    r = s == 0.f ? 0.f : (float)rint(fmin(fmax(((double)x - (double)b) / (double)s, -1.0), 16.0));
  return (uint32_t)fminf(fmaxf(r, 0.f), 15.f);
}

struct WriteArgs {
  StateView c;
  StateRows x;
  int64_t n;
  const int64_t *slots;  // flat slots, or null: append
  IdArray table, lens;
  int64_t width;
  int64_t *slots_out;
  GatherGuard gd;
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

// LPG lanes (a power of two, at least group / 8) share a group; a lane holds eight channels.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_state_write(WriteArgs a, int lpg_shift) {
  const int lpg = 1 << lpg_shift, words = a.c.group >> 3, ng = a.c.dim / a.c.group;
  const int64_t units = a.n * 2 * a.c.heads * ng;
  const int64_t u =
      ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> lpg_shift;
  if (u >= units) return;  // whole groups of lanes leave together
  const int sub = threadIdx.x & (lpg - 1);
  const int g = (int)(u % ng);
  const int64_t r = u / ng;
  const int h = (int)(r % a.c.heads);
  const int kv = (int)((r / a.c.heads) & 1);
  const int64_t t = r / (2 * a.c.heads);
  const int64_t slot = write_slot(a, t, sub == 0);
  if (a.slots_out && sub == 0 && g == 0 && h == 0 && kv == 0) a.slots_out[t] = slot;
  if (slot < 0) return;
  const bool live = sub < words;
  const int ch = g * a.c.group + (live ? sub : 0) * 8;
  float x[8];
  if (kv == 0)
    load8<TYPE>(a.x.k, t * a.x.kt + h * a.x.kh + ch, x);
  else
    load8<TYPE>(a.x.v, t * a.x.vt + h * a.x.vh + ch, x);
  float lo = x[0], hi = x[0], bad = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad += x[i] - x[i];  // NaN when x is NaN or infinite
  }
  for (int o = lpg >> 1; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor(lo, o, 64));
    hi = fmaxf(hi, __shfl_xor(hi, o, 64));
    bad += __shfl_xor(bad, o, 64);
  }
  uint32_t sb = bf16_rne((hi - lo) * (1.f / 15.f)), bb = bf16_rne(lo);
  const float s = bf16_bits(sb << 16), b = bf16_bits(bb << 16);
  const bool nan = !(bad == 0.f) || !(s - s == 0.f) || !(b - b == 0.f);
  uint32_t w = 0;
  if (!nan) {
    const bool tiny = !(s >= 1e-30f);
    const float inv = tiny ? 0.f : 1.f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= code_of(x[i], b, s, inv, tiny) << (4 * i);
  } else {
    sb = bb = 0x7fc0u;
  }
  const int64_t page = slot >> a.c.pshift;
  const int64_t row = ((page * a.c.heads + h) << a.c.pshift) +
                      (slot & ((int64_t(1) << a.c.pshift) - 1));
  if (live)
    *(uint32_t *)((kv ? a.c.vc : a.c.kc) + row * (a.c.dim >> 1) + (ch >> 1)) = w;
  if (sub == 0) (kv ? a.c.vs : a.c.ks)[row * ng + g] = sb | (bb << 16);
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_state_read(StateView c, const int64_t *slots,
                                                         int64_t n, void *k_out, void *v_out,
                                                         GatherGuard gd) {
  const int words = c.dim >> 3;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= n * 2 * c.heads * words) return;
  const int w = (int)(i % words);
  const int64_t r = i / words;
  const int h = (int)(r % c.heads);
  const int64_t t = (r / c.heads) >> 1;
  const int kv = (int)((r / c.heads) & 1);
  const int64_t slot = slots[t];
  const uint64_t total = (uint64_t)c.pages << c.pshift;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && (uint64_t)slot < total) {
    const int64_t row = (((slot >> c.pshift) * c.heads + h) << c.pshift) +
                        (slot & ((int64_t(1) << c.pshift) - 1));
    const uint32_t q = *(const uint32_t *)((kv ? c.vc : c.kc) + row * (c.dim >> 1) + 4 * w);
    const uint32_t m = (kv ? c.vs : c.ks)[row * (c.dim / c.group) + (8 * w) / c.group];
    const float s = scale_of(m), b = base_of(m);
    codes8(q, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * s + b;
  } else if (slot >= 0 && w == 0 && h == 0 && kv == 0) {
    report_bad_id(gd.err, kAsyncErrSlot, slot, total, gd.tag);
  }
  store8<TYPE>(kv ? v_out : k_out, (t * c.heads + h) * c.dim + 8 * w, x);
}

int shift_of(int words) {
  int s = 0;
  while ((1 << s) < words) ++s;
  return s;
}

void launch_write(const WriteArgs &a, StateType type, hipStream_t st) {
  if (a.n <= 0) return;
  const int sh = shift_of(a.c.group >> 3);
  const int64_t lanes = (a.n * 2 * a.c.heads * (a.c.dim / a.c.group)) << sh;
  const int64_t blocks = ceil_div(lanes, kThreads);
  DGS_CHECK(blocks < (int64_t(1) << 31), "state write: too many rows in one call");
  if (type == kStateF32)
    k_state_write<kStateF32><<<(unsigned)blocks, kThreads, 0, st>>>(a, sh);
  else if (type == kStateBF16)
    k_state_write<kStateBF16><<<(unsigned)blocks, kThreads, 0, st>>>(a, sh);
  else
    k_state_write<kStateF16><<<(unsigned)blocks, kThreads, 0, st>>>(a, sh);
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
  a.gd = state_guard(kAsyncErrSlot, c.pages);
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
  a.gd = state_guard(kAsyncErrSlot, c.pages);
  launch_write(a, type, st);
}

void state_read(const StateView &c, const int64_t *slots, int64_t n, StateType type, void *k_out,
                void *v_out, hipStream_t st) {
  if (n <= 0) return;
  const GatherGuard gd = state_guard(kAsyncErrSlot, c.pages);
  const int64_t blocks = ceil_div(n * 2 * c.heads * (c.dim >> 3), kThreads);
  DGS_CHECK(blocks < (int64_t(1) << 31), "state read: too many rows in one call");
  if (type == kStateF32)
    k_state_read<kStateF32><<<(unsigned)blocks, kThreads, 0, st>>>(c, slots, n, k_out, v_out, gd);
  else if (type == kStateBF16)
    k_state_read<kStateBF16>
        <<<(unsigned)blocks, kThreads, 0, st>>>(c, slots, n, k_out, v_out, gd);
  else
    k_state_read<kStateF16><<<(unsigned)blocks, kThreads, 0, st>>>(c, slots, n, k_out, v_out, gd);
  DGS_LAUNCH_CHECK();
}

}  // namespace dgs
